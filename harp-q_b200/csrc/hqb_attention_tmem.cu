// Attention of drafted trees over a paged cache on the tcgen05 tensor cores: tiles of up to 256
// query rows of one (request, key head) against blocks of 128 keys (see hqb_attention.cuh for the
// division of the work).
#include <cuda.h>
#include <cuda_runtime.h>

#include "hqb_attention.cuh"
#include "hqb_internal.h"

namespace hqb {
namespace {

constexpr uint32_t kKeys = 128;      // keys of a block
constexpr uint32_t kRows = 128;      // tensor-memory lanes: rows of one score tile
constexpr uint32_t kKeysWarp = 8;    // tensor-map copies of keys and queries
constexpr uint32_t kCopyWarp = 9;    // plain copies, and the values' last rows
constexpr uint32_t kMmaWarp = 10;
constexpr uint32_t kValuesWarp = 11; // tensor-map copies of values
constexpr uint32_t kTmemThreads = 384;  // warps 0-7 softmax

// One segment as the MMA and softmax warps see it, written by the loading warp.
struct Segment {
  Request q;
  uint32_t head, row0, b0, n;  // n 0: there are no more
  uint32_t two;                // the tile has rows for both score tiles
  uint32_t pad;
};

struct Bars {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4], fix_full[4];
  uint64_t q_full[2], q_empty, s_full[2], p_full[2][2], o_full[2], o_free, joint, drain;
  uint32_t tmem, abort;
  uint32_t broken[8][8];  // by segment: drafted nodes with an infinity or NaN among their values
  Segment segments[4];
};

template <int DP>
struct TmemShape {
  static constexpr uint32_t kHalf = kRows * 128;  // 128 rows of 64 columns
  static constexpr uint32_t kTile = kRows * DP * 2;  // a score tile's queries; a block of keys or of values
  // blocks of keys and of values in flight (values are held for longer)
  static constexpr uint32_t kKeySlots = DP == 128 ? 2 : 4, kValueSlots = DP == 128 ? 3 : 4;
  static constexpr uint32_t kKeyRing = 2 * kTile, kValueRing = kKeyRing + kKeySlots * kTile;
  static constexpr uint32_t kBars = kValueRing + kValueSlots * kTile;
  static constexpr uint32_t kStats = kBars + (sizeof(Bars) + 15) / 16 * 16;
  static constexpr uint32_t kBytes = kStats + 256 * 8;
};

// Tensor maps, all in boxes of 64 columns in 128-byte-swizzled rows: the cache's k and v as
// (column, head, token, page) with boxes of box_rows tokens, a power of two from 8 to 128 that
// divides the page size (0: the cache has no maps and comes by plain copies); the step's own q
// (boxes of half a tile: the group's heads of kRows / group nodes), k and v (boxes of a block)
// as (column, head, token).
struct Maps {
  CUtensorMap ck, cv, q, k, v;
  uint32_t box_rows;
};

// Mathematics: the one-pass softmax of attention_rows_kernel.  A running reference m stands in
// for the maximum: it follows the maximum (less kWeightShift) only when that has grown by more than
// kSlack in the exponent, so weights stay within the type and the sums in tensor memory are rarely
// rescaled; the result is the same sum up to rounding.
// Roles: 4 + 4 warps take the scores of two streams out of tensor memory (a thread a row: no
// shuffles), turn them into weights and put those back, packed in 16 bits over the scores, as
// the A operand of weights x values; a warp brings keys and queries, another one values, into
// 128-byte-swizzled shared memory by tensor-map copies through the page table; one warp issues
// the MMAs of both streams, which keeps them apart (a warp a stream let them fall into step, 3 % slower).
// The last rows of values (past the context's end, drafted nodes) pass a warp that zeroes what must not
// reach a sum.  A tile of more rows than one score tile has its two halves as
// streams, over the same keys (each block is loaded once for both); a smaller tile has the even
// and the odd blocks as streams, joined at the end, so that the scores of one stream are computed
// while the other's weights are.
// Tensor memory: scores 2 x 128 columns, sums 2 x DP columns.  Shared memory at DP 128: queries
// 64 KB, rings of two blocks of keys and three of values, 32 KB each (three and two: 3 % slower).
// Measured, B200, BF16, 64 heads over 8 of 128, 32 trees of up to 64 nodes over up to 8192 tokens: 315 us in a
// short burst (773 TFLOP/s), 380 us in a long loop (641), where the card's power limit holds the clock at 1.5 GHz.
// The profiled launch: 317 us, 126 blocks a CTA, 4040 cycles a block at its 1.6 GHz, the tensor pipe active in 52 %.
// Of these a block of two score tiles takes 3500 between two others: per stream 2250 of softmax (490 to read
// the scores and find the maximum, 880 for each half of the exponentials), then 1100 for 4 + 8 MMAs to the next
// scores, and barriers; the rest are the ends of segments and the first scores of the next.
// Weights are rounded to 16 bits as in attention_rows_kernel, for the same reasons.
// 7 trees of up to 33 nodes over up to 3001 tokens, 12 heads over 4 of 64, FP16: 17.4 us with the join, bound by
// latency (lengths and work division 1.8 us, first scores 2.3, blocks 5, sums and join 6).
template <typename T, int DP>
__global__ void __launch_bounds__(kTmemThreads, 1) attention_tmem_kernel(const __grid_constant__ AttnParams p,
                                                                          const __grid_constant__ Maps maps) {
  using S = TmemShape<DP>;
  extern __shared__ __align__(1024) uint8_t sm[];
  Bars& bars = *reinterpret_cast<Bars*>(sm + S::kBars);
  float2* stats = reinterpret_cast<float2*>(sm + S::kStats);
  volatile uint32_t* abort = &bars.abort;
  const uint32_t tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  uint32_t bad = 0;
  if ((smem_u32(sm) & 1023u) != 0) {  // the swizzle goes by address bits
    griddep_wait();
    if (tid == 0) atomicOr(p.error, HQB_DEVERR_LAUNCH);
    return;
  }
  if (warp == kMmaWarp && lane < 5) {
    const CUtensorMap* all[5] = {&maps.q, &maps.k, &maps.v, &maps.ck, &maps.cv};
    if (lane < 3 || maps.box_rows != 0) prefetch_map(all[lane]);
  }
  if (tid < 64) bars.broken[tid >> 3][tid & 7] = 0;
  if (tid == 0) {
    for (uint32_t i = 0; i < 4; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      mbar_init(&bars.fix_full[i], 1);
    }
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.q_full[i], 1);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i][0], 4);
      mbar_init(&bars.p_full[i][1], 4);
      mbar_init(&bars.o_full[i], 1);
    }
    mbar_init(&bars.o_free, 8);
    mbar_init(&bars.joint, 8);
    mbar_init(&bars.drain, 1);
    bars.abort = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&bars.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(bars.tmem);
  // only now: a dependent that shared the SM and took tensor memory first would wait for this grid,
  // and this CTA for it
  griddep_launch_dependents();
  griddep_wait();
  // a wait that runs out ends every role's loop; nothing is left in flight but this CTA's copies
  // (for a whole warp, whose lanes must go on or stop together)
  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity & 1u))) return true;
    const bool stop = *abort != 0;
    const bool got = !stop && mbar_wait(bar, parity & 1u, p.error);
    if (!stop && !got) *abort = 1u;
    return __all_sync(0xffffffffu, got);
  };
  // a warp's one arrival: 32 lanes' would queue at the barrier
  auto arrive_warp = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  const uint32_t half = p.rows / 2;  // rows of a tile's first score tile
  // Segment seg is announced by phase seg / 2 of q_full[seg & 1].  No warp can be two phases of one
  // barrier late: segment seg + 2 is announced after q_empty of segment seg + 1, which is committed
  // after o_free of segment seg, to which every softmax warp arrives at its end.  For the same
  // reason segments[seg & 3] stays while it is read.
  auto segment = [&](uint32_t seg) -> const Segment* {
    if (!wait_all(&bars.q_full[seg & 1], seg >> 1)) return nullptr;
    const Segment* s = &bars.segments[seg & 3];
    return *const_cast<const volatile uint32_t*>(&s->n) == 0 ? nullptr : s;
  };
  if (warp >= 8) {
    if (warp != kMmaWarp) {
      Walk w;
      const bool work = w.begin(p, blockIdx.x, bad);
      if (!work) w.left = 0;
      const uint32_t dim = p.c.head_dim;
      // Keys and values have a ring of blocks each; block i of a segment takes the ring's next slot, whose
      // turns are told apart by the one warp that fills it in every turn: the keys' warp and the values'
      // warp, or without maps of the cache the copying warp both.  A block is announced once on k_full
      // or v_full.
      const bool mapped = maps.box_rows != 0;
      struct Ring {
        uint32_t slots, slot, turn;
        __device__ __forceinline__ void next() {
          if (++slot == slots) slot = 0, ++turn;
        }
      } keys{S::kKeySlots, 0, 0}, values{S::kValueSlots, 0, 0};
      uint32_t seg = 0;
      uint32_t fixed = 0, fix_turn = 0;  // a bit a slot of values: its last copy went to fix_full, that one's next phase
      bool ok = true;
      // one of the segment's blocks: where its keys begin, among the cached ones or the nodes, and how many
      struct Block {
        bool cached, fix;  // fix: has values to clear
        uint32_t first, valid;
      };
      auto block = [&](uint32_t b) -> Block {
        const bool cached = b < w.q.cached_blocks;
        const uint32_t first = (cached ? b : b - w.q.cached_blocks) * kKeys;
        const uint32_t valid = min(kKeys, (cached ? w.q.ctx : w.q.nodes) - first);
        return {cached, !cached || valid < kKeys, first, valid};
      };
      auto drafted = [&](uint32_t dst, const CUtensorMap* map, uint64_t* bar, uint32_t first) {
        if (lane == 0) mbar_expect_tx(bar, S::kTile);
        __syncwarp();
        if (lane < DP / 64) tma_load_3d(dst + lane * S::kHalf, map, bar, lane * 64, w.head, w.q.start + first);
      };
      if (warp != kCopyWarp) {
        // ---- keys and queries, or values, by tensor-map copies.  (Instructions are fetched from as far as
        // L2, so the loop is kept short and divisions out of it; one warp for both took 1900 cycles a copy,
        // and everything waited for it.)
        const bool is_values = warp == kValuesWarp;
        const CUtensorMap* const cache_map = is_values ? &maps.cv : &maps.ck;
        const CUtensorMap* const step_map = is_values ? &maps.v : &maps.k;
        uint64_t* const empty = is_values ? bars.v_empty : bars.k_empty;
        uint64_t* const full = is_values ? bars.v_full : bars.k_full;
        Ring ring = is_values ? values : keys;
        const uint32_t ring_at = smem_u32(sm) + (is_values ? S::kValueRing : S::kKeyRing);
        // a lane a box: box `box` of the block, columns 64 h ..
        const uint32_t box_shift = mapped ? 31 - __clz(maps.box_rows) : 0;
        const uint32_t h = lane >> (7 - box_shift), box = lane & ((kKeys >> box_shift) - 1);
        const uint32_t lane_at = h * S::kHalf + (box << box_shift) * 128;
        while (ok && w.left != 0) {
          w.open(p);
          const uint32_t rows = w.q.nodes * p.group, row0 = w.tile * p.rows, n = w.b1 - w.b0;
          const bool two = rows - row0 > half;
          const int32_t* table = p.a.tables + static_cast<uint64_t>(w.r) * p.a.table_stride;
          // the page of the lane's box, looked up while the block before is loaded
          uint32_t page = 0, inside = 0;
          auto locate = [&](uint32_t b) {
            const uint32_t key = b * kKeys + (box << box_shift), column = p.by_page.quotient(key);
            const bool real = b < w.q.cached_blocks && key < w.q.ctx && h < DP / 64;
            page = real ? static_cast<uint32_t>(table[column]) : 0u;
            inside = key - column * p.c.page_size;
          };
          if (mapped) locate(w.b0);
          for (uint32_t b = w.b0; b < w.b1; ++b) {
            if (mapped) {
              const Block x = block(b);
              const uint32_t slot = ring.slot, dst = ring_at + slot * S::kTile;
              if (ring.turn > 0 && !(ok = wait_all(&empty[slot], ring.turn - 1))) break;
              uint64_t* bar = &full[slot];
              if (is_values) {
                fixed &= ~(1u << slot);
                if (x.fix) {
                  bar = &bars.fix_full[slot];
                  fixed |= 1u << slot;
                  fix_turn ^= 1u << slot;
                }
              }
              ring.next();
              if (x.cached) {
                if (page >= p.c.num_pages) {
                  bad |= HQB_DEVERR_PAGES;
                  page = 0;
                }
                // boxes past the end of the context are left out (scores of what lies there are hidden,
                // values are cleared)
                const uint32_t real = (x.valid + maps.box_rows - 1) >> box_shift;
                if (lane == 0) mbar_expect_tx(bar, (real << box_shift) * (DP * 2));
                __syncwarp();
                if (h < DP / 64 && box < real) tma_load_4d(dst + lane_at, cache_map, bar, h * 64, w.head, inside, page);
              } else {
                drafted(dst, step_map, bar, x.first);
              }
              if (b + 1 < w.b1) locate(b + 1);
            }
            if (b != w.b0 || is_values) continue;
            // The queries go after the first keys, once the last segment's have been read.  Only the keys' warp
            // may wait for q_empty: a warp that the MMAs do not wait for in every segment could find it two
            // phases on.
            if (seg > 0 && !(ok = wait_all(&bars.q_empty, seg - 1))) break;
            uint64_t* q_full = &bars.q_full[seg & 1];
            // past here the epilogue of segment seg - 3 is over: the flags of segment seg - 4 are free
            if (lane < 8) bars.broken[(seg + 4) & 7][lane] = 0;
            const uint32_t tiles = two ? 2u : 1u;
            if (lane == 0) {
              bars.segments[seg & 3] = Segment{w.q, w.head, row0, w.b0, n, two ? 1u : 0u, 0u};
              mbar_expect_tx(q_full, tiles * half * DP * 2);
            }
            __syncwarp();
            if (lane < tiles * (DP / 64)) {
              const uint32_t t = lane / (DP / 64), c = lane % (DP / 64);
              tma_load_3d(smem_u32(sm + t * S::kTile + c * S::kHalf), &maps.q, q_full, c * 64, w.head * p.group,
                          w.q.start + p.by_group.quotient(row0 + t * half));
            }
          }
          ++seg;
          w.advance(p, bad);
        }
        if (ok && !is_values) {  // the end: with the last queries read, so that no announcement is overtaken
          if (seg > 0) ok = wait_all(&bars.q_empty, seg - 1);
          if (ok && lane == 0) {
            bars.segments[seg & 3].n = 0;
            mbar_arrive(&bars.q_full[seg & 1]);
          }
        }
        if (is_values) values = ring;
        else keys = ring;
      } else {
        // ---- rows of values past the end and drafted nodes' infinities; without maps of the cache all blocks
        if (lane == 0 && !p.whole) note_split(p, w, blockIdx.x, work, bad);
        __syncwarp();
        constexpr uint32_t kPieces = DP / 8;  // 16-byte pieces of a row
        uint32_t waited = 0;  // a bit a slot: the next phase of fix_full
        while (ok && w.left != 0) {
          w.open(p);
          const uint32_t n = w.b1 - w.b0;
          const int32_t* table = p.a.tables + static_cast<uint64_t>(w.r) * p.a.table_stride;
          uint32_t* broken = bars.broken[seg & 7];
          // a block by plain copies; drafted ones by the step's maps
          auto fill = [&](uint32_t b, bool is_values) -> bool {
            const Block x = block(b);
            Ring& ring = is_values ? values : keys;
            const uint32_t slot = ring.slot;
            const uint32_t dst = smem_u32(sm) + (is_values ? S::kValueRing : S::kKeyRing) + slot * S::kTile;
            if (ring.turn > 0 && !wait_all(&(is_values ? bars.v_empty : bars.k_empty)[slot], ring.turn - 1)) return false;
            uint64_t* bar = &(is_values ? bars.v_full : bars.k_full)[slot];
            if (is_values) fixed &= ~(1u << slot);
            if (!x.cached) {
              if (is_values) {
                bar = &bars.fix_full[slot];
                fixed |= 1u << slot;
                fix_turn ^= 1u << slot;
              } else {
                keys.next();
              }
              drafted(dst, is_values ? &maps.v : &maps.k, bar, x.first);
              return true;
            }
            const T* src = static_cast<const T*>(is_values ? p.c.v : p.c.k);
            for (uint32_t r0 = 0; r0 < kKeys; r0 += 32) {
              const uint64_t where = r0 + lane < x.valid ? key_offset(p, table, x.first + r0 + lane, w.head, bad) : 0;
#pragma unroll 4
              for (uint32_t y = 0; y < kPieces; ++y) {
                const uint32_t i = y * 32 + lane, j = i / kPieces, c = i % kPieces, r = r0 + j;
                const uint64_t row = __shfl_sync(0xffffffffu, where, j);
                const bool copy = r < x.valid && c * 8 < dim;
                cp_async16(dst + (c >> 3) * S::kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + (copy ? row + c * 8 : 0),
                           copy ? 16u : 0u);  // (zeros past the end: nothing is left to clear)
              }
            }
            cp_async_commit();
            cp_async_wait<0>();
            fence_proxy_async_smem();
            arrive_warp(bar);
            ring.next();
            return true;
          };
          // a weight of zero must cancel a hidden row of values whatever it holds: rows past the end
          // become zeros, and so do infinities and NaN of drafted nodes, which the rows that see the
          // node get at the end
          auto clear = [&](const Block& x) -> bool {
            const uint32_t slot = values.slot;
            if (!wait_all(&bars.fix_full[slot], waited >> slot)) return false;
            waited ^= 1u << slot;
            uint8_t* const at = sm + S::kValueRing + slot * S::kTile;
            auto piece = [&](uint32_t i) {
              const uint32_t r = i / kPieces, c = i % kPieces;
              return reinterpret_cast<uint4*>(at + (c >> 3) * S::kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4));
            };
            // (the sums' MMAs stop after the 16 keys that hold the last one)
            for (uint32_t i = x.valid * kPieces + lane; i < ((x.valid + 15) & ~15u) * kPieces; i += 32)
              *piece(i) = make_uint4(0, 0, 0, 0);
            for (uint32_t i0 = lane; !x.cached && i0 < x.valid * kPieces; i0 += 32 * 8) {
              uint4 v[8];
#pragma unroll
              for (uint32_t k = 0; k < 8; ++k)
                v[k] = i0 + k * 32 < x.valid * kPieces ? *piece(i0 + k * 32) : make_uint4(0, 0, 0, 0);
#pragma unroll
              for (uint32_t k = 0; k < 8; ++k) {
                constexpr uint32_t kMask = Elem<T>::kExpMask;
                uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                bool found = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if ((u[e] & kMask) == kMask) u[e] &= 0xFFFF0000u, found = true;
                  if ((u[e] >> 16 & kMask) == kMask) u[e] &= 0x0000FFFFu, found = true;
                }
                if (found) {
                  const uint32_t node = x.first + (i0 + k * 32) / kPieces;
                  atomicOr(&broken[node >> 5], 1u << (node & 31));
                  *piece(i0 + k * 32) = make_uint4(u[0], u[1], u[2], u[3]);
                }
              }
            }
            fence_proxy_async_smem();
            arrive_warp(&bars.v_full[slot]);
            return true;
          };
          // (the MMAs ask for up to two blocks of keys before the values of the first)
          for (uint32_t i = 0; i < n; ++i) {
            if (!mapped) {
              if (i == 0 && !(ok = fill(w.b0, false))) break;
              if (i + 1 < n && !(ok = fill(w.b0 + i + 1, false))) break;
              if (!(ok = fill(w.b0 + i, true))) break;
              if (block(w.b0 + i).cached) continue;
            }
            const Block x = block(w.b0 + i);
            if (x.fix && !(ok = clear(x))) break;
            values.next();
          }
          ++seg;
          w.advance(p, bad);
        }
      }
      if (!ok) {  // copies in flight end before the CTA does
        auto drain = [&](const Ring& r, uint64_t* full, bool is_values) {
          for (uint32_t i = 0; i < r.slots; ++i) {
            if (i >= r.slot && r.turn == 0) break;
            if (is_values && (fixed >> i & 1u)) mbar_wait(&bars.fix_full[i], (fix_turn >> i & 1u) ^ 1u, p.error);
            else mbar_wait(&full[i], (i < r.slot ? r.turn : r.turn - 1) & 1u, p.error);
          }
        };
        if (warp == kKeysWarp ? mapped : warp == kCopyWarp && !mapped) drain(keys, bars.k_full, false);
        if (warp == kValuesWarp ? mapped : warp == kCopyWarp && !mapped) drain(values, bars.v_full, true);
      }
      if (bad != 0) atomicOr(p.error, static_cast<int>(bad));
    } else {
      // ---- MMA issuer: the whole warp keeps the schedule, one elected lane issues
      constexpr uint32_t kType = sizeof(T) == 2 && Elem<T>::kExpMask == 0x7F80u ? 1u : 0u;  // BF16 : FP16
      constexpr uint32_t kBase = (1u << 4) | (kType << 7) | (kType << 10) | ((kRows >> 4) << 24);
      constexpr uint32_t kScores = kBase | ((kKeys >> 3) << 17);
      constexpr uint32_t kSums = kBase | (1u << 16) | ((DP >> 3) << 17);  // B (values) MN-major
      uint32_t done = 0, seg = 0, p_at[2] = {0, 0};  // done: blocks of earlier segments
      bool ok = true;
      auto k_wait = [&](uint32_t n) { return wait_all(&bars.k_full[n % S::kKeySlots], n / S::kKeySlots); };
      auto v_wait = [&](uint32_t n) { return wait_all(&bars.v_full[n % S::kValueSlots], n / S::kValueSlots); };
      auto k_done = [&](uint32_t n) { warp_commit(&bars.k_empty[n % S::kKeySlots]); };
      auto v_done = [&](uint32_t n) { warp_commit(&bars.v_empty[n % S::kValueSlots]); };
      // descriptors step by their address field (16-byte units)
      auto scores = [&](uint32_t s, uint32_t tile, uint32_t n) {  // block n's
        const uint32_t qd = uniform(umma_sw128_low(smem_u32(sm + tile * S::kTile), 16));
        const uint32_t kd = uniform(umma_sw128_low(smem_u32(sm) + S::kKeyRing + n % S::kKeySlots * S::kTile, 16));
        const uint32_t to = uniform(tmem + s * 128);
#pragma unroll
        for (uint32_t k = 0; k < DP / 16; ++k) {
          const uint32_t step = (k >> 2) * (S::kHalf >> 4) + (k & 3) * 2;
          warp_mma_f16_ss(to, qd + step, kd + step, kScores, k > 0 ? 1u : 0u);
        }
        warp_commit(&bars.s_full[s]);
      };
      auto weights_wait = [&](uint32_t s, uint32_t half_of) {
        const bool r = wait_all(&bars.p_full[s][half_of], p_at[s]);
        p_at[s] += half_of;
        tc_fence_after();
        return r;
      };
      // the sums of block i, half of its keys as soon as those weights are there
      auto sums = [&](const Segment* g, uint32_t s, uint32_t i, bool first) -> bool {
        const uint32_t vd = uniform(umma_sw128_low(smem_u32(sm) + S::kValueRing + (done + i) % S::kValueSlots * S::kTile, S::kHalf));
        const uint32_t to = uniform(tmem + 256 + s * DP), from = uniform(tmem + s * 128);
        const uint32_t b = g->b0 + i;
        const bool cached = b < g->q.cached_blocks;
        const uint32_t left = uniform((cached ? g->q.ctx : g->q.nodes) - (cached ? b : b - g->q.cached_blocks) * kKeys);
        const uint32_t keep = uniform(first ? 0u : 1u);
#pragma unroll
        for (uint32_t x = 0; x < 2; ++x) {
          if (!weights_wait(s, x)) return false;
#pragma unroll
          for (uint32_t k = x * 4; k < x * 4 + 4; ++k)
            if (k * 16 < left) warp_mma_f16_ts(to, from + k * 8, vd + k * 128, kSums, k > 0 ? 1u : keep);
        }
        return true;
      };
      for (const Segment* g; ok && (g = segment(seg)) != nullptr;) {
        const uint32_t n = g->n;
        if (g->two) {
          if (!(ok = k_wait(done))) break;
          tc_fence_after();
          scores(0, 0, done);
          scores(1, 1, done);
          k_done(done);
          if (seg > 0 && !(ok = wait_all(&bars.o_free, seg - 1))) break;
          if (n == 1) warp_commit(&bars.q_empty);
          // (the blocks of the next turn are waited for before its weights, so that nothing stands between
          // weights that are ready and their MMAs)
          if (!(ok = v_wait(done) && (n == 1 || k_wait(done + 1)))) break;
          for (uint32_t i = 0; i < n; ++i) {
            const uint32_t v = done + i, k = v + 1;
            const bool more = i + 1 < n;
            if (!(ok = sums(g, 0, i, i == 0))) break;
            if (more) scores(0, 0, k);
            else warp_commit(&bars.o_full[0]);
            if (!(ok = sums(g, 1, i, i == 0))) break;
            v_done(v);
            if (!more) {
              warp_commit(&bars.o_full[1]);
              break;
            }
            scores(1, 1, k);
            k_done(k);
            if (i + 2 == n) warp_commit(&bars.q_empty);
            if (!(ok = v_wait(v + 1) && (i + 2 == n || k_wait(k + 1)))) break;
          }
        } else {
          // even blocks are stream 0's, odd ones stream 1's
          if (!(ok = k_wait(done))) break;
          tc_fence_after();
          scores(0, 0, done);
          k_done(done);
          if (n > 1) {
            if (!(ok = k_wait(done + 1))) break;
            tc_fence_after();
            scores(1, 0, done + 1);
            k_done(done + 1);
          }
          if (seg > 0 && !(ok = wait_all(&bars.o_free, seg - 1))) break;
          if (n <= 2) warp_commit(&bars.q_empty);
          for (uint32_t j = 0; j < n; ++j) {
            const uint32_t s = j & 1, v = done + j, k = v + 2;
            const bool more = j + 2 < n;
            if (!(ok = v_wait(v) && (!more || k_wait(k)) && sums(g, s, j, j < 2))) break;
            v_done(v);
            if (more) {
              scores(s, 0, k);
              k_done(k);
              if (j + 3 == n) warp_commit(&bars.q_empty);
            }
          }
          if (ok) {
            warp_commit(&bars.o_full[0]);
            warp_commit(&bars.o_full[1]);
          }
        }
        done += n;
        ++seg;
      }
      if (!ok) {  // MMAs that were issued end before the tensor memory is freed
        warp_commit(&bars.drain);
        mbar_wait(&bars.drain, 0, p.error);
      }
    }
  } else {
    {
      // ---- softmax: stream s, row = tensor-memory lane
      const uint32_t s = warp >> 2, lrow = (warp & 3) * 32 + lane;
      const uint32_t lanes = ((warp & 3) * 32u) << 16;
      const uint32_t sc = tmem + lanes + s * 128, oc = tmem + lanes + 256 + s * DP;
      const float c = p.scale_log2;
      const uint32_t dim = p.c.head_dim;
      uint32_t s_at = 0, seg = 0, joints = 0;
      bool ok = true;
      for (const Segment* g; ok && (g = segment(seg)) != nullptr;) {
        const Request q = g->q;
        const uint32_t rows = q.nodes * p.group, row0 = g->row0, n = g->n, b0 = g->b0;
        const bool two = g->two != 0;
        const uint32_t row = row0 + (two ? s * half : 0u) + lrow;
        const bool live = lrow < half && row < rows;
        const uint32_t node = live ? p.by_group.quotient(row) : 0u;
        const uint32_t mine = two ? n : (n + 1 - s) / 2;
        float m = -INFINITY, l = 0.0f;
        for (uint32_t i = 0; i < mine; ++i) {
          const uint32_t b = b0 + (two ? i : 2 * i + s);
          // which of the block's keys the row sees
          uint32_t sees[4] = {~0u, ~0u, ~0u, ~0u};
          bool all = true;
          if (b >= q.cached_blocks) {
            all = false;
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x) {
              const uint32_t word = (b - q.cached_blocks) * 4 + x;
              sees[x] = live && word * 32 < q.nodes ? node_mask(p, q, node, word) : 0u;
            }
          } else if (b + 1 == q.cached_blocks && q.ctx - b * kKeys < kKeys) {
            all = false;
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x) {
              const int32_t left = static_cast<int32_t>(q.ctx - b * kKeys) - static_cast<int32_t>(x * 32);
              sees[x] = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
            }
          }
          if (!(ok = wait_all(&bars.s_full[s], s_at))) break;
          ++s_at;
          tc_fence_after();
          // Two passes over the scores, 32 columns a piece, in loops that stay short: unrolled over all 128
          // the softmax waits for instructions.  The first pass ends with the first two pieces in registers,
          // where the second begins; the weights of pieces 0, 1 lie over the scores of piece 0, those of
          // 2, 3 over piece 1.
          if (!all) {  // hidden scores become -inf where they lie
#pragma unroll 1
            for (uint32_t x = 0; x < 4; ++x) {
              uint32_t v[32];
              tc_ld_x32(sc + x * 32, v);
              const uint32_t seen = x < 2 ? (x == 0 ? sees[0] : sees[1]) : (x == 2 ? sees[2] : sees[3]);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = (seen >> e & 1u) ? v[e] : 0xFF800000u;
              tc_st_x32(sc + x * 32, v);
            }
            tc_wait_st();
          }
          uint32_t va[32], vb[32];
          float top = -INFINITY;
#pragma unroll 1
          for (uint32_t x = 0; x < 2; ++x) {
            tc_ld_start_x32(sc + (x == 0 ? 64 : 0), va);
            tc_ld_start_x32(sc + (x == 0 ? 96 : 32), vb);
            tc_join(va, vb);
            float t4[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; e += 4)
#pragma unroll
              for (int k = 0; k < 4; ++k) t4[k] = fmaxf(t4[k], fmaxf(__uint_as_float(va[e + k]), __uint_as_float(vb[e + k])));
            top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
          }
          const float tops = fmaf(top, c, -kWeightShift<T>);
          const bool grow = tops > m + kSlack<T> || (m == -INFINITY && tops > m);
          if (ballot(grow) != 0) {
            const float next = grow ? tops : m;
            const float f = grow ? fast_exp2(m - next) : 1.0f;
            l *= f;
            m = next;
            if (i > 0) {  // the sums of the blocks before this one are complete: their MMAs precede this score's
#pragma unroll 1
              for (uint32_t x = 0; x < DP / 16; ++x) {  // few at a time: the scores stay in registers
                uint32_t o[16];
                tc_ld_x16(oc + x * 16, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tc_st_x16(oc + x * 16, o);
              }
            }
          }
          const float use = m == -INFINITY ? 0.0f : m;
          const uint64_t c2 = pack2(c, c), u2 = pack2(-use, -use);
          uint64_t sum2 = pack2(0.0f, 0.0f);
          auto weigh = [&](const uint32_t(&v)[32], uint32_t to) {
            uint32_t w16[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 t = unpack2(fma2(pack2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), c2, u2));
              const float2 y = make_float2(fast_exp2(t.x), fast_exp2(t.y));
              sum2 = add2(sum2, pack2(y.x, y.y));
              w16[e] = Elem<T>::pack(y.x, y.y);
            }
            tc_st_x16(to, w16);
          };
#pragma unroll 1
          for (uint32_t x = 0; x < 2; ++x) {
            weigh(va, sc + x * 32);
            if (x == 0) tc_ld_start_x32(sc + 64, va);
            weigh(vb, sc + x * 32 + 16);
            // half of the weights at a time: the first half's products run under the second's exponentials
            tc_wait_st();
            tc_fence_before();
            arrive_warp(&bars.p_full[s][x]);
            if (x == 0) {
              tc_ld_start_x32(sc + 96, vb);
              tc_join(va, vb);
            }
          }
          const float2 sum = unpack2(sum2);
          l += sum.x + sum.y;
        }
        if (!ok) break;
        // ---- the segment's end
        if (!(ok = wait_all(&bars.o_full[s], seg))) break;
        tc_fence_after();
        float f0 = 1.0f, f1 = 0.0f;  // factors of the two streams' sums (two: of this stream's own)
        uint32_t x0 = 0, x1 = DP / 32;
        const bool pair = !two && n > 1;
        if (!two) {
          stats[s * 128 + lrow] = make_float2(m, l);
          arrive_warp(&bars.joint);
          if (!(ok = wait_all(&bars.joint, joints))) break;
          ++joints;
          const float2 a = stats[lrow], d = stats[128 + lrow];
          m = fmaxf(a.x, d.x);
          const float use = m == -INFINITY ? 0.0f : m;
          f0 = fast_exp2(a.x - use);
          f1 = fast_exp2(d.x - use);
          l = f0 * a.y + f1 * d.y;
          x0 = s * (DP / 64);  // each warpgroup writes half of the columns
          x1 = x0 + DP / 64;
        }
        const bool complete = b0 == 0 && n == q.blocks;
        const uint32_t head = g->head, h = head * p.group + row - node * p.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* out = static_cast<T*>(p.a.out) + (q.start + node) * p.a.out_token_stride + h * p.a.out_head_stride;
        float* keep = part_sums(p, blockIdx.x, b0 == 0 ? 1u : 0u) + (row - row0) * 4;
        const uint32_t base = tmem + lanes + 256 + (two ? s * DP : 0u);
        const volatile uint32_t* broken = bars.broken[seg & 7];
        uint32_t any = 0;
        if (b0 + n > q.cached_blocks)
          for (uint32_t x = 0; x < (q.nodes + 31) / 32; ++x) any |= broken[x];
#pragma unroll 1
        for (uint32_t x = x0; x < x1; ++x) {
          uint32_t v[32];
          tc_ld_x32(base + x * 32, v);
          float o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = f0 * __uint_as_float(v[e]);
          if (pair) {
            tc_ld_x32(base + DP + x * 32, v);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] += f1 * __uint_as_float(v[e]);
          }
          if (any != 0 && live) {
            for (uint32_t j = 0; j < q.nodes; ++j) {
              const uint32_t b = q.cached_blocks + j / kKeys;
              if (b < b0 || b >= b0 + n || !(broken[j >> 5] >> (j & 31) & 1u)) continue;
              if (!(node_mask(p, q, node, j >> 5) >> (j & 31) & 1u)) continue;
              const T* src = static_cast<const T*>(p.a.v) + (q.start + j) * p.a.kv_token_stride + head * p.a.kv_head_stride;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float add = x * 32 + e < dim ? Elem<T>::to_float(src[x * 32 + e]) : 0.0f;
                if (!(fabsf(add) < INFINITY)) o[e] += add;  // weights are positive
              }
            }
          }
          if (live) {
            if (complete) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint4 r;
                r.x = l == 0.0f ? 0u : Elem<T>::pack(o[e] * inv, o[e + 1] * inv);
                r.y = l == 0.0f ? 0u : Elem<T>::pack(o[e + 2] * inv, o[e + 3] * inv);
                r.z = l == 0.0f ? 0u : Elem<T>::pack(o[e + 4] * inv, o[e + 5] * inv);
                r.w = l == 0.0f ? 0u : Elem<T>::pack(o[e + 6] * inv, o[e + 7] * inv);
                if (x * 32 + e < dim) *reinterpret_cast<uint4*>(out + x * 32 + e) = r;
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(keep + (x * 8 + e / 4) * p.rows * 4) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        }
        if (live && (two || s == 0)) {
          if (!complete) part_stats(p, blockIdx.x, b0 == 0 ? 1u : 0u)[row - row0] = make_float2(m, l);
          else if (p.a.lse != nullptr)
            p.a.lse[static_cast<uint64_t>(q.start + node) * p.a.q_heads + h] =
                l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        }
        tc_fence_before();
        arrive_warp(&bars.o_free);
        ++seg;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void* at = nullptr;
    cudaDriverEntryPointQueryResult found{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return static_cast<EncodeTiled>(nullptr);
    }
    return reinterpret_cast<EncodeTiled>(at);
  }();
  return f;
}

// A map of boxes of 64 columns; dims, box: the dimensions after the columns.  false: no such map.
bool encode_map(CUtensorMap* map, const AttnParams& p, const void* base, uint32_t rank, const uint64_t* dims,
                const uint64_t* strides, const uint32_t* box) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  cuuint64_t size[4] = {p.c.head_dim}, step[3];
  cuuint32_t boxes[4] = {64}, ones[4] = {1, 1, 1, 1};
  for (uint32_t i = 0; i + 1 < rank; ++i) {
    size[i + 1] = dims[i];
    step[i] = dims[i] > 1 ? strides[i] * 2 : 16;  // the stride of a dimension of one element is never used
    boxes[i + 1] = box[i];
    if (step[i] == 0 || step[i] % 16 != 0 || step[i] >= (1ull << 40)) return false;
  }
  return encode(map, p.c.dtype == HQB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                const_cast<void*>(base), size, step, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
cudaError_t launch(const AttnParams& p, const Maps& maps, cudaStream_t st) {
  static DeviceOnce once;
  constexpr uint32_t smem = TmemShape<DP>::kBytes;
  static_assert(smem <= 232448, "one CTA's shared memory");
  const cudaError_t e = allow_dynamic_smem(once, reinterpret_cast<const void*>(attention_tmem_kernel<T, DP>), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(attention_tmem_kernel<T, DP>, dim3(p.grid), kTmemThreads, smem, 1, st, p, maps);
}

}  // namespace

template <typename T>
cudaError_t launch_attention_tmem(const AttnParams& p, cudaStream_t st) {
  Maps m{};
  const uint64_t q_dims[2] = {p.a.q_heads, p.a.tokens}, q_strides[2] = {p.a.q_head_stride, p.a.q_token_stride};
  const uint64_t n_dims[2] = {p.c.kv_heads, p.a.tokens}, n_strides[2] = {p.a.kv_head_stride, p.a.kv_token_stride};
  const uint32_t q_box[2] = {p.group, kRows / p.group}, n_box[2] = {1, kKeys};
  if (!encode_map(&m.q, p, p.a.q, 3, q_dims, q_strides, q_box) || !encode_map(&m.k, p, p.a.k, 3, n_dims, n_strides, n_box) ||
      !encode_map(&m.v, p, p.a.v, 3, n_dims, n_strides, n_box))
    return cudaErrorNotSupported;
  // the largest power of two that divides the page size; the swizzle repeats every 8 rows, so
  // smaller pieces of a page come by plain copies
  uint32_t rows = p.c.page_size & (~p.c.page_size + 1);
  rows = rows > kKeys ? kKeys : rows;
  const uint64_t c_dims[3] = {p.c.kv_heads, p.c.page_size, p.c.num_pages};
  const uint64_t c_strides[3] = {p.c.head_stride, p.c.token_stride, p.c.page_stride};
  const uint32_t c_box[3] = {1, rows, 1};
  if (rows >= 8 && encode_map(&m.ck, p, p.c.k, 4, c_dims, c_strides, c_box) &&
      encode_map(&m.cv, p, p.c.v, 4, c_dims, c_strides, c_box))
    m.box_rows = rows;
  return p.dim_pad == 64 ? launch<T, 64>(p, m, st) : launch<T, 128>(p, m, st);
}
template cudaError_t launch_attention_tmem<__half>(const AttnParams&, cudaStream_t);
template cudaError_t launch_attention_tmem<__nv_bfloat16>(const AttnParams&, cudaStream_t);

}  // namespace hqb
