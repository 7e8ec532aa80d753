// Attention of drafted trees over a paged cache on the tcgen05 tensor cores: tiles of up to 256
// query rows of one (request, key head) against blocks of 128 keys (see hqb_attention.cuh for the
// division of the work).
#include <cuda_runtime.h>

#include "hqb_attention.cuh"
#include "hqb_internal.h"

namespace hqb {
namespace {

constexpr uint32_t kKeys = 128;      // keys of a block
constexpr uint32_t kRows = 128;      // rows of one score tile (tensor-memory lanes)
constexpr uint32_t kStreams = 2;     // score tiles in flight, one per softmax warpgroup
constexpr uint32_t kLoaders = 64;
constexpr uint32_t kMmaWarp = 10;
constexpr uint32_t kTmemThreads = 384;  // 8 softmax warps, 2 loaders, the MMA issuer, one idle: 168 registers a thread
constexpr float kSlack = 8.0f;       // log2 of how far the maximum may grow before sums are rescaled

template <int DP>
struct TmemShape {
  static constexpr uint32_t kQTile = kRows * DP * 2;            // one score tile's queries
  static constexpr uint32_t kSlot = kKeys * DP * 2;             // one block of keys or of values
  static constexpr uint32_t kSlots = DP == 128 ? 5 : 8;
  static constexpr uint32_t kRing = kStreams * kQTile;
  static constexpr uint32_t kBars = kRing + kSlots * kSlot;
  static constexpr uint32_t kStats = kBars + 256;
  static constexpr uint32_t kBytes = kStats + 256 * 8;
  static constexpr uint32_t kLag = kSlots - 2;                  // slots a loader thread has in flight
};

struct Bars {
  uint64_t kv_full[8], kv_empty[8];
  uint64_t q_full, q_empty, s_full[2], p_full[2], o_full[2], o_free, joint, drain;
  uint32_t tmem, abort;
  uint32_t broken[8][8];  // by segment: drafted nodes with an infinity or NaN among their values
};
static_assert(sizeof(Bars) <= 512, "");

// Mathematics: the one-pass softmax of attention_rows_kernel.  A running reference m stands in
// for the maximum: it follows the maximum only when that has grown by more than 8 in the
// exponent, so weights stay below 2^8 and the sums in tensor memory are rarely rescaled; the
// result is the same sum up to rounding.
// Roles: 4 + 4 warps take the scores of two streams out of tensor memory (a thread a row: no
// shuffles), turn them into weights and put those back, packed in 16 bits over the scores, as
// the A operand of weights x values; 4 warps copy keys, values and queries into 128-byte-swizzled
// shared memory through the page table; one thread issues the MMAs.  A tile of more than 128 rows
// has its two halves as streams, over the same keys (each block is loaded once for 256 rows); a
// smaller tile has the even and the odd blocks as streams, joined at the end, so that the scores of
// one stream are computed while the other's weights are.
// Tensor memory: scores 2 x 128 columns, sums 2 x DP columns.  Shared memory at DP 128: queries
// 64 KB, a ring of five 32 KB blocks.
template <typename T, int DP>
__global__ void __launch_bounds__(kTmemThreads, 1) attention_tmem_kernel(const __grid_constant__ AttnParams p) {
  using S = TmemShape<DP>;
  extern __shared__ __align__(1024) uint8_t sm[];
  Bars& bars = *reinterpret_cast<Bars*>(sm + S::kBars);
  float2* stats = reinterpret_cast<float2*>(sm + S::kStats + 256);
  volatile uint32_t* abort = &bars.abort;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t bad = 0;
  griddep_launch_dependents();
  if ((smem_u32(sm) & 1023u) != 0) {  // the swizzle goes by address bits
    if (tid == 0) atomicOr(p.error, HQB_DEVERR_LAUNCH);
    return;
  }
  if (tid < 64) bars.broken[tid >> 3][tid & 7] = 0;
  if (tid == 0) {
    for (uint32_t i = 0; i < S::kSlots; ++i) {
      mbar_init(&bars.kv_full[i], kLoaders);
      mbar_init(&bars.kv_empty[i], 1);
    }
    mbar_init(&bars.q_full, kLoaders);
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.o_full[i], 1);
    }
    mbar_init(&bars.o_free, 256);
    mbar_init(&bars.joint, 256);
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
  const uint32_t tmem = bars.tmem;
  griddep_wait();
  // a wait that runs out ends every role's loop; nothing is left in flight but this CTA's copies
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (*abort) return false;
    if (mbar_wait(bar, parity & 1u, p.error)) return true;
    *abort = 1u;
    return false;
  };
  // the same for a whole warp, whose lanes must go on or stop together
  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };
  Walk w;
  if (w.begin(p, blockIdx.x, bad)) {
    if (warp == 8 || warp == 9) {
      // ---- loaders: a warp has two groups of 32 rows of a block; a lane looks up a key of each, and
      // 8 or 16 lanes copy a row
      const uint32_t lw = warp - 8;
      constexpr uint32_t kPieces = DP / 8;  // 16-byte pieces of a row
      const uint32_t dim = p.c.head_dim;
      uint32_t issued = 0, done = 0, seg = 0;
      bool ok = true;
      auto arrive_one = [&]() {
        fence_proxy_async_smem();
        mbar_arrive(&bars.kv_full[done % S::kSlots]);
        ++done;
      };
      // copies rows r0 .. r0 + 31 from the lanes' element offsets `where`
      auto rows_to = [&](uint32_t dst, uint32_t half_bytes, uint32_t r0, const T* src, uint64_t where, bool real) {
        const uint32_t live = ballot(real);
#pragma unroll
        for (uint32_t x = 0; x < kPieces; ++x) {
          const uint32_t at = x * 32 + lane, j = at / kPieces, c = at % kPieces, r = r0 + j;
          const uint64_t row = __shfl_sync(0xffffffffu, where, j);
          const bool copy = (live >> j & 1u) != 0 && c * 8 < dim;
          cp_async16(dst + (c >> 3) * half_bytes + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + (copy ? row + c * 8 : 0),
                     copy ? 16u : 0u);
        }
      };
      while (ok && w.left != 0) {
        w.open(p);
        const Request q = w.q;
        const uint32_t rows = q.nodes * p.group, row0 = w.tile * p.rows, n = w.b1 - w.b0;
        const bool two = rows - row0 > kRows;
        const int32_t* table = p.a.tables + static_cast<uint64_t>(w.r) * p.a.table_stride;
        uint32_t* broken = bars.broken[seg & 7];
        auto load = [&](uint32_t b, bool values) {
          const uint32_t slot = issued % S::kSlots;
          if (issued >= S::kSlots) ok = ok && wait_all(&bars.kv_empty[slot], issued / S::kSlots - 1);
          if (!ok) return;
          const uint32_t dst = smem_u32(sm + S::kRing + slot * S::kSlot);
          constexpr uint32_t kHalf = kKeys * 128;
          for (uint32_t r0 = lw * 64; r0 < lw * 64 + 64; r0 += 32) {
            if (b < q.cached_blocks) {
              const uint32_t key = b * kKeys + r0 + lane;
              const bool real = key < q.ctx;
              const uint64_t where = real ? key_offset(p, table, key, w.head, bad) : 0;
              rows_to(dst, kHalf, r0, static_cast<const T*>(values ? p.c.v : p.c.k), where, real);
            } else {
              const uint32_t node = (b - q.cached_blocks) * kKeys + r0 + lane;
              const bool real = node < q.nodes;
              const uint64_t where = real ? (q.start + node) * p.a.kv_token_stride + w.head * p.a.kv_head_stride : 0;
              if (!values) {
                rows_to(dst, kHalf, r0, static_cast<const T*>(p.a.k), where, real);
              } else {
                // through registers: a weight of zero must cancel a hidden node's values whatever they
                // are, so infinities and NaN become zeros here, and the rows that see the node get
                // them at the end
                const uint32_t live = ballot(real);
  #pragma unroll 4
                for (uint32_t x = 0; x < kPieces; ++x) {
                  const uint32_t at = x * 32 + lane, j = at / kPieces, c = at % kPieces, r = r0 + j;
                  const uint64_t row = __shfl_sync(0xffffffffu, where, j);
                  uint4 v = make_uint4(0, 0, 0, 0);
                  if ((live >> j & 1u) != 0 && c * 8 < dim)
                    v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.a.v) + row + c * 8));
                  uint32_t e[4] = {v.x, v.y, v.z, v.w};
                  bool found = false;
  #pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    constexpr uint32_t kMask = Elem<T>::kExpMask;
                    if ((e[i] & kMask) == kMask) e[i] &= 0xFFFF0000u, found = true;
                    if ((e[i] >> 16 & kMask) == kMask) e[i] &= 0x0000FFFFu, found = true;
                  }
                  if (found) atomicOr(&broken[((b - q.cached_blocks) * kKeys + r) >> 5], 1u << (r & 31));
                  *reinterpret_cast<uint4*>(sm + S::kRing + slot * S::kSlot + (c >> 3) * kHalf + r * 128 +
                                            (((c & 7) ^ (r & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
                }
              }
            }
          }
          cp_async_commit();
          ++issued;
          if (issued - done > S::kLag) {
            cp_async_wait<S::kLag>();
            arrive_one();
          }
        };
        // the first keys, then the queries (the last segment's must have been read), then the rest in
        // the order in which the MMAs take them
        load(w.b0, false);
        if (seg > 0) ok = ok && wait_all(&bars.q_empty, seg - 1);
        if (!ok) break;
        // past here the epilogue of segment seg - 3 is over: the flags of segment seg - 4 are free
        if (lw == 0 && lane < 8) bars.broken[(seg + 4) & 7][lane] = 0;
        for (uint32_t r0 = lw * 64; r0 < (two ? 2 * kRows : kRows); r0 += (r0 & 32) ? 96 : 32) {
          const uint32_t row = row0 + r0 + lane;
          const bool real = row < rows;
          const uint32_t node = real ? row / p.group : 0u;
          const uint64_t where = real ? (q.start + node) * p.a.q_token_stride +
                                            static_cast<uint64_t>(w.head * p.group + row - node * p.group) * p.a.q_head_stride
                                      : 0;
          rows_to(smem_u32(sm + (r0 / kRows) * S::kQTile), kRows * 128, r0 % kRows, static_cast<const T*>(p.a.q), where, real);
        }
        cp_async_commit();
        cp_async_wait<0>();
        while (done < issued) arrive_one();
        fence_proxy_async_smem();
        mbar_arrive(&bars.q_full);
        if (two) {
          for (uint32_t i = 0; ok && i < n; ++i) {
            if (i > 0) load(w.b0 + i, false);
            load(w.b0 + i, true);
          }
        } else {
          if (n > 1) load(w.b0 + 1, false);
          for (uint32_t i = 0; ok && i < n; ++i) {
            load(w.b0 + i, true);
            if (i + 2 < n) load(w.b0 + i + 2, false);
          }
        }
        // the tail of the segment must not wait for the next segment's loads
        cp_async_wait<0>();
        while (done < issued) arrive_one();
        ++seg;
        w.advance(p, bad);
      }
      cp_async_wait<0>();
    } else if (warp == kMmaWarp) {
      // ---- MMA issuer
      if (lane == 0) {
        constexpr uint32_t kType = sizeof(T) == 2 && Elem<T>::kExpMask == 0x7F80u ? 1u : 0u;  // BF16 : FP16
        constexpr uint32_t kBase = (1u << 4) | (kType << 7) | (kType << 10) | ((kRows >> 4) << 24);
        constexpr uint32_t kScores = kBase | ((kKeys >> 3) << 17);
        constexpr uint32_t kSums = kBase | (1u << 16) | ((DP >> 3) << 17);  // B (values) MN-major
        uint32_t slot_at = 0, seg = 0, p_at[2] = {0, 0};
        bool ok = true;
        auto slot_wait = [&](uint32_t n) { return wait(&bars.kv_full[n % S::kSlots], n / S::kSlots); };
        auto slot_addr = [&](uint32_t n) { return smem_u32(sm + S::kRing + (n % S::kSlots) * S::kSlot); };
        auto scores = [&](uint32_t s, uint32_t tile, uint32_t slot) {
          const uint32_t qa = smem_u32(sm + tile * S::kQTile), ka = slot_addr(slot);
#pragma unroll
          for (uint32_t k = 0; k < DP / 16; ++k)
            tc_mma_f16_ss(tmem + s * 128, umma_desc_sw128(qa + (k >> 2) * (kRows * 128) + (k & 3) * 32, 16),
                          umma_desc_sw128(ka + (k >> 2) * (kKeys * 128) + (k & 3) * 32, 16), kScores, k > 0 ? 1u : 0u);
          tc_commit(&bars.s_full[s]);
        };
        auto sums = [&](uint32_t s, uint32_t slot, bool first) {
          const uint32_t va = slot_addr(slot);
#pragma unroll
          for (uint32_t k = 0; k < kKeys / 16; ++k)
            tc_mma_f16_ts(tmem + 256 + s * DP, tmem + s * 128 + k * 8, umma_desc_sw128(va + k * 2048, kKeys * 128), kSums,
                          k > 0 || !first ? 1u : 0u);
        };
        auto weights_wait = [&](uint32_t s) {
          const bool r = wait(&bars.p_full[s], p_at[s]);
          ++p_at[s];
          tc_fence_after();
          return r;
        };
        while (ok && w.left != 0) {
          w.open(p);
          const uint32_t n = w.b1 - w.b0;
          const bool two = w.q.nodes * p.group - w.tile * p.rows > kRows;
          ok = wait(&bars.q_full, seg);
          if (!ok) break;
          if (two) {
            // slots: K0 V0 K1 V1 ...
            if (!(ok = slot_wait(slot_at))) break;
            tc_fence_after();
            scores(0, 0, slot_at);
            scores(1, 1, slot_at);
            tc_commit(&bars.kv_empty[slot_at % S::kSlots]);
            if (n == 1) tc_commit(&bars.q_empty);
            if (seg > 0 && !(ok = wait(&bars.o_free, seg - 1))) break;
            for (uint32_t i = 0; i < n; ++i) {
              const uint32_t v = slot_at + 2 * i + 1, k = v + 1;
              const bool more = i + 1 < n;
              ok = slot_wait(v) && weights_wait(0);
              if (!ok) break;
              sums(0, v, i == 0);
              if (more) {
                if (!(ok = slot_wait(k))) break;
                tc_fence_after();
                scores(0, 0, k);
              } else {
                tc_commit(&bars.o_full[0]);
              }
              if (!(ok = weights_wait(1))) break;
              sums(1, v, i == 0);
              tc_commit(&bars.kv_empty[v % S::kSlots]);
              if (more) {
                scores(1, 1, k);
                tc_commit(&bars.kv_empty[k % S::kSlots]);
                if (i + 2 == n) tc_commit(&bars.q_empty);
              } else {
                tc_commit(&bars.o_full[1]);
              }
            }
          } else {
            // slots: K0 K1 V0 K2 V1 K3 ...
            if (!(ok = slot_wait(slot_at))) break;
            tc_fence_after();
            scores(0, 0, slot_at);
            tc_commit(&bars.kv_empty[slot_at % S::kSlots]);
            uint32_t next = slot_at + 1;
            if (n > 1) {
              if (!(ok = slot_wait(next))) break;
              tc_fence_after();
              scores(1, 0, next);
              tc_commit(&bars.kv_empty[next % S::kSlots]);
              ++next;
            }
            if (n <= 2) tc_commit(&bars.q_empty);
            if (seg > 0 && !(ok = wait(&bars.o_free, seg - 1))) break;
            for (uint32_t j = 0; j < n; ++j) {
              const uint32_t s = j & 1, v = next++;
              ok = slot_wait(v) && weights_wait(s);
              if (!ok) break;
              sums(s, v, j < 2);
              tc_commit(&bars.kv_empty[v % S::kSlots]);
              if (j + 2 < n) {
                const uint32_t k = next++;
                if (!(ok = slot_wait(k))) break;
                tc_fence_after();
                scores(s, 0, k);
                tc_commit(&bars.kv_empty[k % S::kSlots]);
                if (j + 3 == n) tc_commit(&bars.q_empty);
              }
            }
            if (ok) {
              tc_commit(&bars.o_full[0]);
              tc_commit(&bars.o_full[1]);
            }
          }
          slot_at += 2 * n;
          ++seg;
          w.advance(p, bad);
        }
        if (!ok) {  // MMAs that were issued end before the tensor memory is freed
          tc_commit(&bars.drain);
          mbar_wait(&bars.drain, 0, p.error);
        }
      }
    } else if (warp < 8) {
      // ---- softmax: stream s, row = tensor-memory lane
      const uint32_t s = warp >> 2, lrow = (warp & 3) * 32 + lane;
      const uint32_t lanes = ((warp & 3) * 32u) << 16;
      const uint32_t sc = tmem + lanes + s * 128, oc = tmem + lanes + 256 + s * DP;
      const float c = p.scale_log2;
      const uint32_t dim = p.c.head_dim;
      uint32_t s_at = 0, seg = 0, joints = 0;
      bool ok = true;
      while (ok && w.left != 0) {
        w.open(p);
        const Request q = w.q;
        const uint32_t rows = q.nodes * p.group, row0 = w.tile * p.rows, n = w.b1 - w.b0;
        const bool two = rows - row0 > kRows;
        const uint32_t row = row0 + (two ? s * kRows : 0u) + lrow;
        const bool live = row < rows;
        const uint32_t node = live ? row / p.group : 0u;
        const uint32_t mine = two ? n : (n + 1 - s) / 2;
        float m = -INFINITY, l = 0.0f;
        for (uint32_t i = 0; i < mine; ++i) {
          const uint32_t b = w.b0 + (two ? i : 2 * i + s);
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
          float top = -INFINITY;
#pragma unroll
          for (uint32_t x = 0; x < 4; ++x) {
            uint32_t v[32];
            tc_ld_x32(sc + x * 32, v);
            float t0 = -INFINITY, t1 = -INFINITY;
            if (all) {
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                t0 = fmaxf(t0, fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
                t1 = fmaxf(t1, fmaxf(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])));
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) t0 = fmaxf(t0, (sees[x] >> e & 1u) ? __uint_as_float(v[e]) : -INFINITY);
            }
            top = fmaxf(top, fmaxf(t0, t1));
          }
          const float tops = top * c;
          const bool grow = tops > m + kSlack || (m == -INFINITY && tops > m);
          if (ballot(grow) != 0) {
            const float next = grow ? tops : m;
            const float f = grow ? fast_exp2(m - next) : 1.0f;
            l *= f;
            m = next;
            if (i > 0) {  // the sums of the blocks before this one are complete: their MMAs precede this score's
#pragma unroll
              for (uint32_t x = 0; x < DP / 32; ++x) {
                uint32_t v[32];
                tc_ld_x32(oc + x * 32, v);
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                tc_st_x32(oc + x * 32, v);
              }
            }
          }
          const float use = m == -INFINITY ? 0.0f : m;
          const uint64_t c2 = pack2(c, c), u2 = pack2(-use, -use);
          uint64_t sum2 = pack2(0.0f, 0.0f);
#pragma unroll
          for (uint32_t x = 0; x < 4; ++x) {
            uint32_t v[32], w16[16];
            tc_ld_x32(sc + x * 32, v);
            if (!all) {
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = (sees[x] >> e & 1u) ? v[e] : 0xFF800000u;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 t = unpack2(fma2(pack2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), c2, u2));
              const float a = fast_exp2(t.x), d = fast_exp2(t.y);
              sum2 = add2(sum2, pack2(a, d));
              w16[e] = Elem<T>::pack(a, d);
            }
            tc_st_x16(sc + x * 16, w16);
          }
          const float2 sum = unpack2(sum2);
          l += sum.x + sum.y;
          tc_wait_st();
          tc_fence_before();
          mbar_arrive(&bars.p_full[s]);
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
          mbar_arrive(&bars.joint);
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
        const bool complete = w.complete();
        const uint32_t h = w.head * p.group + row - node * p.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* out = static_cast<T*>(p.a.out) + (q.start + node) * p.a.out_token_stride + h * p.a.out_head_stride;
        float* keep = part_row(p, blockIdx.x, w.b0 == 0 ? 1u : 0u, row - row0);
        const uint32_t base = tmem + lanes + 256 + (two ? s * DP : 0u);
        const volatile uint32_t* broken = bars.broken[seg & 7];
        uint32_t any = 0;
        if (w.b1 > q.cached_blocks)
          for (uint32_t x = 0; x < (q.nodes + 31) / 32; ++x) any |= broken[x];
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
              if (b < w.b0 || b >= w.b1 || !(broken[j >> 5] >> (j & 31) & 1u)) continue;
              if (!(node_mask(p, q, node, j >> 5) >> (j & 31) & 1u)) continue;
              const T* src = static_cast<const T*>(p.a.v) + (q.start + j) * p.a.kv_token_stride + w.head * p.a.kv_head_stride;
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
              for (int e = 0; e < 32; e += 2) *reinterpret_cast<float2*>(keep + x * 32 + e) = make_float2(o[e], o[e + 1]);
            }
          }
        }
        if (live && (two || s == 0)) {
          if (!complete) *reinterpret_cast<float2*>(keep + DP) = make_float2(m, l);
          else if (p.a.lse != nullptr)
            p.a.lse[static_cast<uint64_t>(q.start + node) * p.a.q_heads + h] =
                l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        }
        tc_fence_before();
        mbar_arrive(&bars.o_free);
        ++seg;
        w.advance(p, bad);
      }
      if (bad != 0) atomicOr(p.error, static_cast<int>(bad));
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <typename T, int DP>
cudaError_t launch(const AttnParams& p, cudaStream_t st) {
  static DeviceOnce once;
  constexpr uint32_t smem = TmemShape<DP>::kBytes + 512;
  static_assert(smem <= 232448, "one CTA's shared memory");
  const cudaError_t e = allow_dynamic_smem(once, reinterpret_cast<const void*>(attention_tmem_kernel<T, DP>), smem);
  if (e != cudaSuccess) return e;
  attention_tmem_kernel<T, DP><<<p.grid, kTmemThreads, smem, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

template <typename T>
cudaError_t launch_attention_tmem(const AttnParams& p, cudaStream_t st) {
  return p.dim_pad == 64 ? launch<T, 64>(p, st) : launch<T, 128>(p, st);
}
template cudaError_t launch_attention_tmem<__half>(const AttnParams&, cudaStream_t);
template cudaError_t launch_attention_tmem<__nv_bfloat16>(const AttnParams&, cudaStream_t);

}  // namespace hqb
