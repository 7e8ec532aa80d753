// Attention of drafted trees over a paged cache (hqb_tree_attention).
//   attention_rows_kernel  16 query rows a tile on mma.sync: single tokens, small trees, and every
//                          shape that the tensor-memory kernel does not take
//   attention_tmem_kernel  256 query rows a tile on tcgen05 (hqb_attention_tmem.cu)
//   attention_join_kernel  joins the partial results of items that span CTAs
#include <cuda_runtime.h>

#include "hqb_attention.cuh"
#include "hqb_internal.h"

namespace hqb {
namespace {

constexpr uint32_t kKeyBlock = 64;
constexpr uint32_t kChunk = 16;  // keys a warp takes at once

// A CTA's shared memory: the warps' rings of kStages chunks, over which their sums are joined at an
// item's end.
template <int DP, int kRowsWarps, int kStages>
constexpr uint32_t kRowsSmem = kRowsWarps * kStages * 2 * kChunk * DP * 2;

// Mathematics: the softmax over the keys in one pass.  A warp keeps, per row, a reference m (the
// running maximum of t = scale*log2(e) * q.k, less kWeightShift), the sum l of 2^(t - m) and the sums O
// of 2^(t - m) v; a larger reference m' rescales l and O by 2^(m - m').  Warps, and CTAs, that saw different keys
// are joined the same way.
// Split: the warps of a CTA take the segment's 16-key chunks in turn, each with its own
// ring of asynchronous copies, so the loop has no CTA barrier and keeps 2 chunks (16 KB at 128
// dimensions) a warp in flight; the warps are joined once per segment.  Rows: the group's heads
// of all nodes share the keys, so a key is read once per 16 rows.
// Warps: four, two CTAs an SM, so that one CTA's ends of segments lie under the other's copies.  Where
// items are not cut (up to 512 keys): eight for few items, whose rings then hold two chunks each in flight
// (256 keys a CTA; a third starts behind the first wait); four
// or two for more items than SMs, with twelve warps an SM in CTAs of their own.
// Bound by HBM at 16 rows: 32 MMAs a chunk are about 310 cycles of one of the four tensor pipes
// a chunk against 1400 cycles an SM needs to fetch four chunks; by latency at short contexts (launch, lengths,
// page table, keys and the join of the warps follow one another).
// Measured, B200: 16 tokens over contexts of up to 8192, 64 heads over 8 of 128, BF16, 68 us (5.3 TB/s,
// of 6.55 TB/s that a copy reaches), with the join; one token over 301 keys, 32 heads of 128, FP16, 9.0 us.
template <typename T, int DP, bool VEC, int kRowsWarps, int kStages>
__global__ void __launch_bounds__(kRowsWarps * 32, kStages == 2 ? 12 / kRowsWarps : 1) attention_rows_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ __align__(128) uint8_t sm[];
  constexpr uint32_t kRowBytes = DP * 2, kTileBytes = kChunk * kRowBytes, kStageBytes = 2 * kTileBytes;
  constexpr uint32_t kPieces = DP / 8;  // 16-byte pieces of a row
  constexpr int kSteps = DP / 16;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3;
  uint8_t* ring = sm + warp * kStages * kStageBytes;
  const uint32_t ring_a = smem_u32(ring);
  uint32_t bad = 0;
  griddep_launch_dependents();
  griddep_wait();
  Walk w;
  const bool work = w.begin(p, blockIdx.x, bad);
  if (threadIdx.x == 0 && !p.whole) note_split(p, w, blockIdx.x, work, bad);
  if (!work) {
    if (bad != 0 && blockIdx.x == 0) atomicOr(p.error, static_cast<int>(bad));  // there may be no work at all
    return;
  }
  const uint32_t dim = p.c.head_dim;
  const T* const kc = static_cast<const T*>(p.c.k);
  const T* const vc = static_cast<const T*>(p.c.v);
  const T* const kn = static_cast<const T*>(p.a.k);
  const T* const vn = static_cast<const T*>(p.a.v);

  while (w.left != 0) {
    w.open(p);
    const Request q = w.q;
    const uint32_t rows = q.nodes * p.group, row0 = w.tile * 16;
    const int32_t* table = p.a.tables + static_cast<uint64_t>(w.r) * p.a.table_stride;
    // this lane's two rows
    uint32_t node[2];
    bool live[2];
    uint32_t qf[kSteps][4];
    {
      const T* src[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t row = row0 + g + 8 * e;
        live[e] = row < rows;
        node[e] = live[e] ? p.by_group.quotient(row) : 0u;
        const uint32_t h = w.head * p.group + (live[e] ? row - node[e] * p.group : 0u);
        src[e] = static_cast<const T*>(p.a.q) + (q.start + node[e]) * p.a.q_token_stride + h * p.a.q_head_stride;
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t d = s * 16 + (e >> 1) * 8 + qd * 2;
          const T* x = src[e & 1] + d;
          uint32_t v = 0;
          if (VEC) {
            if (live[e & 1] && d < dim) v = *reinterpret_cast<const uint32_t*>(x);
          } else {
            uint32_t lo = 0, hi = 0;
            if (live[e & 1] && d < dim) lo = *reinterpret_cast<const uint16_t*>(x);
            if (live[e & 1] && d + 1 < dim) hi = *reinterpret_cast<const uint16_t*>(x + 1);
            v = lo | hi << 16;
          }
          qf[s][e] = v;
        }
    }
    float acc[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;

    // chunk index of the segment -> its first key among the cached ones, or among the nodes
    const uint32_t chunks = (w.b1 - w.b0) * (kKeyBlock / kChunk);
    auto place = [&](uint32_t i, uint32_t& key, uint32_t& valid) -> bool {  // true: drafted
      const uint32_t b = w.b0 + i / (kKeyBlock / kChunk), off = (i % (kKeyBlock / kChunk)) * kChunk;
      const bool drafted = b >= q.cached_blocks;
      key = (drafted ? b - q.cached_blocks : b) * kKeyBlock + off;
      const uint32_t most = drafted ? q.nodes : q.ctx;
      valid = most > key ? min(kChunk, most - key) : 0u;
      return drafted;
    };
    // lane l < 16 looks up key l of a chunk: its row in the cache or in k, v
    auto look_up = [&](uint32_t i) -> uint64_t {
      uint32_t key, valid;
      const bool drafted = place(i, key, valid);
      const uint32_t j = lane & 15;
      if (j >= valid) return 0;
      if (drafted) return (q.start + key + j) * p.a.kv_token_stride + w.head * p.a.kv_head_stride;
      return key_offset(p, table, key + j, w.head, bad);
    };
    auto load = [&](uint32_t i, uint32_t stage, uint64_t where) {
      uint32_t key, valid;
      const bool drafted = place(i, key, valid);
      if (valid == 0) return;  // not read either
      const T* ks = drafted ? kn : kc;
      const T* vs = drafted ? vn : vc;
      const uint32_t base = ring_a + stage * kStageBytes;
      if (VEC) {
#pragma unroll
        for (uint32_t x = 0; x < kChunk * kPieces / 32; ++x) {
          const uint32_t at = x * 32 + lane, j = at / kPieces, c = at % kPieces;
          const uint64_t row = __shfl_sync(0xffffffffu, where, j);
          const bool real = j < valid && c * 8 < dim;
          const uint64_t off = real ? row + c * 8 : 0;
          const uint32_t dst = base + j * kRowBytes + ((c ^ (j & 7)) << 4);
          cp_async16(dst, ks + off, real ? 16u : 0u);
          cp_async16(dst + kTileBytes, vs + off, real ? 16u : 0u);
        }
      } else {
        for (uint32_t at = lane; at < kChunk * DP; at += 32) {
          const uint32_t j = at / DP, d = at % DP;
          const uint64_t row = __shfl_sync(0xffffffffu, where, j);
          const bool real = j < valid && d < dim;
          uint8_t* dst = ring + stage * kStageBytes + j * kRowBytes + (((d >> 3) ^ (j & 7)) << 4) + (d & 7) * 2;
          const uint16_t zero = 0;
          *reinterpret_cast<uint16_t*>(dst) = real ? *reinterpret_cast<const uint16_t*>(ks + row + d) : zero;
          *reinterpret_cast<uint16_t*>(dst + kTileBytes) = real ? *reinterpret_cast<const uint16_t*>(vs + row + d) : zero;
        }
      }
    };

    // ring prologue: two chunks in flight, the third's lookup under way
#pragma unroll
    for (uint32_t s = 0; s < kStages - 1; ++s) {
      const uint32_t i = warp + s * kRowsWarps;
      if (i < chunks) load(i, s, look_up(i));
      cp_async_commit();
    }
    uint64_t where_next = 0;
    if (warp + (kStages - 1) * kRowsWarps < chunks) where_next = look_up(warp + (kStages - 1) * kRowsWarps);
    uint32_t stage = 0;
    for (uint32_t i = warp; i < chunks; i += kRowsWarps) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      // refill the stage read in the previous turn
      {
        const uint32_t ahead = i + (kStages - 1) * kRowsWarps;
        const uint32_t to = stage == 0 ? kStages - 1 : stage - 1;
        if (ahead < chunks) load(ahead, to, where_next);
        cp_async_commit();
        if (ahead + kRowsWarps < chunks) where_next = look_up(ahead + kRowsWarps);
      }
      uint32_t key, valid;
      const bool drafted = place(i, key, valid);
      const uint32_t base = ring_a + stage * kStageBytes, vbase = base + kTileBytes;
      const uint32_t here = stage;
      stage = stage + 1 == kStages ? 0 : stage + 1;
      if (valid == 0) continue;  // past the context's or the nodes' end
      // which of the chunk's keys each row sees, a bit a key
      uint32_t sees[2] = {(1u << valid) - 1u, (1u << valid) - 1u};
      uint32_t broken = 0;  // keys with an infinity or NaN among their values
      if (drafted) {
#pragma unroll
        for (int e = 0; e < 2; ++e) sees[e] = live[e] ? (node_mask(p, q, node[e], key >> 5) >> (key & 31)) & 0xFFFFu : 0u;
        // a weight of zero must cancel a hidden key's values whatever they are: rows of values
        // with an infinity or NaN are zeroed here and added below for the rows that see them
        uint8_t* vt = ring + here * kStageBytes + kTileBytes;
        for (uint32_t at = lane; at < kChunk * kPieces; at += 32) {
          const uint4 v = *reinterpret_cast<const uint4*>(vt + at * 16);
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            constexpr uint32_t kMask = Elem<T>::kExpMask;
            if ((x[e] & kMask) == kMask || ((x[e] >> 16) & kMask) == kMask) broken |= 1u << (at / kPieces);
          }
        }
        broken = __reduce_or_sync(0xffffffffu, broken);
        if (broken != 0) {
          for (uint32_t at = lane; at < kChunk * kPieces; at += 32)
            if (broken >> (at / kPieces) & 1u) *reinterpret_cast<uint4*>(vt + at * 16) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
      }
      float s[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
      {
        // matrices: keys 0-7 | k 0-7, keys 0-7 | k 8-15, keys 8-15 | k 0-7, keys 8-15 | k 8-15
        const uint32_t j = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          uint32_t b[4];
          ldmatrix_x4(base + j * kRowBytes + (((st * 2 + half) ^ (j & 7)) << 4), b);
          Elem<T>::mma(s[0], qf[st][0], qf[st][1], qf[st][2], qf[st][3], b[0], b[1]);
          Elem<T>::mma(s[1], qf[st][0], qf[st][1], qf[st][2], qf[st][3], b[2], b[3]);
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bit = n * 8 + qd * 2 + (e & 1);
          s[n][e] = (sees[e >> 1] >> bit & 1u) ? s[n][e] * p.scale_log2 : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
      float use[2];
      bool grew = false;
      float factor[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
        const float next = fmaxf(m[e], top[e] - kWeightShift<T>);
        grew |= next != m[e];
        use[e] = next == -INFINITY ? 0.0f : next;
        factor[e] = fast_exp2(m[e] - use[e]);
        m[e] = next;
      }
      if (ballot(grew) != 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) l[e] *= factor[e];
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] *= factor[e >> 1];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] = fast_exp2(s[n][e] - use[e >> 1]);
          l[e >> 1] += s[n][e];
        }
      // Weights as the A operand of weights x values: the tensor cores multiply 16-bit types at full rate, and the
      // rounding (half a unit of the type a weight, either way) is of the output's own size.  The sum of weights
      // keeps the unrounded ones, since the log of it is an output in FP32.
      const uint32_t a0 = Elem<T>::pack(s[0][0], s[0][1]), a1 = Elem<T>::pack(s[0][2], s[0][3]);
      const uint32_t a2 = Elem<T>::pack(s[1][0], s[1][1]), a3 = Elem<T>::pack(s[1][2], s[1][3]);
      {
        // matrices: keys 0-7 | d 0-7, keys 8-15 | d 0-7, keys 0-7 | d 8-15, keys 8-15 | d 8-15
        const uint32_t j = lane & 15, half = lane >> 4;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          uint32_t b[4];
          ldmatrix_x4_trans(vbase + j * kRowBytes + (((n * 2 + half) ^ (j & 7)) << 4), b);
          Elem<T>::mma(acc[2 * n], a0, a1, a2, a3, b[0], b[1]);
          Elem<T>::mma(acc[2 * n + 1], a0, a1, a2, a3, b[2], b[3]);
        }
      }
      for (uint32_t rest = broken; rest != 0; rest &= rest - 1) {
        const uint32_t j = __ffs(rest) - 1, from = g * 4 + (j & 7) / 2;
        float weight[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x0 = __shfl_sync(0xffffffffu, s[0][2 * e], from), x1 = __shfl_sync(0xffffffffu, s[0][2 * e + 1], from);
          const float x2 = __shfl_sync(0xffffffffu, s[1][2 * e], from), x3 = __shfl_sync(0xffffffffu, s[1][2 * e + 1], from);
          weight[e] = j < 8 ? (j & 1 ? x1 : x0) : (j & 1 ? x3 : x2);
        }
        const T* row = vn + (q.start + key + j) * p.a.kv_token_stride + w.head * p.a.kv_head_stride;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t d = n * 8 + qd * 2 + (e & 1);
            if (d < dim && (sees[e >> 1] >> j & 1u)) {
              const float v = Elem<T>::to_float(row[d]);
              acc[n][e] += fabsf(v) < INFINITY ? weight[e >> 1] * v : v;  // weights are positive
            }
          }
      }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    // join the warps: sums in shared memory over the (drained) rings, [warp][16][DP + 2]
    __syncthreads();
    constexpr uint32_t kPitch = DP + 2;
    static_assert(kRowsWarps * 16 * kPitch * 4 <= kRowsSmem<DP, kRowsWarps, kStages>, "the join area fits the rings");
    float* joint = reinterpret_cast<float*>(sm);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* row = joint + (warp * 16 + g + 8 * e) * kPitch;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
        *reinterpret_cast<float2*>(row + n * 8 + qd * 2) = make_float2(acc[n][2 * e], acc[n][2 * e + 1]);
      if (qd == 0) *reinterpret_cast<float2*>(row + DP) = make_float2(m[e], l[e]);
    }
    __syncthreads();
    {
      constexpr uint32_t kEach = kRowsWarps * 2;  // threads a row
      const uint32_t row = threadIdx.x / kEach, part = threadIdx.x % kEach;
      float mm = -INFINITY, ll = 0.0f, f[kRowsWarps];
#pragma unroll
      for (uint32_t x = 0; x < kRowsWarps; ++x) mm = fmaxf(mm, joint[(x * 16 + row) * kPitch + DP]);
      const float mu = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
      for (uint32_t x = 0; x < kRowsWarps; ++x) {
        f[x] = fast_exp2(joint[(x * 16 + row) * kPitch + DP] - mu);
        ll += f[x] * joint[(x * 16 + row) * kPitch + DP + 1];
      }
      const uint32_t at = row0 + row;
      const bool complete = w.complete();
      if (at < rows) {
        const uint32_t nd = p.by_group.quotient(at), h = w.head * p.group + at - nd * p.group;
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        T* out = static_cast<T*>(p.a.out) + (q.start + nd) * p.a.out_token_stride + h * p.a.out_head_stride;
        float* keep = part_sums(p, blockIdx.x, w.b0 == 0 ? 1u : 0u) + row * 4;
        for (uint32_t d = part * 2; d < DP; d += kEach * 2) {
          float2 o = make_float2(0.0f, 0.0f);
#pragma unroll
          for (uint32_t x = 0; x < kRowsWarps; ++x) {
            const float2 v = *reinterpret_cast<const float2*>(joint + (x * 16 + row) * kPitch + d);
            o.x += f[x] * v.x;
            o.y += f[x] * v.y;
          }
          if (complete) {
            if (VEC) {
              if (d < dim) *reinterpret_cast<uint32_t*>(out + d) = ll == 0.0f ? 0u : Elem<T>::pack(o.x * inv, o.y * inv);
            } else {
              if (d < dim) out[d] = Elem<T>::from_float(ll == 0.0f ? 0.0f : o.x * inv);
              if (d + 1 < dim) out[d + 1] = Elem<T>::from_float(ll == 0.0f ? 0.0f : o.y * inv);
            }
          } else {
            *reinterpret_cast<float2*>(keep + (d >> 2) * p.rows * 4 + (d & 3)) = o;
          }
        }
        if (part == 0) {
          if (!complete) part_stats(p, blockIdx.x, w.b0 == 0 ? 1u : 0u)[row] = make_float2(mm, ll);
          else if (p.a.lse != nullptr)
            p.a.lse[static_cast<uint64_t>(q.start + nd) * p.a.q_heads + h] =
                ll == 0.0f ? -INFINITY : (mu + log2f(ll)) * 0.6931471805599453f;
        }
      }
    }
    __syncthreads();  // the rings are free again
    w.advance(p, bad);
  }
  if (bad != 0) atomicOr(p.error, static_cast<int>(bad));
}

constexpr uint32_t kJoinRows = 32;
constexpr uint32_t kJoinThreads = 512;

// One CTA per (CTA of the attention, 32 rows): the partial results of the item that begins there
// and spans later CTAs, in their order, joined by their maxima.  A thread has 4 columns of a row
// and reads up to 4 partial results at once, a warp 32 neighbouring rows; the outputs are turned in
// shared memory so that they leave in whole rows (2-byte stores of 32 rows at once took four
// times as long as all the rest).  Bound by latency: splits, statistics, sums, and the CTAs an SM holds at once:
// with eight partial results in registers one CTA an SM, and 32 trees of up to 64 nodes over 8192 tokens took
// 324 us in all; with four, two CTAs, 318 us; with two, three, 316 us but 18.2 for 17.4 us at 7 trees of 33.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads, 2) attention_join_kernel(const __grid_constant__ AttnParams p) {
  __shared__ __align__(16) T turned[kJoinRows][HQB_MAX_HEAD_DIM + 8];
  const uint32_t first = blockIdx.x;
  griddep_launch_dependents();
  griddep_wait();
  const Split q = p.splits[first];
  if (q.last == first) return;
  const uint32_t row0 = blockIdx.y * kJoinRows, lrow = threadIdx.x % kJoinRows, row = row0 + lrow;
  const uint32_t rows = q.nodes * p.group, dim = p.c.head_dim;
  if (q.tile * p.rows + row0 >= rows) return;
  auto place = [&](uint32_t r, uint32_t& token, uint32_t& head) {
    const uint32_t at = q.tile * p.rows + r, node = p.by_group.quotient(at);
    token = q.start + node;
    head = q.head * p.group + at - node * p.group;
  };
  if (row < p.rows) {
    for (uint32_t d = threadIdx.x / kJoinRows * 4; d < dim; d += kJoinThreads / kJoinRows * 4) {
      float m = -INFINITY, l = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (uint32_t c0 = first; c0 <= q.last; c0 += 4) {
        float2 s[4];
        float4 v[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          s[k] = make_float2(-INFINITY, 0.0f);
          v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (c0 + k <= q.last) {
            const uint32_t c = c0 + k, slot = c == first ? 1u : 0u;
            s[k] = part_stats(p, c, slot)[row];
            v[k] = *reinterpret_cast<const float4*>(part_sums(p, c, slot) + ((d >> 2) * p.rows + row) * 4);
          }
        }
        float top = m;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) top = fmaxf(top, s[k].x);
        const float use = top == -INFINITY ? 0.0f : top, old = fast_exp2(m - use);
        l *= old;
        o.x *= old, o.y *= old, o.z *= old, o.w *= old;
        m = top;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          if (c0 + k > q.last) break;
          const float f = fast_exp2(s[k].x - use);
          l += f * s[k].y;
          o.x += f * v[k].x, o.y += f * v[k].y, o.z += f * v[k].z, o.w += f * v[k].w;
        }
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint2 r;
      r.x = l == 0.0f ? 0u : Elem<T>::pack(o.x * inv, o.y * inv);
      r.y = l == 0.0f ? 0u : Elem<T>::pack(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(&turned[lrow][d]) = r;
      if (d == 0 && p.a.lse != nullptr && q.tile * p.rows + row < rows) {
        uint32_t token, head;
        place(row, token, head);
        p.a.lse[static_cast<uint64_t>(token) * p.a.q_heads + head] =
            l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      }
    }
  }
  __syncthreads();
  const uint32_t pieces = p.vec ? dim / 8 : dim;
  for (uint32_t i = threadIdx.x; i < kJoinRows * pieces; i += kJoinThreads) {
    const uint32_t r = i / pieces, c = i - r * pieces;
    if (row0 + r >= p.rows || q.tile * p.rows + row0 + r >= rows) break;
    uint32_t token, head;
    place(row0 + r, token, head);
    T* out = static_cast<T*>(p.a.out) + token * p.a.out_token_stride + head * p.a.out_head_stride;
    if (p.vec) *reinterpret_cast<uint4*>(out + c * 8) = *reinterpret_cast<const uint4*>(&turned[r][c * 8]);
    else out[c] = turned[r][c];
  }
}

struct Shape {
  uint32_t rows, block, max_tiles, dim_pad, grid, whole, warps;
  uint64_t splits_bytes, parts_bytes;
  uint64_t bytes() const { return 256 + round_up(splits_bytes + parts_bytes, 256); }  // with the error word
};

bool shape_ok(const hqb_paged_cache* c, const hqb_attention_args* a) {
  if (!paged_cache_ok(c) || a == nullptr) return false;
  if (c->head_dim > HQB_MAX_HEAD_DIM || a->max_new == 0 || a->max_new > HQB_MAX_NODES) return false;
  if (a->q_heads == 0 || a->q_heads % c->kv_heads != 0 || a->q_heads > 65535) return false;
  if (a->requests > 0x7FFFFFu || a->tokens > 0x7FFFFFFFu || a->max_context > 0x7FFFFFFFu) return false;
  if (a->mask_words != 0 && a->mask_words * 32ull < a->max_new) return false;
  return true;
}

// 16-byte copies need 16-byte rows everywhere; anything else goes element by element.
bool aligned_rows(const hqb_paged_cache* c, const hqb_attention_args* a) {
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) |
                              reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                              reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->out);
  const uint64_t strides = c->page_stride | c->token_stride | c->head_stride | a->q_token_stride | a->q_head_stride |
                           a->kv_token_stride | a->kv_head_stride | a->out_token_stride | a->out_head_stride |
                           c->head_dim;
  return (addresses & 15u) == 0 && (strides & 7u) == 0;
}

// Items of up to 512 keys are not cut: one CTA's work of a few microseconds, where cutting it would
// add a second launch.
bool whole_items(const hqb_attention_args* a) { return static_cast<uint64_t>(a->max_context) + a->max_new <= 512; }

// Whether the tensor-memory kernel can take a shape: heads of up to 128, groups that fit a score
// tile, more rows than one tile of the rows kernel, or than two where items are not cut.  B200, us,
// rows / tensor-memory kernel, BF16, 64 heads over 8 of 128: 51 requests of 3 nodes and 1 token 14.7 /
// 24.6; 40 of 9 and 58 tokens 27.3 / 23.8; 32 of 64 and 400 tokens 194 / 66; 16 requests over 4096
// tokens: 2 nodes 45 / -, 4 nodes 97 / 53.
bool tmem_shape(const hqb_paged_cache* c, const hqb_attention_args* a) {
  const uint32_t group = a->q_heads / c->kv_heads;
  return c->head_dim <= 128 && group <= 128 && a->max_new * group > (whole_items(a) ? 32u : 16u);
}

// ... and the call: its masked scores are -inf * scale; a stride of zero (a broadcast input) or
// one past 2^39 elements has no tensor map.
bool takes_tmem(const hqb_paged_cache* c, const hqb_attention_args* a, bool aligned) {
  auto mapped = [](uint64_t n, uint64_t stride) { return n <= 1 || (stride > 0 && stride < (1ull << 39)); };
  return aligned && a->scale > 0.0f && tmem_shape(c, a) && mapped(a->q_heads, a->q_head_stride) &&
         mapped(a->tokens, a->q_token_stride) && mapped(c->kv_heads, a->kv_head_stride) &&
         mapped(a->tokens, a->kv_token_stride);
}

Shape shape_of(const hqb_paged_cache* c, const hqb_attention_args* a, bool tmem, int sms) {
  Shape s{};
  const uint32_t group = a->q_heads / c->kv_heads;
  s.dim_pad = c->head_dim <= 64 ? 64u : c->head_dim <= 128 ? 128u : 256u;
  s.rows = tmem ? 2 * (128 / group * group) : 16u;  // a score tile holds whole nodes
  s.block = tmem ? 128u : kKeyBlock;
  s.max_tiles = (a->max_new * group + s.rows - 1) / s.rows;
  s.grid = static_cast<uint32_t>(sms) * (tmem || s.dim_pad == 256 ? 1u : 2u);
  const uint64_t items = static_cast<uint64_t>(a->requests) * c->kv_heads * s.max_tiles;
  s.whole = whole_items(a) ? 1u : 0u;
  s.warps = 4;
  if (s.whole) {
    // few items: eight warps each; more than SMs: four, or two, twelve warps an SM
    const uint64_t n = static_cast<uint64_t>(sms);
    s.warps = items <= n ? 8u : items <= 3 * n ? 4u : 2u;
    const uint64_t slots = n * (tmem || s.dim_pad == 256 || s.warps == 8 ? 1 : 12 / s.warps);
    s.grid = static_cast<uint32_t>(items < slots ? (items > 0 ? items : 1) : slots);
  }
  s.splits_bytes = s.whole ? 0 : static_cast<uint64_t>(s.grid) * sizeof(Split);
  s.parts_bytes = s.whole ? 0 : static_cast<uint64_t>(s.grid) * 2 * s.rows * (s.dim_pad + 2) * 4;
  return s;
}

template <typename T, int DP, bool VEC, int kRowsWarps, int kStages>
cudaError_t launch_warps(const AttnParams& p, cudaStream_t st) {
  static DeviceOnce once;
  constexpr uint32_t smem = kRowsSmem<DP, kRowsWarps, kStages>;
  const cudaError_t e =
      allow_dynamic_smem(once, reinterpret_cast<const void*>(attention_rows_kernel<T, DP, VEC, kRowsWarps, kStages>), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(attention_rows_kernel<T, DP, VEC, kRowsWarps, kStages>, dim3(p.grid), kRowsWarps * 32, smem, 1, st, p);
}

template <typename T, int DP, bool VEC>
cudaError_t launch_rows(const AttnParams& p, cudaStream_t st) {
  if constexpr (DP <= 128) {
    if (p.whole && p.warps == 2) return launch_warps<T, DP, VEC, 2, 2>(p, st);
    if (p.whole && p.warps == 4) return launch_warps<T, DP, VEC, 4, 2>(p, st);
    if (p.whole) return launch_warps<T, DP, VEC, 8, 3>(p, st);
  }
  return launch_warps<T, DP, VEC, 4, 3>(p, st);
}

template <typename T, bool VEC>
cudaError_t launch_dim(const AttnParams& p, cudaStream_t st) {
  if (p.dim_pad == 64) return launch_rows<T, 64, VEC>(p, st);
  if (p.dim_pad == 128) return launch_rows<T, 128, VEC>(p, st);
  return launch_rows<T, 256, VEC>(p, st);
}

template <typename T>
cudaError_t launch_attention(const AttnParams& p, bool vec, bool tmem, cudaStream_t st) {
  cudaError_t e = tmem ? launch_attention_tmem<T>(p, st) : vec ? launch_dim<T, true>(p, st) : launch_dim<T, false>(p, st);
  if (e != cudaSuccess || p.whole) return e;
  const uint32_t rows = p.rows < p.a.max_new * p.group ? p.rows : p.a.max_new * p.group;
  return launch_dependent(attention_join_kernel<T>, dim3(p.grid, (rows + kJoinRows - 1) / kJoinRows), kJoinThreads, 0, 1, st, p);
}

}  // namespace
}  // namespace hqb

using namespace hqb;

extern "C" {

HQB_API uint64_t hqb_tree_attention_workspace_bytes(const hqb_paged_cache* c, const hqb_attention_args* a, int device) {
  if (!shape_ok(c, a)) return 0;
  const int sms = device_sm_count(device);
  if (sms <= 0) return 0;
  // the call chooses its kernel by alignment and scale too: room for either
  const uint64_t rows = shape_of(c, a, false, sms).bytes(), tmem = tmem_shape(c, a) ? shape_of(c, a, true, sms).bytes() : 0;
  return tmem > rows ? tmem : rows;
}

HQB_API int hqb_tree_attention(const hqb_paged_cache* c, const hqb_attention_args* a, void* workspace,
                               uint64_t workspace_bytes, void* stream) {
  if (!shape_ok(c, a)) return HQB_ERR_INVALID;
  if (a->mask != nullptr && a->mask_words == 0) return HQB_ERR_INVALID;
  if (a->requests > 0 && a->tokens > 0) {
    if (a->starts == nullptr || a->context_lens == nullptr || a->q == nullptr || a->k == nullptr || a->v == nullptr ||
        a->out == nullptr)
      return HQB_ERR_INVALID;
    if (a->table_stride > 0 && (a->tables == nullptr || c->k == nullptr || c->v == nullptr)) return HQB_ERR_INVALID;
  }
  const cudaError_t prior = take_prior_error();
  if (prior != cudaSuccess) return prior;
  if (a->requests == 0 || a->tokens == 0) return HQB_OK;
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const int sms = device_sm_count(device);
  if (sms <= 0) return HQB_ERR_INVALID;
  const bool vec = aligned_rows(c, a), tmem = takes_tmem(c, a, vec);
  const Shape s = shape_of(c, a, tmem, sms);
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 ||
      workspace_bytes < s.bytes())
    return HQB_ERR_INVALID;
  if (static_cast<uint64_t>(a->requests) * c->kv_heads * s.max_tiles > 0x7FFFFFFFull) return HQB_ERR_UNSUPPORTED;
  AttnParams p{};
  p.a = *a;
  p.c = *c;
  p.error = static_cast<int*>(workspace);
  p.splits = reinterpret_cast<Split*>(static_cast<uint8_t*>(workspace) + 256);
  p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256 + s.splits_bytes);
  p.group = a->q_heads / c->kv_heads;
  p.rows = s.rows;
  p.block_shift = s.block == 128 ? 7 : 6;
  p.by_page = Divisor::of(c->page_size);
  p.by_group = Divisor::of(p.group);
  p.by_rows = Divisor::of(p.rows);
  p.dim_pad = s.dim_pad;
  p.min_blocks = 4;
  p.whole = s.whole;
  p.grid = s.grid;
  p.warps = s.warps;
  p.vec = vec ? 1u : 0u;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  cudaStream_t st = as_stream(stream);
  return c->dtype == HQB_F16 ? launch_attention<__half>(p, vec, tmem, st)
                             : launch_attention<__nv_bfloat16>(p, vec, tmem, st);
}

}  // extern "C"
