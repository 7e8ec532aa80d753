// Low-rank adapters of many requests beside a shared projection (hqb_lora).
//   lora_kernel       y = base + scale * B (A x) for one tile of tokens of one adapter a cluster
//   lora_plan_kernel  groups the tokens of a large call by adapter into tiles
#include <cuda_runtime.h>

#include <type_traits>

#include "hqb_internal.h"
#include "hqb_serve.cuh"

namespace hqb {
namespace {

constexpr uint32_t kCluster = 8;         // CTAs that share a tile: the portable cluster size
constexpr uint32_t kThreads = 256;
constexpr uint32_t kDirectTokens = 256;  // up to here every cluster finds its own tile
constexpr uint32_t kMaxAdapters = 16383;

struct LoraTile {
  uint32_t group;  // adapter, or `adapters` for tokens without one
  uint32_t first;  // in the plan's token order
  uint32_t count;
  uint32_t pad;
};

struct LoraParams {
  hqb_lora_set s;
  const void* x;
  const int32_t* ids;
  const void* base;
  void* y;
  int* error;
  uint32_t* tile_count;  // planned calls
  LoraTile* tiles;
  uint32_t* order;
  uint64_t x_stride, base_stride, y_stride;
  uint32_t tokens;
  uint32_t planned;
  uint32_t in_place;  // base is y: tokens without an adapter need no work
  uint32_t tile_rows;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// The address in CTA `rank` of the cluster that corresponds to this CTA's `a`.
__device__ __forceinline__ uint32_t peer_smem(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_load(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void peer_store16(uint32_t a, uint16_t v) {
  asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory");
}
__device__ __forceinline__ void peer_store(uint32_t a, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

__device__ __forceinline__ uint32_t group_of(const LoraParams& p, uint32_t token, uint32_t& bad) {
  const int32_t id = __ldg(p.ids + token);
  if (id < 0) return p.s.adapters;
  if (static_cast<uint32_t>(id) >= p.s.adapters) {
    bad |= HQB_DEVERR_INDEX;
    return p.s.adapters;
  }
  return static_cast<uint32_t>(id);
}

// Eight consecutive 16-bit elements at `src`, of which `real` exist (zeros after them).
template <bool VEC>
__device__ __forceinline__ uint4 load8(const void* src, int64_t real) {
  if (VEC) return real > 0 ? __ldg(static_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
  const uint16_t* s = static_cast<const uint16_t*>(src);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = 2 * i < real ? s[2 * i] : 0, hi = 2 * i + 1 < real ? s[2 * i + 1] : 0;
    w[i] = lo | hi << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int RP>
struct LoraShape {
  static constexpr int kTiles8 = RP / 8;
  static constexpr int kGroups = RP <= 32 ? 1 : RP / 32;       // 32-rank pieces (16 ranks: one of 8-byte loads)
  static constexpr uint32_t kPitch = RP <= 32 ? RP : RP + 32;  // elements of a row of terms: conflict-free reads
};

// Terms of the inner vector per output type: FP32 outputs take 22 or more bits of it.
template <typename T, typename Y>
constexpr int kTerms = std::is_same<Y, float>::value ? (std::is_same<T, __half>::value ? 2 : 3) : 1;

template <typename T, typename Y, int RP, int M>
constexpr uint32_t kLoraSmem = 64 * 4 + M * 4 + M * 4 + kTerms<T, Y> * M * LoraShape<RP>::kPitch * 2 + M * RP * 4 +
                               (M == 16 ? 8 : 4) * M * RP * 4;

// Mathematics: t = A x (FP32 sums of exact 16-bit products), y = base + scale B t.
// Split: a cluster of 8 CTAs takes one tile of up to M tokens of one adapter.  First its CTAs and
// their warps divide the columns of x and A (every element of x is read once, straight into MMA
// fragments: the columns of a 32-column step may be taken in any order, so a lane's 16 bytes are
// both k-halves of two MMAs); the partial t are summed in warp order, then through distributed
// shared memory in CTA order, so the bits do not depend on timing.  Then the CTAs divide the rows
// of B and of the output: the four 8-row tiles of a 32-row step take rows 8(g/2)+2j+(g%2), which
// gives each lane 8 adjacent outputs of a token.  One launch, no scratch, no atomics.
// Bound by bytes: x, base and y once, A and B once a tile (from L2 for every tile but the first).
template <typename T, typename Y, int RP, int M, bool VEC>
__global__ void __launch_bounds__(kThreads) lora_kernel(const __grid_constant__ LoraParams p) {
  using S = LoraShape<RP>;
  constexpr int kMW = M == 16 ? 1 : 2;               // 16-row tiles a warp multiplies in the first product
  constexpr uint32_t kWM = M == 16 ? 1 : 2;          // warps along the rows
  constexpr uint32_t kSlices = 8 / kWM;              // warps along the columns
  constexpr int kN = kTerms<T, Y>;
  extern __shared__ __align__(128) uint8_t sm[];
  uint32_t* s_info = reinterpret_cast<uint32_t*>(sm);                       // 64 words
  int32_t* s_token = reinterpret_cast<int32_t*>(sm + 256);                  // [M], -1: no row
  float* s_factor = reinterpret_cast<float*>(s_token + M);                  // [M]
  T* s_terms = reinterpret_cast<T*>(s_factor + M);                          // [kN][M][kPitch]
  float* s_sum = reinterpret_cast<float*>(s_terms + kN * M * S::kPitch);    // [M][RP] this CTA's t
  float* s_part = s_sum + M * RP;                                           // [kSlices][M][RP]
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const uint32_t cta = cluster_rank(), tile = blockIdx.x / kCluster;
  uint32_t bad = 0;
  griddep_wait();

  // ---- the tile: an adapter and its tokens
  uint32_t group, count;
  if (p.planned) {
    if (tile >= *p.tile_count) return;
    const LoraTile t = p.tiles[tile];
    group = t.group;
    count = t.count;
    for (uint32_t i = tid; i < M; i += kThreads) s_token[i] = i < count ? static_cast<int32_t>(p.order[t.first + i]) : -1;
  } else {
    // the cluster of a token that has a multiple of M tokens of its adapter before it takes
    // that token and the adapter's next M - 1
    group = group_of(p, tile, bad);
    const bool same = tid < p.tokens && group_of(p, tid, bad) == group;
    const uint32_t votes = ballot(same);
    if (lane == 0) s_info[warp] = votes;
    for (uint32_t i = tid; i < M; i += kThreads) s_token[i] = -1;
    __syncthreads();
    uint32_t before = 0, mine = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
      const uint32_t v = s_info[w], n = __popc(v);
      all += n;
      if (w < (tile >> 5)) before += n;
      if (w == (tile >> 5)) before += __popc(v & ((1u << (tile & 31)) - 1u));
      if (w < warp) mine += n;
    }
    if (before % M != 0) return;
    mine += __popc(votes & ((1u << lane) - 1u));
    if (same && mine >= before && mine < before + M) s_token[mine - before] = static_cast<int32_t>(tid);
    count = min(static_cast<uint32_t>(M), all - before);
  }
  __syncthreads();
  uint32_t rank = 0;
  float scale = 0.0f;
  if (group < p.s.adapters) {
    const int32_t v = p.s.ranks != nullptr ? __ldg(p.s.ranks + group) : static_cast<int32_t>(p.s.max_rank);
    if (v < 0 || v > static_cast<int32_t>(p.s.max_rank)) bad |= HQB_DEVERR_INDEX;
    rank = v < 0 ? 0u : min(static_cast<uint32_t>(v), p.s.max_rank);
    scale = p.s.scales != nullptr ? __ldg(p.s.scales + group) : 1.0f;
  }
  if (bad != 0) atomicOr(p.error, static_cast<int>(bad));
  if (rank == 0 && p.in_place) return;
  const uint64_t cols = p.s.cols, rows = p.s.rows;

  if (rank != 0) {
    // ---- t = A x, this CTA's columns
    const T* a = static_cast<const T*>(p.s.a) + static_cast<uint64_t>(group) * p.s.max_rank * cols;
    const uint32_t wm = warp % kWM, slice = warp / kWM;
    const T* xr[kMW][2];
    bool xl[kMW][2];
#pragma unroll
    for (int i = 0; i < kMW; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int32_t t = s_token[(wm * kMW + i) * 16 + g + 8 * e];
        xl[i][e] = t >= 0;
        xr[i][e] = static_cast<const T*>(p.x) + static_cast<uint64_t>(max(t, 0)) * p.x_stride;
      }
    float acc[kMW][S::kTiles8][4];
#pragma unroll
    for (int i = 0; i < kMW; ++i)
#pragma unroll
      for (int n = 0; n < S::kTiles8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.0f;
    const uint32_t steps = static_cast<uint32_t>((cols + 31) / 32);
    const uint32_t step0 = static_cast<uint64_t>(steps) * cta / kCluster, step1 = static_cast<uint64_t>(steps) * (cta + 1) / kCluster;
    constexpr int kAhead = RP <= 32 ? (M == 16 ? 4 : 2) : (M == 16 && RP == 64 ? 2 : 1);
    for (uint32_t st = step0 + slice; st < step1; st += kSlices * kAhead) {
      uint4 xv[kAhead][kMW][2], av[kAhead][S::kTiles8];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t s = st + u * kSlices;
        const uint64_t col = static_cast<uint64_t>(s) * 32 + q * 8;
        const int64_t real = s < step1 ? static_cast<int64_t>(cols) - static_cast<int64_t>(col) : 0;
#pragma unroll
        for (int i = 0; i < kMW; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) xv[u][i][e] = load8<VEC>(xr[i][e] + col, xl[i][e] ? real : 0);
#pragma unroll
        for (int n = 0; n < S::kTiles8; ++n)
          av[u][n] = load8<VEC>(a + (n * 8 + g) * cols + col, n * 8 + g < rank ? real : 0);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int n = 0; n < S::kTiles8; ++n)
#pragma unroll
          for (int i = 0; i < kMW; ++i) {
            Elem<T>::mma(acc[i][n], xv[u][i][0].x, xv[u][i][1].x, xv[u][i][0].y, xv[u][i][1].y, av[u][n].x, av[u][n].y);
            Elem<T>::mma(acc[i][n], xv[u][i][0].z, xv[u][i][1].z, xv[u][i][0].w, xv[u][i][1].w, av[u][n].z, av[u][n].w);
          }
    }
#pragma unroll
    for (int i = 0; i < kMW; ++i)
#pragma unroll
      for (int n = 0; n < S::kTiles8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(s_part + (slice * M + (wm * kMW + i) * 16 + g + 8 * e) * RP + n * 8 + q * 2) =
              make_float2(acc[i][n][2 * e], acc[i][n][2 * e + 1]);
    __syncthreads();
    for (uint32_t i = tid; i < M * RP; i += kThreads) {
      float v = 0.0f;
#pragma unroll
      for (uint32_t k = 0; k < kSlices; ++k) v += s_part[k * M * RP + i];
      s_sum[i] = v;
    }
    cluster_sync();
    // ---- sum over the CTAs; each owns M / 8 rows, a warp a row, and hands the row's terms and
    // factor to all of them
    for (uint32_t own = warp; own < M / kCluster; own += kThreads / 32) {
      const uint32_t row = cta * (M / kCluster) + own;
      constexpr int kPer = (RP + 31) / 32;
      float v[kPer], top = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t r = i * 32 + lane;
        float sum = 0.0f;
        if (r < RP) {
          const uint32_t at = smem_u32(s_sum + row * RP + r);
#pragma unroll
          for (uint32_t c = 0; c < kCluster; ++c) sum += peer_load(peer_smem(at, c));
        }
        v[i] = r < rank ? sum : 0.0f;
        top = fmaxf(top, fabsf(v[i]));
      }
      // FP16 terms: the row scaled by a power of two to its largest magnitude (exact), so that
      // neither large nor small activations leave the type's range; BF16 has FP32's range
      int e = 0;
      if (std::is_same<T, __half>::value) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (top > 0.0f && top < INFINITY) e = max(-100, min(100, ilogbf(top) - 14));
      }
      const float down = ldexpf(1.0f, -e);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t r = i * 32 + lane;
        float rest = v[i] * down;
#pragma unroll
        for (int k = 0; k < kN; ++k) {
          const T term = Elem<T>::from_float(rest);
          const float back = Elem<T>::to_float(term);
          if (r < RP) {
            const uint32_t at = smem_u32(s_terms + (k * M + row) * S::kPitch + r);
#pragma unroll
            for (uint32_t c = 0; c < kCluster; ++c) peer_store16(peer_smem(at, c), *reinterpret_cast<const uint16_t*>(&term));
          }
          // an infinity or NaN is all in its first term
          rest = fabsf(back) < INFINITY ? rest - back : 0.0f;
        }
      }
      if (lane < kCluster) peer_store(peer_smem(smem_u32(s_factor + row), lane), scale * ldexpf(1.0f, e));
    }
    cluster_sync();
  }

  // ---- y = base + factor * B t, this CTA's rows of B
  const T* b = static_cast<const T*>(p.s.b) + static_cast<uint64_t>(min(group, p.s.adapters - 1)) * p.s.max_rank * rows;
  const uint32_t steps = static_cast<uint32_t>((rows + 31) / 32);
  const uint32_t step0 = static_cast<uint64_t>(steps) * cta / kCluster, step1 = static_cast<uint64_t>(steps) * (cta + 1) / kCluster;
  for (uint32_t st = step0 + warp; st < step1; st += kThreads / 32) {
    uint4 bv[4][S::kGroups];
    if (rank != 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t n = static_cast<uint64_t>(st) * 32 + 8 * (g >> 1) + 2 * j + (g & 1);
        const T* row = b + n * p.s.max_rank;
#pragma unroll
        for (int k = 0; k < S::kGroups; ++k) {
          if constexpr (RP == 16) {
            const int32_t left = n < rows ? static_cast<int32_t>(rank) - static_cast<int32_t>(q * 4) : 0;
            uint2 v = make_uint2(0, 0);
            if (VEC) {
              if (left > 0) v = __ldg(reinterpret_cast<const uint2*>(row + q * 4));
              if (left < 4) v.y &= left == 3 ? 0xFFFFu : 0u;
              if (left < 2) v.x &= left == 1 ? 0xFFFFu : 0u;
            } else {
              const uint4 w = load8<false>(row + q * 4, left < 4 ? left : 4);
              v = make_uint2(w.x, w.y);
            }
            bv[j][k] = make_uint4(v.x, v.y, 0, 0);
          } else {
            const int32_t left = n < rows ? static_cast<int32_t>(rank) - static_cast<int32_t>(k * 32 + q * 8) : 0;
            uint4 v = load8<VEC>(row + k * 32 + q * 8, left);
            if (VEC && left < 8) {  // columns past the adapter's rank may hold anything
              v.x &= left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u;
              v.y &= left >= 4 ? 0xFFFFFFFFu : left == 3 ? 0xFFFFu : 0u;
              v.z &= left >= 6 ? 0xFFFFFFFFu : left == 5 ? 0xFFFFu : 0u;
              v.w &= left == 7 ? 0xFFFFu : 0u;
            }
            bv[j][k] = v;
          }
        }
      }
    }
    const uint64_t n0 = static_cast<uint64_t>(st) * 32 + q * 8;
    const int64_t real = static_cast<int64_t>(rows) - static_cast<int64_t>(n0);
#pragma unroll
    for (int mt = 0; mt < M / 16; ++mt) {
      if (mt * 16 >= static_cast<int>(count)) break;
      float out[2][8];
      int32_t token[2];
      // base first: its loads run under the products
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        token[e] = s_token[mt * 16 + g + 8 * e];
#pragma unroll
        for (int i = 0; i < 8; ++i) out[e][i] = 0.0f;
        if (token[e] >= 0 && p.base != nullptr) {
          const Y* src = static_cast<const Y*>(p.base) + static_cast<uint64_t>(token[e]) * p.base_stride + n0;
          if (VEC && real > 0) {
            if constexpr (sizeof(Y) == 4) {
              const float4 lo = reinterpret_cast<const float4*>(src)[0], hi = reinterpret_cast<const float4*>(src)[1];
              out[e][0] = lo.x; out[e][1] = lo.y; out[e][2] = lo.z; out[e][3] = lo.w;
              out[e][4] = hi.x; out[e][5] = hi.y; out[e][6] = hi.z; out[e][7] = hi.w;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(src);
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = Elem<T>::unpack(w[i]);
                out[e][2 * i] = f.x;
                out[e][2 * i + 1] = f.y;
              }
            }
          } else if (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i < real) {
                if constexpr (sizeof(Y) == 4) out[e][i] = src[i];
                else out[e][i] = Elem<T>::to_float(src[i]);
              }
          }
        }
      }
      if (rank != 0) {
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
#pragma unroll
        for (int t = kN - 1; t >= 0; --t) {  // small terms first
          const T* lo = s_terms + (t * M + mt * 16 + g) * S::kPitch;
          const T* hi = lo + 8 * S::kPitch;
#pragma unroll
          for (int k = 0; k < S::kGroups; ++k) {
            if constexpr (RP == 16) {
              const uint2 u = *reinterpret_cast<const uint2*>(lo + q * 4), v = *reinterpret_cast<const uint2*>(hi + q * 4);
#pragma unroll
              for (int j = 0; j < 4; ++j) Elem<T>::mma(acc[j], u.x, v.x, u.y, v.y, bv[j][k].x, bv[j][k].y);
            } else {
              const uint4 u = *reinterpret_cast<const uint4*>(lo + k * 32 + q * 8);
              const uint4 v = *reinterpret_cast<const uint4*>(hi + k * 32 + q * 8);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                Elem<T>::mma(acc[j], u.x, v.x, u.y, v.y, bv[j][k].x, bv[j][k].y);
                Elem<T>::mma(acc[j], u.z, v.z, u.w, v.w, bv[j][k].z, bv[j][k].w);
              }
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = s_factor[mt * 16 + g + 8 * e];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            out[e][2 * j] += f * acc[j][2 * e];
            out[e][2 * j + 1] += f * acc[j][2 * e + 1];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (token[e] < 0) continue;
        Y* dst = static_cast<Y*>(p.y) + static_cast<uint64_t>(token[e]) * p.y_stride + n0;
        if (VEC) {
          if (real <= 0) continue;
          if constexpr (sizeof(Y) == 4) {
            reinterpret_cast<float4*>(dst)[0] = make_float4(out[e][0], out[e][1], out[e][2], out[e][3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(out[e][4], out[e][5], out[e][6], out[e][7]);
          } else {
            *reinterpret_cast<uint4*>(dst) = make_uint4(Elem<T>::pack(out[e][0], out[e][1]), Elem<T>::pack(out[e][2], out[e][3]),
                                                        Elem<T>::pack(out[e][4], out[e][5]), Elem<T>::pack(out[e][6], out[e][7]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < real) {
              if constexpr (sizeof(Y) == 4) dst[i] = out[e][i];
              else dst[i] = Elem<T>::from_float(out[e][i]);
            }
        }
      }
    }
  }
}

// Groups the tokens by adapter: counts, offsets, then each token to its group's next place.  The
// order within a group may change between runs; a token's output does not depend on it.
__global__ void __launch_bounds__(1024) lora_plan_kernel(const __grid_constant__ LoraParams p) {
  extern __shared__ uint32_t count[];  // [groups], then the groups' next places
  __shared__ uint32_t red[2][32];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, groups = p.s.adapters + 1;
  uint32_t bad = 0;
  griddep_launch_dependents();
  for (uint32_t i = tid; i < groups; i += 1024) count[i] = 0;
  __syncthreads();
  for (uint32_t t = tid; t < p.tokens; t += 1024) atomicAdd(&count[group_of(p, t, bad)], 1u);
  __syncthreads();
  uint32_t tokens = 0, tiles = 0;
  for (uint32_t g0 = 0; g0 < groups; g0 += 1024) {
    const uint32_t grp = g0 + tid;
    uint32_t n = grp < groups ? count[grp] : 0;
    if (p.in_place && grp == p.s.adapters) n = 0;
    const uint32_t nt = (n + p.tile_rows - 1) / p.tile_rows;
    uint32_t a = n, b = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= static_cast<uint32_t>(o)) a += ua, b += ub;
    }
    if (lane == 31) red[0][warp] = a, red[1][warp] = b;
    __syncthreads();
    uint32_t fa = tokens, fb = tiles;
#pragma unroll 4
    for (uint32_t w = 0; w < 32; ++w) {
      if (w < warp) fa += red[0][w], fb += red[1][w];
      tokens += red[0][w];
      tiles += red[1][w];
    }
    fa += a - n;
    fb += b - nt;
    if (grp < groups) count[grp] = fa;
    for (uint32_t k = 0; k < nt; ++k)
      p.tiles[fb + k] = LoraTile{grp, fa + k * p.tile_rows, min(p.tile_rows, n - k * p.tile_rows), 0u};
    __syncthreads();
  }
  for (uint32_t t = tid; t < p.tokens; t += 1024) {
    const uint32_t grp = group_of(p, t, bad);
    if (p.in_place && grp == p.s.adapters) continue;
    p.order[atomicAdd(&count[grp], 1u)] = t;
  }
  if (tid == 0) *p.tile_count = tiles;
  if (bad != 0) atomicOr(p.error, static_cast<int>(bad));
}

struct Layout {
  uint64_t tiles, order, total;
  uint32_t max_tiles;
};

Layout layout(const hqb_lora_set* s, uint32_t tokens, uint32_t tile_rows) {
  Layout l{};
  // every group may end in a partly filled tile
  const uint64_t groups = static_cast<uint64_t>(s->adapters) + 1;
  l.max_tiles = static_cast<uint32_t>(tokens / tile_rows + (groups < tokens ? groups : tokens));
  l.tiles = 512;
  l.order = l.tiles + round_up(static_cast<uint64_t>(l.max_tiles) * sizeof(LoraTile), 256);
  l.total = l.order + round_up(static_cast<uint64_t>(tokens) * 4, 256);
  return l;
}

bool set_ok(const hqb_lora_set* s) {
  if (s == nullptr || s->rows == 0 || s->cols == 0 || s->adapters == 0 || s->max_rank == 0 || s->max_rank > HQB_MAX_RANK)
    return false;
  if (s->rows > 0x7FFFFFFFull || s->cols > 0x7FFFFFFFull) return false;
  return s->dtype == HQB_F16 || s->dtype == HQB_BF16;
}

template <typename T, typename Y, int RP, int M, bool VEC>
cudaError_t launch_lora(const LoraParams& p, uint32_t tiles, cudaStream_t st) {
  static DeviceOnce once;
  constexpr uint32_t smem = kLoraSmem<T, Y, RP, M>;
  const void* f = reinterpret_cast<const void*>(lora_kernel<T, Y, RP, M, VEC>);
  const cudaError_t e = allow_dynamic_smem(once, f, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles * kCluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kCluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.planned ? 2 : 1;  // a planned call follows its own plan kernel
  return cudaLaunchKernelEx(&cfg, lora_kernel<T, Y, RP, M, VEC>, p);
}

template <typename T, typename Y>
cudaError_t launch_rank(const LoraParams& p, bool vec, uint32_t tiles, cudaStream_t st) {
  if (!vec) return launch_lora<T, Y, 128, 16, false>(p, tiles, st);
  const uint32_t r = p.s.max_rank;
  if (p.tile_rows == 16) {
    if (r <= 16) return launch_lora<T, Y, 16, 16, true>(p, tiles, st);
    if (r <= 32) return launch_lora<T, Y, 32, 16, true>(p, tiles, st);
    if (r <= 64) return launch_lora<T, Y, 64, 16, true>(p, tiles, st);
    return launch_lora<T, Y, 128, 16, true>(p, tiles, st);
  }
  if (r <= 16) return launch_lora<T, Y, 16, 64, true>(p, tiles, st);
  if (r <= 32) return launch_lora<T, Y, 32, 64, true>(p, tiles, st);
  if (r <= 64) return launch_lora<T, Y, 64, 64, true>(p, tiles, st);
  return launch_lora<T, Y, 128, 64, true>(p, tiles, st);
}

}  // namespace
}  // namespace hqb

using namespace hqb;

extern "C" {

HQB_API uint64_t hqb_lora_workspace_bytes(const hqb_lora_set* s, uint32_t tokens, int device) {
  (void)device;
  if (!set_ok(s) || tokens > 0x7FFFFFFFu) return 0;
  return tokens <= kDirectTokens ? 256 : layout(s, tokens, 16).total;
}

HQB_API int hqb_lora(const hqb_lora_set* s, const void* x, uint64_t x_stride, const int32_t* ids, uint32_t tokens,
                     const void* base, uint64_t base_stride, void* y, int y_dtype, uint64_t y_stride, void* workspace,
                     uint64_t workspace_bytes, void* stream) {
  if (!set_ok(s) || tokens > 0x7FFFFFFFu) return HQB_ERR_INVALID;
  if (y_dtype != s->dtype && y_dtype != HQB_F32) return HQB_ERR_INVALID;
  if (tokens > 0) {
    if (s->a == nullptr || s->b == nullptr || x == nullptr || ids == nullptr || y == nullptr) return HQB_ERR_INVALID;
    if (x_stride < s->cols || y_stride < s->rows || (base != nullptr && base_stride < s->rows)) return HQB_ERR_INVALID;
    if (base == y && base_stride != y_stride) return HQB_ERR_INVALID;
  }
  if (s->adapters > kMaxAdapters) return HQB_ERR_UNSUPPORTED;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 ||
      workspace_bytes < hqb_lora_workspace_bytes(s, tokens, 0))
    return HQB_ERR_INVALID;
  const cudaError_t prior = take_prior_error();
  if (prior != cudaSuccess) return prior;
  if (tokens == 0) return HQB_OK;
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(s->a) | reinterpret_cast<uintptr_t>(s->b) |
                              reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(base) |
                              reinterpret_cast<uintptr_t>(y);
  const uint64_t sizes = s->cols | s->rows | s->max_rank | x_stride | y_stride | (base != nullptr ? base_stride : 0);
  const bool vec = (addresses & 15u) == 0 && (sizes & 7u) == 0;
  LoraParams p{};
  p.s = *s;
  p.x = x;
  p.ids = ids;
  p.base = base;
  p.y = y;
  p.x_stride = x_stride;
  p.base_stride = base_stride;
  p.y_stride = y_stride;
  p.tokens = tokens;
  p.planned = tokens > kDirectTokens ? 1u : 0u;
  p.in_place = base == y ? 1u : 0u;
  p.tile_rows = vec && p.planned ? 64u : 16u;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.error = reinterpret_cast<int*>(ws);
  cudaStream_t st = as_stream(stream);
  uint32_t tiles = tokens;
  if (p.planned) {
    const Layout l = layout(s, tokens, p.tile_rows);
    p.tile_count = reinterpret_cast<uint32_t*>(ws + 256);
    p.tiles = reinterpret_cast<LoraTile*>(ws + l.tiles);
    p.order = reinterpret_cast<uint32_t*>(ws + l.order);
    tiles = l.max_tiles;
    if (tiles > 0x7FFFFFFFu / kCluster) return HQB_ERR_UNSUPPORTED;
    static DeviceOnce once;
    const cudaError_t e = allow_dynamic_smem(once, reinterpret_cast<const void*>(lora_plan_kernel), (kMaxAdapters + 1) * 4);
    if (e != cudaSuccess) return e;
    lora_plan_kernel<<<1, 1024, (s->adapters + 1) * 4, st>>>(p);
    const cudaError_t e2 = cudaGetLastError();
    if (e2 != cudaSuccess) return e2;
  }
  if (s->dtype == HQB_F16)
    return y_dtype == HQB_F32 ? launch_rank<__half, float>(p, vec, tiles, st) : launch_rank<__half, __half>(p, vec, tiles, st);
  return y_dtype == HQB_F32 ? launch_rank<__nv_bfloat16, float>(p, vec, tiles, st)
                            : launch_rank<__nv_bfloat16, __nv_bfloat16>(p, vec, tiles, st);
}

}  // extern "C"
