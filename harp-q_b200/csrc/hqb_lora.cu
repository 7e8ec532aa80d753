// Low-rank adapters of many requests beside a shared projection (hqb_lora).
//   lora_kernel         y = base + scale * B (A x) for up to 16 tokens of one adapter a cluster, in one
//                       launch: decode steps, and rows that no 16-byte access fits
// Calls of many tokens, three launches:
//   lora_plan_kernel    groups the tokens by adapter into tiles
//   lora_lay_kernel     rows of B in multiples of 8 ranks (only where max_rank is not one)
//   lora_shrink_kernel  t = A x
//   lora_expand_kernel  y = base + scale * B t
#include <cuda_runtime.h>

#include <type_traits>

#include "hqb_internal.h"
#include "hqb_serve.cuh"

namespace hqb {
namespace {

constexpr uint32_t kCluster = 8;         // CTAs that share a tile: the portable cluster size
constexpr uint32_t kThreads = 256;
// Up to kVoteTokens tokens, or kCountTokens of fewer than kCountGroups adapters, every cluster finds its own
// tile; above, and where the shrink and expand kernels run, lora_plan_kernel finds them all.  B200, us, own /
// planned, FP16, rank 16, 4096 x 4096: 300 tokens of 8 adapters 8.8 / 10.8; 600 of 64 17.3 / 17.8, of 128
// 25.2 / 24.5; 1000 of 64 18.4 / 18.9, of 900 121 / 96.
constexpr uint32_t kVoteTokens = kThreads, kCountTokens = 4 * kThreads, kCountGroups = 96;
// A call of more than kVoteTokens tokens keeps to lora_kernel up to this many tokens * padded rank.  B200, us,
// lora_kernel / shrink + expand, 8 adapters: rank 16, 4096 x 4096, FP16: 1024 tokens 17.4 / 25.6, 2048 tokens
// 26.2 / 23.6; rank 24, 1024 x 8192, BF16: 777 tokens 15.3 / 23.2; rank 64, 11008 x 4096, FP16: 300 tokens
// 21.6 / 30.8, 777 tokens 42.8 / 36.8; rank 64, 4096 x 4096, BF16: 500 tokens 21.9 / 23.7.
constexpr uint64_t kClusterWork = 32768;
constexpr uint32_t kMaxAdapters = 16383;
constexpr uint32_t kLayAdapters = 8;  // adapters whose rows of B are laid out for any number of tokens

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
  uint32_t max_tiles;
  uint32_t splits;    // column ranges of the first product
  uint32_t stages;    // of lora_kernel's rings
  uint32_t pitch;     // elements of a row of b
  void* laid;         // lora_lay_kernel: b in rows of `pitch`, which then is the call's b
  float* inner;       // [splits][max_tiles][tile_rows][padded rank]
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
  const int32_t id = p.ids[token];
  if (id < 0) return p.s.adapters;
  if (static_cast<uint32_t>(id) >= p.s.adapters) {
    bad |= HQB_DEVERR_INDEX;
    return p.s.adapters;
  }
  return static_cast<uint32_t>(id);
}

// Eight consecutive 16-bit elements at `src`, of which `real` exist (zeros after them).  From L2: every
// element is read once (777 tokens of rank 24 16.7 us through L1, 15.5 us so).
template <bool VEC>
__device__ __forceinline__ uint4 load8(const void* src, int64_t real) {
  if (VEC) return real > 0 ? __ldcg(static_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
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

// Terms of the inner vector per output type: FP32 outputs take 22 or more bits of it.  16-bit outputs, which
// are rounded to the same type anyway, take one: its rounding adds about as much again to an output's error.
// B200, us, one term / two: one token 5.9 / 6.1, 777 tokens 15.4 / 15.8, 8192 tokens 116 / 145.
template <typename T, typename Y>
constexpr int kTerms = std::is_same<Y, float>::value ? (std::is_same<T, __half>::value ? 2 : 3) : 1;

// A row of t as terms of T: v[i] is rank i * 32 + lane, already zero past the adapter's rank.  FP16
// terms are of the row scaled by a power of two to its largest magnitude (exact), so that neither
// large nor small activations leave the type's range; BF16 has FP32's range.  put(k, rank, bits)
// takes the terms; the row's factor is returned.
template <typename T, int RP, int KN, typename Put>
__device__ __forceinline__ float split_row(const float (&v)[(RP + 31) / 32], uint32_t lane, float scale, Put put) {
  constexpr int kPer = (RP + 31) / 32;
  int e = 0;
  if (std::is_same<T, __half>::value) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = fmaxf(top, fabsf(v[i]));
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
    for (int k = 0; k < KN; ++k) {
      const T term = Elem<T>::from_float(rest);
      const float back = Elem<T>::to_float(term);
      if (r < RP) put(k, r, *reinterpret_cast<const uint16_t*>(&term));
      rest = fabsf(back) < INFINITY ? rest - back : 0.0f;  // an infinity or NaN is all in its first term
    }
  }
  return scale * ldexpf(1.0f, e);
}

// The second product for one tile: steps of 32 outputs, a warp a step.  The four 8-row tiles of B of
// a step take rows 8(g/2)+2j+(g%2) of it, which gives each lane 8 adjacent outputs of a token.
// B and base come by asynchronous copies into a ring of which every lane reads back exactly what
// it copied itself, so the loop has no barrier, and the first stages can be in flight before t is
// known (start() may run under the first product).
template <typename T, typename Y, int RP, int M>
struct Expand {
  using S = LoraShape<RP>;
  static constexpr int kN = kTerms<T, Y>;
  static constexpr int kBaseVecs = sizeof(Y) == 4 ? 2 : 1;             // 16-byte pieces of 8 outputs
  static constexpr uint32_t kBBytes = RP == 16 ? 4 * 8 : 4 * S::kGroups * 16;  // a lane's B of a step
  static constexpr uint32_t kBaseBytes = M / 16 * 2 * kBaseVecs * 16;
  static constexpr uint32_t kStage = 32 * (kBBytes + kBaseBytes);      // a warp's bytes of a step

  static constexpr int kRowsEach = M / 8;  // rows of a lane: g and g + 8 of every 16
  // terms of a lane that stay in registers over the steps, where they are few
  static constexpr bool kHold = kN == 1 && RP > 16 && M / 16 * S::kGroups <= 8;

  const T* b;                  // the lane's first B row of step 0
  const Y* base[kRowsEach];    // the lane's rows (i * 8 + g) at its first output of step 0; past the tile's its first
  Y* y[kRowsEach];
  uint64_t rows;
  uint32_t pitch, rank, count, ring, stages, lane;
  bool based;

  __device__ __forceinline__ void prepare(const LoraParams& p, uint32_t group, uint32_t rank_, uint32_t count_,
                                          const int32_t* s_token, uint32_t ring_, uint32_t stages_) {
    lane = threadIdx.x & 31;
    const uint32_t g = lane >> 2, q = lane & 3;
    rows = p.s.rows, pitch = p.pitch, rank = rank_, count = count_, ring = ring_, stages = stages_;
    based = p.base != nullptr;
    b = static_cast<const T*>(p.s.b) + (static_cast<uint64_t>(min(group, p.s.adapters - 1)) * rows + 8 * (g >> 1) + (g & 1)) * pitch +
        q * (RP == 16 ? 4 : 8);
#pragma unroll
    for (int i = 0; i < kRowsEach; ++i) {
      const int32_t t = s_token[(i >> 1) * 16 + g + 8 * (i & 1)];
      const uint64_t row = static_cast<uint64_t>(t < 0 ? s_token[0] : t);
      base[i] = static_cast<const Y*>(p.base) + row * p.base_stride + q * 8;
      y[i] = static_cast<Y*>(p.y) + row * p.y_stride + q * 8;
    }
  }
  // copies of step st into stage at `to` (shared address)
  __device__ __forceinline__ void load(uint32_t st, uint32_t to) const {
    const uint32_t g = lane >> 2, q = lane & 3;
    const uint64_t n0 = static_cast<uint64_t>(st) * 32;
    const uint32_t left = rows - n0 < 32 ? static_cast<uint32_t>(rows - n0) : 32u;  // outputs of the step
    if (rank != 0) {
      const T* row = b + n0 * pitch;
      if (left == 32 && rank == RP) {  // all of it: no sizes to choose
#pragma unroll
        for (int j = 0; j < 4; ++j, row += 2 * pitch) {
          if constexpr (RP == 16) {
            cp_async8(to + (j * 32 + lane) * 8, row, 8u);
          } else {
#pragma unroll
            for (int k = 0; k < S::kGroups; ++k) cp_async16(to + ((j * S::kGroups + k) * 32 + lane) * 16, row + k * 32, 16u);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j, row += 2 * pitch) {
          const bool inside = 8 * (g >> 1) + 2 * j + (g & 1) < left;
          if constexpr (RP == 16) {
            const bool real = inside && q * 4 < rank;
            cp_async8(to + (j * 32 + lane) * 8, real ? row : b, real ? 8u : 0u);
          } else {
#pragma unroll
            for (int k = 0; k < S::kGroups; ++k) {
              const bool real = inside && k * 32 + q * 8 < rank;
              cp_async16(to + ((j * S::kGroups + k) * 32 + lane) * 16, real ? row + k * 32 : b, real ? 16u : 0u);
            }
          }
        }
      }
    }
    if (based && q * 8 < left) {
#pragma unroll
      for (int i = 0; i < kRowsEach; ++i) {
        if (M == 16 && i * 8 + g >= count) break;  // few rows: none is copied in vain
#pragma unroll
        for (int v = 0; v < kBaseVecs; ++v)
          cp_async16(to + 32 * kBBytes + ((i * kBaseVecs + v) * 32 + lane) * 16, base[i] + n0 + v * 4, 16u);
      }
    }
  }
  // the first stages - 1 steps of a warp that takes steps first, first + 8, ... below end
  __device__ __forceinline__ void start(uint32_t first, uint32_t end) const {
    for (uint32_t s = 0; s + 1 < stages; ++s) {
      if (first + s * 8 < end) load(first + s * 8, ring + s * kStage);
      cp_async_commit();
    }
  }
  __device__ __forceinline__ void run(uint32_t first, uint32_t end, const T* terms, const float* factor) const {
    const uint32_t g = lane >> 2, q = lane & 3;
    uint32_t stage = 0;
    float f[kRowsEach];
    uint4 held[kHold ? M / 16 : 1][kHold ? S::kGroups : 1][2];
    if (rank != 0) {
#pragma unroll
      for (int i = 0; i < kRowsEach; ++i) f[i] = factor[(i >> 1) * 16 + g + 8 * (i & 1)];
      if constexpr (kHold) {
#pragma unroll
        for (int mt = 0; mt < M / 16; ++mt)
#pragma unroll
          for (int k = 0; k < S::kGroups; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              held[mt][k][e] = *reinterpret_cast<const uint4*>(terms + (mt * 16 + g + 8 * e) * S::kPitch + k * 32 + q * 8);
      }
    }
    for (uint32_t st = first; st < end; st += 8) {
      {
        const uint32_t ahead = st + (stages - 1) * 8, to = stage == 0 ? stages - 1 : stage - 1;
        if (ahead < end) load(ahead, ring + to * kStage);
        cp_async_commit();
      }
      cp_async_wait_dynamic(stages - 1);
      const uint32_t at = ring + stage * kStage;
      stage = stage + 1 == stages ? 0 : stage + 1;
      uint4 bv[4][S::kGroups];
      if (rank != 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < S::kGroups; ++k) {
            if constexpr (RP == 16) {
              const uint2 v = lds64a(at + (j * 32 + lane) * 8);
              bv[j][k] = make_uint4(v.x, v.y, 0, 0);
            } else {
              bv[j][k] = lds128a(at + ((j * S::kGroups + k) * 32 + lane) * 16);
            }
          }
        if (rank < RP) {  // columns past the adapter's rank may hold anything
#pragma unroll
          for (int k = 0; k < S::kGroups; ++k) {
            const int32_t left = static_cast<int32_t>(rank) - static_cast<int32_t>(RP == 16 ? q * 4 : k * 32 + q * 8);
            const uint32_t m0 = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u, m1 = left >= 4 ? 0xFFFFFFFFu : left == 3 ? 0xFFFFu : 0u;
            const uint32_t m2 = left >= 6 ? 0xFFFFFFFFu : left == 5 ? 0xFFFFu : 0u, m3 = left >= 8 ? 0xFFFFFFFFu : left == 7 ? 0xFFFFu : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) bv[j][k].x &= m0, bv[j][k].y &= m1, bv[j][k].z &= m2, bv[j][k].w &= m3;
          }
        }
      }
      const uint64_t n0 = static_cast<uint64_t>(st) * 32;
      const bool inside = n0 + q * 8 < rows;
#pragma unroll
      for (int mt = 0; mt < M / 16; ++mt) {
        if (mt * 16 >= static_cast<int>(count)) break;
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
        if (rank != 0) {
#pragma unroll
          for (int t = kN - 1; t >= 0; --t) {  // small terms first
            const T* lo = terms + (t * M + mt * 16 + g) * S::kPitch;
            const T* hi = lo + 8 * S::kPitch;
#pragma unroll
            for (int k = 0; k < S::kGroups; ++k) {
              if constexpr (RP == 16) {
                const uint2 u = *reinterpret_cast<const uint2*>(lo + q * 4), v = *reinterpret_cast<const uint2*>(hi + q * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) Elem<T>::mma(acc[j], u.x, v.x, u.y, v.y, bv[j][k].x, bv[j][k].y);
              } else {
                uint4 u, v;
                if constexpr (kHold) u = held[mt][k][0], v = held[mt][k][1];
                else u = *reinterpret_cast<const uint4*>(lo + k * 32 + q * 8), v = *reinterpret_cast<const uint4*>(hi + k * 32 + q * 8);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  Elem<T>::mma(acc[j], u.x, v.x, u.y, v.y, bv[j][k].x, bv[j][k].y);
                  Elem<T>::mma(acc[j], u.z, v.z, u.w, v.w, bv[j][k].z, bv[j][k].w);
                }
              }
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = mt * 2 + e;
          if (mt * 16 + 8 * e + g >= count || !inside) continue;
          float out[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) out[x] = 0.0f;
          if (based) {
            const uint32_t from = at + 32 * kBBytes + i * kBaseVecs * 512 + lane * 16;
            const uint4 v = lds128a(from);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            if constexpr (sizeof(Y) == 4) {
              const uint4 u = lds128a(from + 512);
              const uint32_t z[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int x = 0; x < 4; ++x) out[x] = __uint_as_float(w[x]), out[4 + x] = __uint_as_float(z[x]);
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float2 h = Elem<T>::unpack(w[x]);
                out[2 * x] = h.x, out[2 * x + 1] = h.y;
              }
            }
          }
          if (rank != 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              out[2 * j] = fmaf(f[i], acc[j][2 * e], out[2 * j]);
              out[2 * j + 1] = fmaf(f[i], acc[j][2 * e + 1], out[2 * j + 1]);
            }
          }
          Y* dst = y[i] + n0;
          if constexpr (sizeof(Y) == 4) {
            reinterpret_cast<float4*>(dst)[0] = make_float4(out[0], out[1], out[2], out[3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(out[4], out[5], out[6], out[7]);
          } else {
            *reinterpret_cast<uint4*>(dst) = make_uint4(Elem<T>::pack(out[0], out[1]), Elem<T>::pack(out[2], out[3]),
                                                        Elem<T>::pack(out[4], out[5]), Elem<T>::pack(out[6], out[7]));
          }
        }
      }
    }
    cp_async_wait<0>();
  }
};

// The tile of a planned call, or the tile that a cluster finds by itself: an adapter (`adapters`:
// none), its tokens in s_token (-1 past them) and their count; false: nothing to do.
// s_info: 64 words and the votes; s_count: a word a group, up to kCountGroups (neither in planned calls).
template <int M>
__device__ __forceinline__ bool find_tile(const LoraParams& p, uint32_t tile, int32_t* s_token, uint32_t* s_info, uint32_t* s_count,
                                          uint32_t& group, uint32_t& count, uint32_t& bad) {
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (p.planned) {
    if (tile >= *p.tile_count) return false;
    const LoraTile t = p.tiles[tile];
    group = t.group;
    count = t.count;
    for (uint32_t i = tid; i < M; i += kThreads) s_token[i] = i < count ? static_cast<int32_t>(p.order[t.first + i]) : -1;
  } else if (p.tokens > kVoteTokens) {
    // tokens counted by group; the groups' tiles lie in the groups' order, their tokens in the tokens' order
    constexpr uint32_t kEach = kCountTokens / kThreads;
    uint32_t* s_votes = s_info + 64;  // members by 32 tokens
    const uint32_t groups = p.s.adapters + 1;
    if (tid < kCountGroups) s_count[tid] = 0;
    for (uint32_t i = tid; i < M; i += kThreads) s_token[i] = -1;
    uint32_t own[kEach];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint32_t t = k * kThreads + tid;
      own[k] = t < p.tokens ? group_of(p, t, bad) : groups;
    }
    if (bad != 0 && tile == 0) atomicOr(p.error, static_cast<int>(bad));
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint32_t lead = __shfl_sync(0xffffffffu, own[k], 0), same = ballot(own[k] == lead);
      if (same == 0xffffffffu) {  // a run of one adapter: 32 additions to one word would queue
        if (lane == 0 && lead < groups) atomicAdd(&s_count[lead], 32u);
      } else if (own[k] < groups) {
        atomicAdd(&s_count[own[k]], 1u);
      }
    }
    __syncthreads();
    const uint32_t tiles = tid >= groups || (tid == p.s.adapters && p.in_place) ? 0u : (s_count[tid] + M - 1) / M;
    uint32_t inc = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= static_cast<uint32_t>(o)) inc += up;
    }
    if (lane == 31) s_info[warp] = inc;
    __syncthreads();
    uint32_t at = inc - tiles, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += s_info[w];
      all += s_info[w];
    }
    if (tile >= all) return false;
    if (tile >= at && tile - at < tiles) {
      s_info[32] = tid;
      s_info[33] = (tile - at) * M;
    }
    __syncthreads();
    group = s_info[32];
    const uint32_t first = s_info[33];
    count = min(static_cast<uint32_t>(M), s_count[group] - first);
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint32_t votes = ballot(own[k] == group);
      if (lane == 0) s_votes[k * (kThreads / 32) + warp] = __popc(votes);
    }
    __syncthreads();
    const uint32_t mine = s_votes[lane];
    uint32_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= static_cast<uint32_t>(o)) before += up;
    }
    before -= mine;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint32_t votes = ballot(own[k] == group);
      const uint32_t place = __shfl_sync(0xffffffffu, before, k * (kThreads / 32) + warp) + __popc(votes & ((1u << lane) - 1u));
      if (own[k] == group && place >= first && place - first < M) s_token[place - first] = static_cast<int32_t>(k * kThreads + tid);
    }
  } else {
    // a token with a multiple of M tokens of its adapter before it begins a tile of that token and the
    // adapter's next M - 1; cluster i takes the i-th tile, in the order of their first tokens
    const bool mine = tid < p.tokens;
    const uint32_t own = mine ? group_of(p, tid, bad) : 0xFFFFu;
    if (bad != 0 && tile == 0) atomicOr(p.error, static_cast<int>(bad));
    // tokens of the same group among the earlier ones, by the votes on each bit of the group (15 at
    // most: kMaxAdapters): a warp's peers are the AND of its votes, each taken as the own bit is
    const uint32_t bits = 32 - __clz(p.s.adapters);
    uint32_t* s_votes = s_info + 64;  // [warp][16], the last its live tokens
    const uint32_t live = ballot(mine);
    uint32_t peers = live;
    for (uint32_t i = 0; i < bits; ++i) {
      const uint32_t v = ballot(own >> i & 1u);
      peers &= own >> i & 1u ? v : ~v;
      if (lane == 0) s_votes[warp * 16 + i] = v;
    }
    if (lane == 0) s_votes[warp * 16 + 15] = live;
    for (uint32_t i = tid; i < M; i += kThreads) s_token[i] = -1;
    __syncthreads();
    uint32_t before = __popc(peers & ((1u << lane) - 1u));
    for (uint32_t w = 0; w < warp && warp * 32 < p.tokens; ++w) {
      uint32_t m = s_votes[w * 16 + 15];
      for (uint32_t i = 0; i < bits; ++i) {
        const uint32_t v = s_votes[w * 16 + i];
        m &= own >> i & 1u ? v : ~v;
      }
      before += __popc(m);
    }
    const bool first = mine && before % M == 0 && !(own == p.s.adapters && p.in_place);
    const uint32_t votes = ballot(first);
    if (lane == 0) s_info[warp] = __popc(votes);
    __syncthreads();
    uint32_t index = __popc(votes & ((1u << lane) - 1u)), all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
      if (w < warp) index += s_info[w];
      all += s_info[w];
    }
    if (tile >= all) return false;
    if (first && index == tile) {
      s_info[32] = own;
      s_info[33] = before;
    }
    __syncthreads();
    group = s_info[32];
    const uint32_t place = before - s_info[33];
    const bool member = own == group && before >= s_info[33] && place < M;
    if (member) s_token[place] = static_cast<int32_t>(tid);
    count = __syncthreads_count(member);
  }
  __syncthreads();
  return true;
}

// An adapter's rank (0 for none) and factor.
__device__ __forceinline__ uint32_t adapter(const LoraParams& p, uint32_t group, float& scale, uint32_t& bad) {
  scale = 0.0f;
  if (group >= p.s.adapters) return 0;
  const int32_t v = p.s.ranks != nullptr ? p.s.ranks[group] : static_cast<int32_t>(p.s.max_rank);
  if (v < 0 || v > static_cast<int32_t>(p.s.max_rank)) bad |= HQB_DEVERR_INDEX;
  scale = p.s.scales != nullptr ? p.s.scales[group] : 1.0f;
  return v < 0 ? 0u : min(static_cast<uint32_t>(v), p.s.max_rank);
}

constexpr uint32_t kSliceWarps = 8;  // warps along the columns in lora_kernel

template <typename T, typename Y, int RP>
struct LoraSmem {
  static constexpr uint32_t kToken = 256 + kThreads / 32 * 64, kFactor = kToken + 64, kTermsAt = kFactor + 64;
  static constexpr uint32_t kSum = kTermsAt + kTerms<T, Y> * 16 * LoraShape<RP>::kPitch * 2;
  static constexpr uint32_t kPart = kSum + 16 * RP * 4;
  static constexpr uint32_t kRing = kPart + kSliceWarps * 16 * RP * 4;
  // as many stages as leave room for two CTAs an SM, else as fit one
  static constexpr uint32_t kTwo = kRing < 110 * 1024 ? (110 * 1024 - kRing) / (8 * Expand<T, Y, RP, 16>::kStage) : 0;
  static constexpr uint32_t kOne = (227 * 1024 - kRing) / (8 * Expand<T, Y, RP, 16>::kStage);
  static constexpr uint32_t kMost = kTwo > 6 ? 6 : kTwo >= 2 ? kTwo : kOne >= 2 ? 2 : 1;
  static_assert(kOne >= 1, "a stage fits");
  static_assert(kRing - kPart >= kCountGroups * 4 && kCountGroups <= kThreads, "the counts of groups lie over the partial sums");
  static_assert(kCountTokens == 32 * 32, "a lane for every 32 tokens");
  // no more than a warp has steps: what is not needed lets more CTAs share an SM
  static uint32_t stages(uint64_t rows) {
    const uint64_t steps = (rows + 32 * 8 * kCluster - 1) / (32 * 8 * kCluster);
    return steps < kMost ? static_cast<uint32_t>(steps) : kMost;
  }
  static uint32_t bytes(uint32_t stages) { return kRing + 8 * stages * Expand<T, Y, RP, 16>::kStage; }
};

// Mathematics: t = A x (FP32 sums of exact 16-bit products), y = base + scale B t.
// Split: a cluster of 8 CTAs takes one tile of up to 16 tokens of one adapter.  First its CTAs and
// their warps divide the columns of x and A (every element of x is read once, straight into MMA
// fragments: the columns of a 32-column step may be taken in any order, so a lane's 16 bytes are
// both k-halves of two MMAs); the partial t are summed in warp order, then through distributed
// shared memory in CTA order, so the bits do not depend on timing.  Then the CTAs divide the rows
// of B and of the output.  All stages of a warp's ring but one are filled from the start, under the
// first product: one of its two steps of 32 outputs at 4096 rows of rank 16, one of six at 12288 rows of
// rank 32 with FP32 results (where two stages fit, half of each for base rows of 16 tokens).  One
// launch, no scratch, no atomics.
// Bound by latency (two trips to memory and two cluster barriers) up to a few adapters, then by the
// adapters' bytes and the waves of clusters.  Measured, B200: one token of rank 16, 4096 x 4096, FP16, 5.5 us;
// 48 tokens of 16 adapters of rank 32, 12288 x 4096, FP32 result, 12.0 us (1.8 TB/s); 777 tokens of 6 of rank 24,
// 1024 x 8192, BF16, 15.4 us.  (Three CTAs an SM at ranks up to 32, in 80 registers: 14.4 us the last one,
// but 13.7 for 12.0 us the one before.)
template <typename T, typename Y, int RP, bool VEC>
__global__ void __launch_bounds__(kThreads) lora_kernel(const __grid_constant__ LoraParams p) {
  using S = LoraShape<RP>;
  using L = LoraSmem<T, Y, RP>;
  constexpr int kN = kTerms<T, Y>;
  constexpr uint32_t M = 16;
  extern __shared__ __align__(128) uint8_t sm[];
  uint32_t* s_info = reinterpret_cast<uint32_t*>(sm);             // 64 words, the votes
  int32_t* s_token = reinterpret_cast<int32_t*>(sm + L::kToken);  // [M], -1: no row
  float* s_factor = reinterpret_cast<float*>(sm + L::kFactor);    // [M]
  T* s_terms = reinterpret_cast<T*>(sm + L::kTermsAt);            // [kN][M][kPitch]
  float* s_sum = reinterpret_cast<float*>(sm + L::kSum);          // [M][RP] this CTA's t
  float* s_part = reinterpret_cast<float*>(sm + L::kPart);        // [kSliceWarps][M][RP]
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const uint32_t cta = cluster_rank(), tile = blockIdx.x / kCluster;
  uint32_t bad = 0, group, count;
  griddep_launch_dependents();
  griddep_wait();
  if (!find_tile<M>(p, tile, s_token, s_info, reinterpret_cast<uint32_t*>(s_part), group, count, bad)) return;
  float scale;
  const uint32_t rank = adapter(p, group, scale, bad);
  if (bad != 0) atomicOr(p.error, static_cast<int>(bad));
  if (rank == 0 && p.in_place) return;
  const uint64_t cols = p.s.cols, rows = p.s.rows;
  const T* b = static_cast<const T*>(p.s.b) + static_cast<uint64_t>(min(group, p.s.adapters - 1)) * p.s.max_rank * rows;
  const uint32_t n_steps = static_cast<uint32_t>((rows + 31) / 32);
  const uint32_t n0 = static_cast<uint64_t>(n_steps) * cta / kCluster, n1 = static_cast<uint64_t>(n_steps) * (cta + 1) / kCluster;
  Expand<T, Y, RP, M> x2;
  x2.prepare(p, group, rank, count, s_token, smem_u32(sm) + L::kRing + warp * p.stages * Expand<T, Y, RP, M>::kStage, p.stages);
  if (VEC) x2.start(n0 + warp, n1);

  if (rank != 0) {
    // ---- t = A x, this CTA's columns
    const T* a = static_cast<const T*>(p.s.a) + static_cast<uint64_t>(group) * p.s.max_rank * cols;
    const T* xr[2];
    bool xl[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int32_t t = s_token[g + 8 * e];
      xl[e] = t >= 0;
      xr[e] = static_cast<const T*>(p.x) + static_cast<uint64_t>(max(t, 0)) * p.x_stride;
    }
    float acc[S::kTiles8][4];
#pragma unroll
    for (int n = 0; n < S::kTiles8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
    const uint32_t steps = static_cast<uint32_t>((cols + 31) / 32);
    const uint32_t step0 = static_cast<uint64_t>(steps) * cta / kCluster, step1 = static_cast<uint64_t>(steps) * (cta + 1) / kCluster;
    constexpr int kAhead = RP <= 32 ? 4 : RP == 64 ? 2 : 1;
    for (uint32_t st = step0 + warp; st < step1; st += kSliceWarps * kAhead) {
      uint4 xv[kAhead][2], av[kAhead][S::kTiles8];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t s = st + u * kSliceWarps;
        const uint64_t col = static_cast<uint64_t>(s) * 32 + q * 8;
        const int64_t real = s < step1 ? static_cast<int64_t>(cols) - static_cast<int64_t>(col) : 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) xv[u][e] = load8<VEC>(xr[e] + col, xl[e] ? real : 0);
#pragma unroll
        for (int n = 0; n < S::kTiles8; ++n)
          av[u][n] = load8<VEC>(a + (n * 8 + g) * cols + col, n * 8 + g < rank ? real : 0);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int n = 0; n < S::kTiles8; ++n) {
          Elem<T>::mma(acc[n], xv[u][0].x, xv[u][1].x, xv[u][0].y, xv[u][1].y, av[u][n].x, av[u][n].y);
          Elem<T>::mma(acc[n], xv[u][0].z, xv[u][1].z, xv[u][0].w, xv[u][1].w, av[u][n].z, av[u][n].w);
        }
    }
#pragma unroll
    for (int n = 0; n < S::kTiles8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(s_part + (warp * M + g + 8 * e) * RP + n * 8 + q * 2) =
            make_float2(acc[n][2 * e], acc[n][2 * e + 1]);
    __syncthreads();
    for (uint32_t i = tid; i < M * RP; i += kThreads) {
      float v = 0.0f;
#pragma unroll
      for (uint32_t k = 0; k < kSliceWarps; ++k) v += s_part[k * M * RP + i];
      s_sum[i] = v;
    }
    cluster_sync();
    // ---- sum over the CTAs; each owns 2 rows, a warp a row, and hands the row's terms and factor to
    // all of them
    if (warp < M / kCluster) {
      const uint32_t row = cta * (M / kCluster) + warp;
      constexpr int kPer = (RP + 31) / 32;
      float v[kPer];
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
      }
      const float f = split_row<T, RP, kN>(v, lane, scale, [&](int k, uint32_t r, uint16_t bits) {
        const uint32_t at = smem_u32(s_terms + (k * M + row) * S::kPitch + r);
#pragma unroll
        for (uint32_t c = 0; c < kCluster; ++c) peer_store16(peer_smem(at, c), bits);
      });
      if (lane < kCluster) peer_store(peer_smem(smem_u32(s_factor + row), lane), f);
    }
    cluster_sync();
  }
  if constexpr (VEC) {
    x2.run(n0 + warp, n1, s_terms, s_factor);
  } else {
    // ---- y = base + factor * B t element by element, this CTA's rows of B
    for (uint64_t i = static_cast<uint64_t>(n0) * 32 * count + tid; i < static_cast<uint64_t>(n1) * 32 * count; i += kThreads) {
      const uint64_t n = i / count;
      const uint32_t m = static_cast<uint32_t>(i - n * count);
      if (n >= rows) break;
      const uint64_t t = static_cast<uint64_t>(s_token[m]);
      float v = 0.0f;
      for (uint32_t r = 0; r < rank; ++r) {
        float term = 0.0f;
  #pragma unroll
        for (int k = kN - 1; k >= 0; --k) term += Elem<T>::to_float(s_terms[(k * M + m) * S::kPitch + r]);
        v = fmaf(term, Elem<T>::to_float(b[n * p.s.max_rank + r]), v);
      }
      float out = rank != 0 ? s_factor[m] * v : 0.0f;
      if constexpr (sizeof(Y) == 4) {
        if (p.base != nullptr) out += static_cast<const float*>(p.base)[t * p.base_stride + n];
        static_cast<float*>(p.y)[t * p.y_stride + n] = out;
      } else {
        if (p.base != nullptr) out += Elem<T>::to_float(static_cast<const T*>(p.base)[t * p.base_stride + n]);
        static_cast<T*>(p.y)[t * p.y_stride + n] = Elem<T>::from_float(out);
      }
    }
  }
}

// Rows of a tile of a planned call: 64, or half of that where two stages of the expand kernel's ring
// would not fit shared memory.
template <int RP, int YBytes>
constexpr int kTileRows = RP <= 32 || (RP == 64 && YBytes == 2) ? 64 : 32;
constexpr uint32_t kShrinkCols = 128, kShrinkStages = 3;

template <int RP, int M>
constexpr uint32_t kShrinkSmem = 512 + kShrinkStages * (M + RP) * kShrinkCols * 2;

// t = A x of one tile and one range of columns, FP32, to the workspace [split][tile row][RP].
// Split: 16 rows by RP / (8 / row tiles) ranks a warp; x and A come in chunks of kShrinkCols columns by
// asynchronous copies, in a ring of kShrinkStages chunks.  A lane reads 16 bytes of a row at a time (both k-halves of
// two MMAs); piece c of row r lies at c ^ 4(r & 1), which those reads meet without conflicts.
// Bound by instructions (issue slots 74 % busy before the copies' addresses left the loop, 30.8 us; since
// then 25.6 us) at 8192 tokens of rank 64 and 4096 columns, BF16; x alone would take 10.2 us from HBM.
// Tiles of 128 rows, and four warps along the columns of a chunk, were slower.
template <typename T, int RP, int M>
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  constexpr uint32_t kWM = M / 16, kWN = 8 / kWM;                 // warps along rows, along ranks
  constexpr int kNT = RP / 8 / kWN;                               // 8-rank tiles of a warp
  constexpr uint32_t kStage = (M + RP) * kShrinkCols * 2, kPieces = kShrinkCols / 8;
  extern __shared__ __align__(128) uint8_t sm[];
  int32_t* s_token = reinterpret_cast<int32_t*>(sm);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const uint32_t tile = blockIdx.x / p.splits, split = blockIdx.x - tile * p.splits;
  uint32_t bad = 0, group, count;
  griddep_launch_dependents();
  griddep_wait();
  if (!find_tile<M>(p, tile, s_token, nullptr, nullptr, group, count, bad)) return;
  float scale;
  const uint32_t rank = adapter(p, group, scale, bad);
  if (rank == 0) return;
  const uint64_t cols = p.s.cols;
  const T* a = static_cast<const T*>(p.s.a) + static_cast<uint64_t>(group) * p.s.max_rank * cols;
  const T* x = static_cast<const T*>(p.x);
  const uint32_t chunks = static_cast<uint32_t>((cols + kShrinkCols - 1) / kShrinkCols);
  const uint32_t c0 = static_cast<uint64_t>(chunks) * split / p.splits, c1 = static_cast<uint64_t>(chunks) * (split + 1) / p.splits;
  const uint32_t ring = smem_u32(sm) + 512;
  // a thread copies the same piece of every 16th row of x, then of A, of every chunk
  constexpr uint32_t kCopies = (M + RP) * kPieces / kThreads, kCopyRows = kThreads / kPieces;
  const uint32_t piece = tid % kPieces, row = tid / kPieces;
  const T* src[kCopies];
  uint32_t real = 0;  // a bit a copy
#pragma unroll
  for (uint32_t i = 0; i < kCopies; ++i) {
    const uint32_t r = i * kCopyRows + row;
    const int32_t t = r < M ? s_token[r] : r - M < rank ? static_cast<int32_t>(r - M) : -1;
    const uint64_t at = static_cast<uint64_t>(max(t, 0));
    src[i] = (r < M ? x + at * p.x_stride : a + at * cols) + piece * 8;
    real |= t >= 0 ? 1u << i : 0u;
  }
  const uint32_t dst = ring + row * (kShrinkCols * 2) + ((piece ^ ((row & 1) << 2)) << 4);
  auto load = [&](uint32_t chunk, uint32_t stage) {
    const uint32_t to = dst + stage * kStage;
    const uint64_t col = static_cast<uint64_t>(chunk) * kShrinkCols;
    const uint32_t copies = col + piece * 8 < cols ? real : 0u;
    const uint64_t off = copies != 0 ? col : 0;
#pragma unroll
    for (uint32_t i = 0; i < kCopies; ++i)
      cp_async16(to + i * kCopyRows * (kShrinkCols * 2), src[i] + off, copies >> i & 1u ? 16u : 0u);
  };
  static_assert((M + RP) * kPieces % kThreads == 0 && kCopyRows % 2 == 0 && kCopies <= 32, "whole copies");
  const uint32_t wm = warp % kWM, wn = warp / kWM;
  float acc[kNT][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
  for (uint32_t s = 0; s + 1 < kShrinkStages; ++s) {
    if (c0 + s < c1) load(c0 + s, s);
    cp_async_commit();
  }
  uint32_t stage = 0;
  for (uint32_t c = c0; c < c1; ++c) {
    cp_async_wait<kShrinkStages - 2>();
    __syncthreads();
    const uint32_t ahead = c + kShrinkStages - 1;
    if (ahead < c1) load(ahead, stage == 0 ? kShrinkStages - 1 : stage - 1);
    cp_async_commit();
    const uint32_t at = ring + stage * kStage;
    stage = stage + 1 == kShrinkStages ? 0 : stage + 1;
#pragma unroll
    for (uint32_t h = 0; h < kShrinkCols / 32; ++h) {
      const uint32_t swap = (g & 1) << 2, piece = ((h * 4 + q) ^ swap) << 4;
      const uint4 u = lds128a(at + (wm * 16 + g) * (kShrinkCols * 2) + piece);
      const uint4 v = lds128a(at + (wm * 16 + g + 8) * (kShrinkCols * 2) + piece);
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const uint4 w = lds128a(at + (M + (wn * kNT + n) * 8 + g) * (kShrinkCols * 2) + piece);
        Elem<T>::mma(acc[n], u.x, v.x, u.y, v.y, w.x, w.y);
        Elem<T>::mma(acc[n], u.z, v.z, u.w, v.w, w.z, w.w);
      }
    }
  }
  cp_async_wait<0>();
  float* to = p.inner + (static_cast<uint64_t>(split) * p.max_tiles + tile) * M * RP;
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float2*>(to + (wm * 16 + g + 8 * e) * RP + (wn * kNT + n) * 8 + q * 2) =
          make_float2(acc[n][2 * e], acc[n][2 * e + 1]);
}

template <typename T, typename Y, int RP>
struct ExpandSmem {
  static constexpr int M = kTileRows<RP, sizeof(Y)>;
  static constexpr uint32_t kToken = 0, kFactor = M * 4, kTermsAt = 2 * M * 4;
  static constexpr uint32_t kRing = kTermsAt + kTerms<T, Y> * M * LoraShape<RP>::kPitch * 2;
  static constexpr uint32_t kFit = (226 * 1024 - kRing) / (8 * Expand<T, Y, RP, M>::kStage);
  static constexpr uint32_t kStages = kFit > 4 ? 4 : kFit;
  static constexpr uint32_t kBytes = kRing + 8 * kStages * Expand<T, Y, RP, M>::kStage;
  static_assert(kStages >= 2, "a ring has two stages at least");
};

// y = base + scale B t for the tiles of a planned call: the steps of 32 outputs of all tiles in order
// are dealt to the CTAs (one an SM) in equal contiguous ranges.  At each tile's start the warps sum
// the tile's t over the column ranges in their order and split it into terms, while the ring's
// first copies of B and base are under way.
// Two warps a scheduler wait for their own instructions more than for HBM: 11008 outputs of 8192 tokens,
// rank 64, BF16, take 80 us (4.5 TB/s of base and y), of which the bytes need 55.  Rings of more
// stages, 16 warps and tiles of 128 rows were slower.
template <typename T, typename Y, int RP>
__global__ void __launch_bounds__(kThreads) lora_expand_kernel(const __grid_constant__ LoraParams p) {
  using S = LoraShape<RP>;
  using L = ExpandSmem<T, Y, RP>;
  constexpr int M = L::M, kN = kTerms<T, Y>, kPer = (RP + 31) / 32, kRowsEach = M / 8;
  extern __shared__ __align__(128) uint8_t sm[];
  int32_t* s_token = reinterpret_cast<int32_t*>(sm + L::kToken);
  float* s_factor = reinterpret_cast<float*>(sm + L::kFactor);
  T* s_terms = reinterpret_cast<T*>(sm + L::kTermsAt);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t bad = 0;
  griddep_launch_dependents();
  griddep_wait();
  const uint32_t steps = static_cast<uint32_t>((p.s.rows + 31) / 32);
  const uint64_t units = static_cast<uint64_t>(*p.tile_count) * steps;
  uint64_t u = units * blockIdx.x / gridDim.x;
  const uint64_t u1 = units * (blockIdx.x + 1) / gridDim.x;
  while (u < u1) {
    const uint32_t tile = static_cast<uint32_t>(u / steps), first = static_cast<uint32_t>(u - static_cast<uint64_t>(tile) * steps);
    const uint32_t end = static_cast<uint32_t>(u1 - u < steps - first ? first + (u1 - u) : steps);
    u += end - first;
    __syncthreads();  // the last tile's terms and tokens have been read
    uint32_t group, count;
    find_tile<M>(p, tile, s_token, nullptr, nullptr, group, count, bad);
    float scale;
    const uint32_t rank = adapter(p, group, scale, bad);
    Expand<T, Y, RP, M> x2;
    x2.prepare(p, group, rank, count, s_token, smem_u32(sm) + L::kRing + warp * L::kStages * Expand<T, Y, RP, M>::kStage, L::kStages);
    x2.start(first + warp, end);
    if (rank != 0) {
      float v[kRowsEach][kPer];
#pragma unroll
      for (int r = 0; r < kRowsEach; ++r)
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[r][i] = 0.0f;
      const float* from = p.inner + (static_cast<uint64_t>(tile) * M + warp * kRowsEach) * RP + lane;
#pragma unroll 2
      for (uint32_t sp = 0; sp < p.splits; ++sp, from += static_cast<uint64_t>(p.max_tiles) * M * RP)
#pragma unroll
        for (int r = 0; r < kRowsEach; ++r)
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (i * 32 + lane < rank) v[r][i] += from[r * RP + i * 32];
#pragma unroll
      for (int r = 0; r < kRowsEach; ++r) {
        const uint32_t row = warp * kRowsEach + r;
        const float f = split_row<T, RP, kN>(v[r], lane, scale, [&](int k, uint32_t x, uint16_t bits) {
          reinterpret_cast<uint16_t*>(s_terms)[(k * M + row) * S::kPitch + x] = bits;
        });
        if (lane == 0) s_factor[row] = f;
      }
    }
    __syncthreads();
    x2.run(first + warp, end, s_terms, s_factor);
  }
  if (bad != 0) atomicOr(p.error, static_cast<int>(bad));
}

// Groups the tokens by adapter: counts, offsets, then each token to its group's next place.  The
// order within a group may change between runs; a token's output does not depend on it.  One CTA: bound by
// latency (two passes over the ids); 8192 tokens 8 us, of which the kernels after it wait for all.
__global__ void __launch_bounds__(1024) lora_plan_kernel(const __grid_constant__ LoraParams p) {
  extern __shared__ uint32_t count[];  // [groups], then the groups' next places
  __shared__ uint32_t red[2][32];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, groups = p.s.adapters + 1;
  uint32_t bad = 0;
  griddep_launch_dependents();
  griddep_wait();
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

// B in rows of a multiple of 8 ranks, zeros after the last: 16-byte copies need such rows, and without them
// the second product goes element by element.  Bound by the bytes of B, read and written once.
__global__ void __launch_bounds__(256) lora_lay_kernel(const __grid_constant__ LoraParams p) {
  const uint32_t pieces = p.pitch / 8;
  const uint64_t total = static_cast<uint64_t>(p.s.adapters) * p.s.rows * pieces;
  griddep_launch_dependents();
  griddep_wait();
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
    const uint64_t row = i / pieces;
    const uint32_t r = static_cast<uint32_t>(i - row * pieces) * 8;
    const uint16_t* src = static_cast<const uint16_t*>(p.s.b) + row * p.s.max_rank;
    uint16_t v[8];
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) v[k] = r + k < p.s.max_rank ? src[r + k] : 0;
    static_cast<uint4*>(p.laid)[i] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}

uint32_t padded_rank(uint32_t r) { return r <= 16 ? 16u : r <= 32 ? 32u : r <= 64 ? 64u : 128u; }

struct Layout {
  uint64_t tiles, order, inner, total;
  uint32_t max_tiles, splits;
};

// tile_rows 16: the tiles of lora_kernel, which keeps t to itself.
Layout layout(const hqb_lora_set* s, uint32_t tokens, uint32_t tile_rows) {
  Layout l{};
  // every group may end in a partly filled tile
  const uint64_t groups = static_cast<uint64_t>(s->adapters) + 1;
  l.max_tiles = static_cast<uint32_t>(tokens / tile_rows + (groups < tokens ? groups : tokens));
  // column ranges: two CTAs an SM at about the usual tiles, 256 columns a range at least
  const uint32_t usual = tokens / tile_rows + 1;
  uint32_t splits = usual < 296 ? 296 / usual : 1;
  const uint64_t most = (s->cols + 255) / 256;
  splits = splits > most ? static_cast<uint32_t>(most) : splits;
  const uint32_t few = groups >= 512 ? 1u : static_cast<uint32_t>(512 / groups);
  splits = splits > few ? few : splits;
  l.splits = splits > 16 ? 16 : splits;
  l.tiles = 512;
  l.order = l.tiles + round_up(static_cast<uint64_t>(l.max_tiles) * sizeof(LoraTile), 256);
  l.inner = l.order + round_up(static_cast<uint64_t>(tokens) * 4, 256);
  l.total = l.inner;
  if (tile_rows != 16) {
    // splits * max_tiles at most: splits * (tokens / tile_rows) <= 296 where splits > 1, and splits *
    // groups <= max(512, groups).  Room for that, so that what a call needs never shrinks with its tokens.
    const uint64_t cut = 296 + (groups > 512 ? groups : 512), tiles = cut > l.max_tiles ? cut : l.max_tiles;
    l.total += round_up(tiles * tile_rows * padded_rank(s->max_rank) * 4, 256);
  }
  return l;
}

// Whether a call lays B out: rows that no 16-byte copy fits, and tokens enough to pay for all adapters.  B200, us,
// laid out / element by element, FP16, rank 27, 4096 x 4096: 1 token of 4 adapters 7.6 / 13.0; 48 of 8 9.4 / 28.5;
// 256 of 130 45 / 115; 300 of 8 11.0 / 71; 2000 of 200 84 / 545; 1 of 8 at rank 57 and 11008 rows 14.0 / 22.2.
bool lays_out(const hqb_lora_set* s, uint32_t tokens) {
  return (s->max_rank & 7u) != 0 && s->adapters <= kLayAdapters + tokens / 2;
}
uint64_t laid_bytes(const hqb_lora_set* s) {
  return round_up(static_cast<uint64_t>(s->adapters) * s->rows * round_up(s->max_rank, 8) * 2, 256);
}

bool set_ok(const hqb_lora_set* s) {
  if (s == nullptr || s->rows == 0 || s->cols == 0 || s->adapters == 0 || s->max_rank == 0 || s->max_rank > HQB_MAX_RANK)
    return false;
  if (s->rows > 0x7FFFFFFFull || s->cols > 0x7FFFFFFFull) return false;
  return s->dtype == HQB_F16 || s->dtype == HQB_BF16;
}

// One launch with `smem` bytes, as clusters of `cluster` CTAs.
template <typename K>
cudaError_t launch(K kernel, DeviceOnce& once, uint32_t grid, uint32_t smem, uint32_t cluster, const LoraParams& p,
                   cudaStream_t st) {
  const cudaError_t e = allow_dynamic_smem(once, reinterpret_cast<const void*>(kernel), smem);
  return e != cudaSuccess ? e : launch_dependent(kernel, dim3(grid), kThreads, smem, cluster, st, p);
}

template <typename T, typename Y, int RP, bool VEC>
cudaError_t launch_tile(LoraParams p, uint32_t tiles, cudaStream_t st) {
  using L = LoraSmem<T, Y, RP>;
  static DeviceOnce once;
  p.stages = L::stages(p.s.rows);
  const cudaError_t e =
      allow_dynamic_smem(once, reinterpret_cast<const void*>(lora_kernel<T, Y, RP, VEC>), L::bytes(L::kMost));
  if (e != cudaSuccess) return e;
  return launch_dependent(lora_kernel<T, Y, RP, VEC>, dim3(tiles * kCluster), kThreads, L::bytes(p.stages), kCluster, st, p);
}

template <typename T, typename Y, int RP>
cudaError_t launch_rank(const LoraParams& p, uint32_t tiles, int sms, cudaStream_t st) {
  if (p.tile_rows == 16) return launch_tile<T, Y, RP, true>(p, tiles, st);
  static DeviceOnce once_shrink, once_expand;
  constexpr int M = kTileRows<RP, sizeof(Y)>;
  const cudaError_t e = launch(lora_shrink_kernel<T, RP, M>, once_shrink, tiles * p.splits, kShrinkSmem<RP, M>, 1, p, st);
  if (e != cudaSuccess) return e;
  return launch(lora_expand_kernel<T, Y, RP>, once_expand, static_cast<uint32_t>(sms), ExpandSmem<T, Y, RP>::kBytes, 1, p, st);
}

template <typename T, typename Y>
cudaError_t launch_lora(const LoraParams& p, bool vec, uint32_t tiles, int sms, cudaStream_t st) {
  if (!vec) return launch_tile<T, Y, 128, false>(p, tiles, st);
  switch (padded_rank(p.s.max_rank)) {
    case 16: return launch_rank<T, Y, 16>(p, tiles, sms, st);
    case 32: return launch_rank<T, Y, 32>(p, tiles, sms, st);
    case 64: return launch_rank<T, Y, 64>(p, tiles, sms, st);
    default: return launch_rank<T, Y, 128>(p, tiles, sms, st);
  }
}

uint32_t planned_rows(const hqb_lora_set* s, uint32_t tokens, bool vec, bool wide_y) {
  if (!vec || static_cast<uint64_t>(tokens) * padded_rank(s->max_rank) <= kClusterWork) return 16;
  switch (padded_rank(s->max_rank)) {
    case 16: return wide_y ? kTileRows<16, 4> : kTileRows<16, 2>;
    case 32: return wide_y ? kTileRows<32, 4> : kTileRows<32, 2>;
    case 64: return wide_y ? kTileRows<64, 4> : kTileRows<64, 2>;
    default: return wide_y ? kTileRows<128, 4> : kTileRows<128, 2>;
  }
}

}  // namespace
}  // namespace hqb

using namespace hqb;

extern "C" {

HQB_API uint64_t hqb_lora_workspace_bytes(const hqb_lora_set* s, uint32_t tokens, int device) {
  (void)device;
  if (!set_ok(s) || tokens > 0x7FFFFFFFu) return 0;
  const uint64_t laid = lays_out(s, tokens) ? laid_bytes(s) : 0;
  if (tokens <= kVoteTokens) return 256 + laid;
  // the call's kernels depend on its alignment and output type too: room for any
  uint64_t most = layout(s, tokens, 16).total;
  for (const bool wide_y : {false, true}) {
    const uint64_t n = layout(s, tokens, planned_rows(s, tokens, true, wide_y)).total;
    most = n > most ? n : most;
  }
  return most + laid;
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
  const uint64_t sizes = s->cols | s->rows | x_stride | y_stride | (base != nullptr ? base_stride : 0);
  const bool fits = (addresses & 15u) == 0 && (sizes & 7u) == 0, lay = fits && lays_out(s, tokens);
  const bool vec = fits && (lay || (s->max_rank & 7u) == 0);
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
  p.in_place = base == y ? 1u : 0u;
  p.tile_rows = tokens > kVoteTokens ? planned_rows(s, tokens, vec, y_dtype == HQB_F32) : 16u;
  p.planned = tokens > kVoteTokens && (p.tile_rows != 16 || tokens > kCountTokens || s->adapters >= kCountGroups) ? 1u : 0u;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.error = reinterpret_cast<int*>(ws);
  cudaStream_t st = as_stream(stream);
  // tiles at most: every group may end in a partly filled one
  const uint32_t groups = s->adapters + 1, full = tokens / 16 + groups;
  uint32_t tiles = tokens < full ? tokens : full;
  p.pitch = s->max_rank;
  if (lay) {
    p.pitch = static_cast<uint32_t>(round_up(s->max_rank, 8));
    p.laid = ws + hqb_lora_workspace_bytes(s, tokens, 0) - laid_bytes(s);
    const uint64_t blocks = (static_cast<uint64_t>(s->adapters) * s->rows * (p.pitch / 8) + 255) / 256;
    const cudaError_t e = launch_dependent(lora_lay_kernel, dim3(static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16)),
                                           256, 0, 1, st, p);
    if (e != cudaSuccess) return e;
    p.s.b = p.laid;
  }
  if (p.planned) {
    const Layout l = layout(s, tokens, p.tile_rows);
    p.tile_count = reinterpret_cast<uint32_t*>(ws + 256);
    p.tiles = reinterpret_cast<LoraTile*>(ws + l.tiles);
    p.order = reinterpret_cast<uint32_t*>(ws + l.order);
    p.inner = reinterpret_cast<float*>(ws + l.inner);
    p.max_tiles = l.max_tiles;
    p.splits = l.splits;
    tiles = l.max_tiles;
    if (tiles > 0x7FFFFFFFu / 16) return HQB_ERR_UNSUPPORTED;
    static DeviceOnce once;
    cudaError_t e = allow_dynamic_smem(once, reinterpret_cast<const void*>(lora_plan_kernel), (kMaxAdapters + 1) * 4);
    if (e == cudaSuccess) e = launch_dependent(lora_plan_kernel, dim3(1), 1024, (s->adapters + 1) * 4, 1, st, p);
    if (e != cudaSuccess) return e;
  }
  int device = 0;
  const cudaError_t e3 = cudaGetDevice(&device);
  if (e3 != cudaSuccess) return e3;
  const int sms = device_sm_count(device);
  if (sms <= 0) return cudaErrorInvalidDevice;
  if (s->dtype == HQB_F16)
    return y_dtype == HQB_F32 ? launch_lora<__half, float>(p, vec, tiles, sms, st)
                              : launch_lora<__half, __half>(p, vec, tiles, sms, st);
  return y_dtype == HQB_F32 ? launch_lora<__nv_bfloat16, float>(p, vec, tiles, sms, st)
                            : launch_lora<__nv_bfloat16, __nv_bfloat16>(p, vec, tiles, sms, st);
}

}  // extern "C"
