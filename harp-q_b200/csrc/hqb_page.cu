// Paged-cache operators of a decode step.
//   page_plan_kernel     request lengths -> token starts, page tables, slots, positions, tree masks
//   cache_append_kernel  rows of new keys and values -> cache slots
#include <cuda_runtime.h>

#include <type_traits>

#include "hqb_internal.h"
#include "hqb_serve.cuh"

namespace hqb {
namespace {

constexpr uint32_t kPlanThreads = 256;
constexpr uint32_t kPlanWords = HQB_MAX_NODES / 32;

// Exclusive sum of v over the CTA's threads, plus *carry; *carry grows by the sum of all.
// 64-bit: a sum of garbage lengths must not wrap into a valid-looking start.
__device__ __forceinline__ uint64_t block_exclusive_sum(uint64_t v, uint64_t* carry, uint64_t* red) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= static_cast<uint32_t>(o)) inc += up;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  uint64_t before = *carry, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  __syncthreads();
  *carry += all;
  return before + inc - v;
}

// Every CTA owns an equal range of the step's tokens and scans the requests up to it by itself
// (256 at a time: the lengths come from L2, a scan is two shuffles rounds and a shared-memory
// round), so the whole plan is one launch without any hand-over between CTAs.  A token finds
// its request by a binary search of the chunk's starts.  CTA 0 also writes the per-request
// outputs.  New page columns are written by the first token in them.
// What bounds it: latency (launch, three dependent loads, scan, search, a load per ancestor), not bytes.
// Measured, B200: 64 requests of one token 3.1 us; 512 trees of up to 64 nodes 7.3 us, in a CUDA graph.
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const __grid_constant__ hqb_page_plan_args a,
                                                                 uint32_t per_cta) {
  __shared__ uint64_t red[kPlanThreads / 32];
  __shared__ uint32_t s_start[kPlanThreads + 1], s_ctx[kPlanThreads], s_held[kPlanThreads], s_fresh[kPlanThreads];
  const uint32_t tid = threadIdx.x;
  griddep_launch_dependents();
  griddep_wait();
  const uint32_t t0 = min(a.token_capacity, blockIdx.x * per_cta), t1 = min(a.token_capacity, t0 + per_cta);
  const bool scribe = blockIdx.x == 0, paged = a.tables != nullptr;
  uint32_t bad = 0;
  uint64_t head = 0;
  if (paged) {
    const int32_t h = *a.free_head;
    if (h < 0 || static_cast<uint32_t>(h) > a.free_count) bad |= HQB_DEVERR_INDEX;
    head = h < 0 ? 0u : min(static_cast<uint32_t>(h), a.free_count);
  }
  uint64_t tokens = 0, fresh_all = 0;  // before the chunk
  for (uint32_t r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
    const uint32_t r = r0 + tid;
    const bool live = r < a.requests;
    int32_t ctx = live ? a.context_lens[r] : 0, n = live ? a.new_lens[r] : 0;
    if (ctx < 0 || n < 0) bad |= HQB_DEVERR_INDEX;
    ctx = max(ctx, 0);
    n = max(n, 0);
    const uint64_t first = block_exclusive_sum(static_cast<uint64_t>(n), &tokens, red);
    const uint64_t cap = a.token_capacity;
    const uint32_t start = static_cast<uint32_t>(first < cap ? first : cap);
    const uint32_t end = static_cast<uint32_t>(first + n < cap ? first + n : cap);
    if (first + n > cap) bad |= HQB_DEVERR_INDEX;
    const uint32_t filled = (static_cast<uint32_t>(ctx) + a.page_size - 1) / a.page_size;
    uint32_t held = filled, fresh = 0;
    if (paged && live) {
      if (a.held != nullptr) {
        const int32_t v = a.held[r];
        if (v < 0) bad |= HQB_DEVERR_INDEX;
        held = static_cast<uint32_t>(max(v, 0));
      }
      if (held > a.table_stride) {
        bad |= HQB_DEVERR_INDEX;
        held = a.table_stride;
      }
      if (held < filled) bad |= HQB_DEVERR_INDEX;
      if (end > start) {
        const uint64_t need = (static_cast<uint64_t>(ctx) + (end - start) + a.page_size - 1) / a.page_size;
        if (need > a.table_stride) bad |= HQB_DEVERR_PAGES;
        const uint32_t fit = static_cast<uint32_t>(need < a.table_stride ? need : a.table_stride);
        fresh = fit > held ? fit - held : 0u;
      }
    }
    uint64_t fresh_first = 0;
    if (paged) fresh_first = block_exclusive_sum(fresh, &fresh_all, red);
    // the first free page of the request; one past the free pages reads as "none" below
    const uint64_t page_first = head + fresh_first;
    s_start[tid] = start;
    s_ctx[tid] = static_cast<uint32_t>(ctx);
    s_held[tid] = held;
    s_fresh[tid] = static_cast<uint32_t>(page_first < a.free_count ? page_first : a.free_count);
    if (tid == kPlanThreads - 1) s_start[kPlanThreads] = end;
    if (scribe && live) {
      a.starts[r] = static_cast<int32_t>(start);
      if (r == a.requests - 1) a.starts[a.requests] = static_cast<int32_t>(end);
      const uint64_t left = page_first < a.free_count ? a.free_count - page_first : 0;
      if (paged && left < fresh) bad |= HQB_DEVERR_PAGES;
      if (paged && a.held_out != nullptr)
        a.held_out[r] = static_cast<int32_t>(held + (left < fresh ? static_cast<uint32_t>(left) : fresh));
    }
    __syncthreads();
    const uint32_t c0 = max(t0, s_start[0]), c1 = min(t1, s_start[kPlanThreads]);
    for (uint32_t t = c0 + tid; t < c1; t += kPlanThreads) {
      // the last request whose start is not past t (requests without tokens share a start and
      // come before the one that has them)
      uint32_t lo = 0, hi = kPlanThreads;
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (s_start[mid] <= t) lo = mid; else hi = mid;
      }
      const uint32_t rr = r0 + lo, node = t - s_start[lo], ctx_r = s_ctx[lo];
      if (a.token_request != nullptr) a.token_request[t] = static_cast<int32_t>(rr);
      uint32_t depth = node;
      if (a.parents != nullptr) {
        const bool given = t < a.parent_count;  // then its ancestors are too
        if (!given) bad |= HQB_DEVERR_INDEX;
        const int32_t* parent = a.parents + s_start[lo];
        uint32_t words[kPlanWords];
#pragma unroll
        for (uint32_t w = 0; w < kPlanWords; ++w) words[w] = 0;
        depth = 0;
        uint32_t at = node;
        int32_t up = given ? parent[at] : -1;
        for (;;) {
          if (a.mask != nullptr && (at >> 5) >= a.mask_words) bad |= HQB_DEVERR_INDEX;
#pragma unroll
          for (uint32_t w = 0; w < kPlanWords; ++w) words[w] |= w == (at >> 5) ? 1u << (at & 31) : 0u;
          if (up < -1 || up >= static_cast<int32_t>(at)) bad |= HQB_DEVERR_INDEX;
          if (up < 0 || up >= static_cast<int32_t>(at)) break;  // a root; parents come strictly earlier
          at = static_cast<uint32_t>(up);
          up = parent[at];
          ++depth;
        }
        if (a.mask != nullptr) {
          uint32_t* row = a.mask + static_cast<uint64_t>(t) * a.mask_words;
#pragma unroll
          for (uint32_t w = 0; w < kPlanWords; ++w)
            if (w < a.mask_words) row[w] = words[w];
        }
      }
      if (a.positions != nullptr) a.positions[t] = static_cast<int32_t>(ctx_r + depth);
      if (paged) {
        const uint32_t place = ctx_r + node, column = place / a.page_size, inside = place - column * a.page_size;
        int32_t* row = a.tables + static_cast<uint64_t>(rr) * a.table_stride;
        int32_t page = -1;
        if (column < a.table_stride) {
          const uint32_t held_r = s_held[lo];
          if (column < held_r) {
            page = row[column];
          } else {
            // columns before the first token's (a request that holds too few) are its to write
            for (uint32_t c = node == 0 ? held_r : column; c <= column; ++c) {
              const uint64_t at = static_cast<uint64_t>(s_fresh[lo]) + (c - held_r);
              if (at >= a.free_count) break;
              const int32_t got = a.free_pages[at];
              if (c == column) page = got;
              if (inside == 0 || node == 0) row[c] = got;
            }
          }
        }
        if (page < 0 || static_cast<uint32_t>(page) >= a.num_pages) {
          bad |= HQB_DEVERR_PAGES;
          page = -1;
        }
        if (a.slots != nullptr)
          a.slots[t] = page < 0 ? -1 : static_cast<int32_t>(static_cast<uint32_t>(page) * a.page_size + inside);
      }
    }
    __syncthreads();
    if (!scribe && tokens >= t1) break;
  }
  if (scribe && tid == 0) {
    if (a.requests == 0) a.starts[0] = 0;
    if (paged && a.free_head_out != nullptr) {
      const uint64_t h = head + fresh_all;
      *a.free_head_out = static_cast<int32_t>(h < a.free_count ? h : a.free_count);
    }
  }
  for (uint64_t t = (tokens > t0 ? tokens : t0) + tid; t < t1; t += kPlanThreads) {
    if (a.token_request != nullptr) a.token_request[t] = -1;
    if (a.positions != nullptr) a.positions[t] = -1;
    if (paged && a.slots != nullptr) a.slots[t] = -1;
    if (a.mask != nullptr)
      for (uint32_t w = 0; w < a.mask_words; ++w) a.mask[t * a.mask_words + w] = 0;
  }
  if (bad != 0 && a.flags != nullptr) atomicOr(a.flags, static_cast<int>(bad));
}

struct AppendParams {
  const uint8_t* src[2];
  uint8_t* dst[2];
  const int32_t* rows;
  const int32_t* slots;
  int* flags;
  uint64_t token_stride, head_stride;             // source, elements
  uint64_t c_page, c_token, c_head;               // cache, elements
  uint32_t count, source_rows, heads, dim, page_size, num_slots;
};

// One element of the source as the cache's type: the same bits where the types agree, else one
// rounding from FP32 (which holds every 16-bit value).
template <typename S, typename T>
struct AppendElem;
template <typename T>
struct AppendElem<T, T> {
  static __device__ __forceinline__ T get(T v) { return v; }
};
template <typename T>
struct AppendElem<float, T> {
  static __device__ __forceinline__ T get(float v) { return Elem<T>::from_float(v); }
};
template <>
struct AppendElem<__half, __nv_bfloat16> {
  static __device__ __forceinline__ __nv_bfloat16 get(__half v) { return __float2bfloat16_rn(__half2float(v)); }
};
template <>
struct AppendElem<__nv_bfloat16, __half> {
  static __device__ __forceinline__ __half get(__nv_bfloat16 v) { return __float2half_rn(__bfloat162float(v)); }
};

// W consecutive elements a thread: 8 (16 bytes written, 16 or 32 read) where sizes, strides and
// addresses are multiples of that, else 1.  A thread moves the same piece of k and of v, so two
// independent copies are in flight per thread.  Bound by the copy itself (HBM, or L2 at the few
// rows of a decode step, where the launch dominates).  Measured, B200: 8192 picked rows of 8 heads of 128,
// BF16, 12.5 us over buffers larger than L2 (5.4 TB/s; a plain copy reaches 6.55); 16 rows of 32 heads 1.6 us.
template <typename S, typename T, int W>
__global__ void __launch_bounds__(256) cache_append_kernel(const __grid_constant__ AppendParams p) {
  const uint32_t pieces = p.dim / W, row_pieces = pieces * p.heads;
  const uint64_t total = static_cast<uint64_t>(p.count) * row_pieces;
  uint32_t bad = 0;
  griddep_launch_dependents();
  griddep_wait();
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
    const uint32_t entry = static_cast<uint32_t>(i / row_pieces);
    const uint32_t j = static_cast<uint32_t>(i - static_cast<uint64_t>(entry) * row_pieces);
    const uint32_t head = j / pieces, d = (j - head * pieces) * W;
    const int32_t slot = p.slots[entry], row = p.rows != nullptr ? p.rows[entry] : static_cast<int32_t>(entry);
    if (slot < 0 || row < 0) continue;
    if (static_cast<uint32_t>(slot) >= p.num_slots) { bad |= HQB_DEVERR_PAGES; continue; }
    if (static_cast<uint32_t>(row) >= p.source_rows) { bad |= HQB_DEVERR_INDEX; continue; }
    const uint32_t page = static_cast<uint32_t>(slot) / p.page_size, token = static_cast<uint32_t>(slot) - page * p.page_size;
    const uint64_t from = row * p.token_stride + head * p.head_stride + d;
    const uint64_t to = page * p.c_page + token * p.c_token + head * p.c_head + d;
    if constexpr (W == 8 && sizeof(S) == 2) {
      uint4 v[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) v[s] = *reinterpret_cast<const uint4*>(p.src[s] + from * 2);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if constexpr (!std::is_same<S, T>::value) {
          const S* e = reinterpret_cast<const S*>(&v[s]);
          alignas(16) T o[8];
#pragma unroll
          for (int w = 0; w < 8; ++w) o[w] = AppendElem<S, T>::get(e[w]);
          v[s] = *reinterpret_cast<const uint4*>(o);
        }
        *reinterpret_cast<uint4*>(p.dst[s] + to * 2) = v[s];
      }
    } else if constexpr (W == 8) {
      float4 v[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        v[s][0] = reinterpret_cast<const float4*>(p.src[s] + from * 4)[0];
        v[s][1] = reinterpret_cast<const float4*>(p.src[s] + from * 4)[1];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint4 o;
        o.x = Elem<T>::pack(v[s][0].x, v[s][0].y);
        o.y = Elem<T>::pack(v[s][0].z, v[s][0].w);
        o.z = Elem<T>::pack(v[s][1].x, v[s][1].y);
        o.w = Elem<T>::pack(v[s][1].z, v[s][1].w);
        *reinterpret_cast<uint4*>(p.dst[s] + to * 2) = o;
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        reinterpret_cast<T*>(p.dst[s])[to] = AppendElem<S, T>::get(reinterpret_cast<const S*>(p.src[s])[from]);
    }
  }
  if (bad != 0 && p.flags != nullptr) atomicOr(p.flags, static_cast<int>(bad));
}

template <typename S, typename T>
cudaError_t launch_append(const AppendParams& p, bool wide, cudaStream_t st) {
  const uint64_t total = static_cast<uint64_t>(p.count) * p.heads * (wide ? p.dim / 8 : p.dim);
  const uint64_t blocks = (total + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16);
  return launch_dependent(wide ? cache_append_kernel<S, T, 8> : cache_append_kernel<S, T, 1>, dim3(grid), 256, 0, 1, st, p);
}

}  // namespace

bool paged_cache_ok(const hqb_paged_cache* c) {
  if (c == nullptr || c->kv_heads == 0 || c->head_dim == 0 || c->page_size == 0 || c->num_pages == 0) return false;
  if (c->dtype != HQB_F16 && c->dtype != HQB_BF16) return false;
  // slots are int32
  return static_cast<uint64_t>(c->num_pages) * c->page_size <= 0x7FFFFFFFull;
}

}  // namespace hqb

using namespace hqb;

extern "C" {

HQB_API int hqb_page_plan(const hqb_page_plan_args* a, void* stream) {
  if (a == nullptr || a->starts == nullptr) return HQB_ERR_INVALID;
  if (a->requests > 0 && (a->context_lens == nullptr || a->new_lens == nullptr)) return HQB_ERR_INVALID;
  if (a->requests > 0x7FFFFFFEu || a->token_capacity > 0x7FFFFFFFu) return HQB_ERR_INVALID;
  if (a->page_size == 0) return HQB_ERR_INVALID;
  if (a->mask != nullptr && (a->parents == nullptr || a->mask_words == 0 || a->mask_words > HQB_MAX_NODES / 32))
    return HQB_ERR_INVALID;
  if (a->tables != nullptr) {
    if (a->table_stride == 0 || a->num_pages == 0 || a->free_head == nullptr || a->free_count > 0x7FFFFFFFu ||
        (a->free_count > 0 && a->free_pages == nullptr) ||
        static_cast<uint64_t>(a->num_pages) * a->page_size > 0x7FFFFFFFull)
      return HQB_ERR_INVALID;
    // every CTA reads the counts while one writes them
    if (a->held_out != nullptr && a->held_out == a->held) return HQB_ERR_INVALID;
    if (a->free_head_out == a->free_head) return HQB_ERR_INVALID;
  } else if (a->slots != nullptr || a->held_out != nullptr || a->free_head_out != nullptr) {
    return HQB_ERR_INVALID;
  }
  const cudaError_t prior = take_prior_error();
  if (prior != cudaSuccess) return prior;
  uint32_t grid = (a->token_capacity + kPlanThreads - 1) / kPlanThreads;
  grid = grid < 1 ? 1 : grid > 148 ? 148 : grid;
  const uint32_t per_cta = (a->token_capacity + grid - 1) / grid;
  return launch_dependent(page_plan_kernel, dim3(grid), kPlanThreads, 0, 1, as_stream(stream), *a, per_cta);
}

HQB_API int hqb_cache_append(const hqb_paged_cache* c, const void* k, const void* v, int dtype, uint64_t token_stride,
                             uint64_t head_stride, uint32_t source_rows, const int32_t* rows, const int32_t* slots,
                             uint32_t count, int* flags, void* stream) {
  if (!paged_cache_ok(c) || c->k == nullptr || c->v == nullptr) return HQB_ERR_INVALID;
  if (dtype != HQB_F16 && dtype != HQB_BF16 && dtype != HQB_F32) return HQB_ERR_INVALID;
  if (count > 0x7FFFFFFFu || source_rows > 0x7FFFFFFFu) return HQB_ERR_INVALID;
  if (count > 0 && (k == nullptr || v == nullptr || slots == nullptr)) return HQB_ERR_INVALID;
  const cudaError_t prior = take_prior_error();
  if (prior != cudaSuccess) return prior;
  if (count == 0) return HQB_OK;
  AppendParams p{};
  p.src[0] = static_cast<const uint8_t*>(k);
  p.src[1] = static_cast<const uint8_t*>(v);
  p.dst[0] = static_cast<uint8_t*>(c->k);
  p.dst[1] = static_cast<uint8_t*>(c->v);
  p.rows = rows;
  p.slots = slots;
  p.flags = flags;
  p.token_stride = token_stride;
  p.head_stride = head_stride;
  p.c_page = c->page_stride;
  p.c_token = c->token_stride;
  p.c_head = c->head_stride;
  p.count = count;
  p.source_rows = source_rows;
  p.heads = c->kv_heads;
  p.dim = c->head_dim;
  p.page_size = c->page_size;
  p.num_slots = c->num_pages * c->page_size;
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                              reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v);
  const uint64_t strides = token_stride | head_stride | c->page_stride | c->token_stride | c->head_stride;
  const bool wide = (addresses & 15u) == 0 && (strides & 7u) == 0 && (c->head_dim & 7u) == 0;
  cudaStream_t st = as_stream(stream);
  if (c->dtype == HQB_F16) {
    if (dtype == HQB_F16) return launch_append<__half, __half>(p, wide, st);
    if (dtype == HQB_BF16) return launch_append<__nv_bfloat16, __half>(p, wide, st);
    return launch_append<float, __half>(p, wide, st);
  }
  if (dtype == HQB_BF16) return launch_append<__nv_bfloat16, __nv_bfloat16>(p, wide, st);
  if (dtype == HQB_F16) return launch_append<__half, __nv_bfloat16>(p, wide, st);
  return launch_append<float, __nv_bfloat16>(p, wide, st);
}

}  // extern "C"
