// Host-side helpers shared by the library's translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "harpq_b200.h"

namespace hqb {

inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

inline bool mul_ok(uint64_t a, uint64_t b, uint64_t* out) {
  if (a != 0 && b > UINT64_MAX / a) return false;
  *out = a * b;
  return true;
}

inline uint64_t round_up(uint64_t v, uint64_t a) { return (v + a - 1) / a * a; }

// Returns a pending CUDA error without clearing anything else; the caller
// propagates it instead of launching (reference: progressive_gemv.cu:427-433).
inline cudaError_t take_prior_error() { return cudaGetLastError(); }

int device_sm_count(int device);

// Devices (bits) on which a kernel's dynamic shared memory limit has been raised.
using DeviceOnce = std::atomic<uint64_t>;

// Raises a kernel's dynamic shared memory limit on the current device, once per device.
inline cudaError_t allow_dynamic_smem(DeviceOnce& done, const void* kernel, uint32_t bytes) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// Launches a kernel as a programmatic dependent of the one before it in the stream: its CTAs may
// start while that one ends.  Only for kernels that run griddepcontrol.wait before their first
// access to global memory (in at least one thread of a grid that would otherwise end early), and that
// read by plain loads: the read-only path (__ldg) is for data that nobody writes while the kernel
// runs, and its loads may move above the wait; the kernel before may still be writing when this one
// starts.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, uint32_t threads, uint32_t smem, uint32_t cluster,
                             cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The int8-limb GEMV on the reference's raw layout (hqb_raw_i8.cu): 128x128 tiles,
// group 128, prefix 1..4, batch one, FP32 x / y.  HQB_ERR_UNSUPPORTED (nothing
// enqueued) when the geometry, alignment or shared-memory size rules it out.
struct RawI8Launch {
  const hqb_geometry* geometry;
  const uint8_t* codes[HQB_MAX_STAGES];
  const uint16_t* scales[HQB_MAX_STAGES];
  uint32_t prefix;
  const float* x;
  const float* bias;
  float* y;
};
int launch_raw_i8(const RawI8Launch& a, void* stream);
uint32_t raw_i8_smem_bytes(uint64_t padded_cols);

// Whether a paged cache's description (its pointers aside) can be used at all (hqb_page.cu).
bool paged_cache_ok(const hqb_paged_cache* c);

}  // namespace hqb
