// Host-side helpers shared by the library's translation units: the per-thread error
// detail of the last failing call, status helpers, and the per-device state (SM count,
// kernel attributes set once per device), tensor-map encoding and kernel launches.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/nvfp4_group_gemm.h"

namespace nvfp4 {

// Detail text of the last failure on this thread (nvfp4_last_error_detail).
extern thread_local std::string g_last_error;

// Record a formatted detail and return `code`.
int fail(int code, const char* fmt, ...);
// NVFP4_ERR_CUDA with the CUDA error's name and text.
int cuda_fail(cudaError_t e, const char* what);

// cuTensorMapEncodeTiled (resolved through the runtime) without interleave, zero fill outside
// the tensor. False when the encoder is missing or rejects the map.
bool encode_tiled_map(CUtensorMap* map, CUtensorMapDataType type, unsigned rank, void* addr,
                      const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                      const cuuint32_t* elem_strides, CUtensorMapSwizzle swizzle,
                      CUtensorMapL2promotion promotion);

// Launch with programmatic stream serialization: the kernel may be scheduled while its
// predecessor in the stream drains, and must run griddepcontrol.wait before it touches memory.
// `grid` is a multiple of `cluster`, the CTAs per cluster.
template <typename... Params, typename... Args>
cudaError_t launch_clusters(void (*kernel)(Params...), int64_t grid, int cluster, int threads,
                            int smem, cudaStream_t stream, const Args&... args) {
  if (grid <= 0) return cudaSuccess;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), int64_t grid, int threads, int smem,
                             cudaStream_t stream, const Args&... args) {
  return launch_clusters(kernel, grid, 1, threads, smem, stream, args...);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kMaxDevices = 64;

struct DeviceState {
  std::once_flag once;
  int status = NVFP4_OK;
  int num_sms = 0;
  int pair_clusters = 0;        // CTA pairs that can be resident at once (plain pair kernel)
  int pair_clusters_gated = 0;  // same for the gated pair kernel
  std::string detail;
};

// The state of the calling thread's current device, initialised on first use (compute
// capability check, kernel shared-memory attributes, occupancy). NVFP4_OK and *out, or the
// failure status with its detail recorded.
int current_device_state(DeviceState** out);

}  // namespace nvfp4
