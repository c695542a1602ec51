// Host-side helpers that the translation units of libmegaup.so share: the
// thread's error message, 4-D tensor maps, and the word a kernel without a
// caller-provided status word reports a failed wait in.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/megaup.h"

namespace mup {

// Stores the calling thread's error message and returns `code`.
int host_fail(int code, const char* fmt, ...);

#define MUP_HOST_CUDA(expr)                                                                       \
  do {                                                                                            \
    cudaError_t e_ = (expr);                                                                      \
    if (e_ != cudaSuccess)                                                                        \
      return ::mup::host_fail(MUP_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e_));      \
  } while (0)

// BF16 tensor [dim3, dim2, dim1, dim0] with dim0 contiguous -> 4-D tiled map
// with the 128-byte swizzle; box dim0 is 64 elements. Strides in elements.
int encode_map_4d(CUtensorMap* map, const void* base, const uint64_t dims[4], const int64_t strides[3],
                  const uint32_t box[4]);

// The library's own status word of a device (pinned, device-mapped, created at
// the device's first use, also under stream capture). Reports and clears a
// failure that an earlier kernel of this device left there.
int device_status_word(int device, uint32_t** device_ptr);

// Makes `device` current for a scope. Set even where it is current already: a thread that made no CUDA call yet (an
// autograd thread's first one) has no context, which the driver's tensor-map encoder needs.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (cudaGetDevice(&previous_) != cudaSuccess) previous_ = -1;
    error_ = cudaSetDevice(device);
    changed_ = error_ == cudaSuccess && previous_ != device && previous_ >= 0;
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(previous_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  cudaError_t error() const { return error_; }

 private:
  int previous_ = -1;
  bool changed_ = false;
  cudaError_t error_ = cudaSuccess;
};

// Whether kernels are launched so that they may begin while the kernel before them runs (MEGA_UP_PDL).
bool early_launches();

// A launch of that kind (`cluster` > 1: in clusters of so many CTAs). The kernel waits for the end of the one before
// itself (grid_dep_wait) before it touches global memory that is not constant.
template <typename... Params, typename... Args>
inline cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, int smem, int cluster,
                                cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid, config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = static_cast<size_t>(smem), config.stream = stream;
  cudaLaunchAttribute attributes[2]{};
  config.attrs = attributes;
  if (early_launches()) {
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    config.numAttrs = 1;
  }
  if (cluster > 1) {
    cudaLaunchAttribute& a = attributes[config.numAttrs++];
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = static_cast<unsigned>(cluster), a.val.clusterDim.y = 1, a.val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&config, kernel, args...);
}

// Launch attributes of a kernel are set once per device; `mask` is the static
// word of one kernel.
template <typename Kernel>
inline cudaError_t allow_smem_once(Kernel kernel, int bytes, int device, uint64_t* mask) {
  const uint64_t bit = 1ull << (device & 63);
  if (__atomic_load_n(mask, __ATOMIC_ACQUIRE) & bit) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) __atomic_fetch_or(mask, bit, __ATOMIC_RELEASE);
  return e;
}

}  // namespace mup
