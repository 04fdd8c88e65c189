// tg_host.h -- host-side helpers shared by the library's translation units.
#ifndef TG_HOST_H
#define TG_HOST_H

#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>

#include "../../include/tgsample.h"

namespace tg {

// Records the calling thread's last error (tg_last_error_string) and returns
// `code`.  Never throws.
__attribute__((visibility("hidden"))) int32_t set_error(int32_t code, const char* msg) noexcept;

inline int32_t set_cuda_error(cudaError_t e, const char* what) noexcept {
  char msg[256];
  snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(e));
  return set_error(TG_ERR_CUDA, msg);
}

// Makes `dev` current for a scope.
class CurrentDevice {
 public:
  explicit CurrentDevice(int dev) {
    cudaGetDevice(&prev_);
    if (prev_ != dev) cudaSetDevice(dev);
    dev_ = dev;
  }
  ~CurrentDevice() {
    if (prev_ != dev_) cudaSetDevice(prev_);
  }
  CurrentDevice(const CurrentDevice&) = delete;
  CurrentDevice& operator=(const CurrentDevice&) = delete;

 private:
  int prev_ = 0, dev_ = 0;
};

// Launches `kernel` on `st` as a programmatic dependent of the previous work on
// the stream: it is set up while that work drains, and waits on the device
// (griddepcontrol.wait) before it reads anything that work writes.
// `cluster` > 1 makes clusters of that many blocks.
template <class... KArgs, class... Args>
cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, cudaStream_t st, int cluster,
                         const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace tg

#define TG_TRY(call)                                             \
  do {                                                           \
    const cudaError_t e_ = (call);                               \
    if (e_ != cudaSuccess) return tg::set_cuda_error(e_, #call); \
  } while (0)

#endif  // TG_HOST_H
