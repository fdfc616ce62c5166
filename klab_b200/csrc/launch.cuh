// Host side that the batched operators share: a launch that may begin while the one before it ends, and the SM count.
#pragma once
#include <atomic>

#include <cuda_runtime.h>

#include "klab_b200.h"

namespace klab {

// kernel<<<grid, threads, smem, stream>>>(args...), with programmatic serialization unless KLAB_OPT_PDL is 0.
template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, void* stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = klab_get_option(KLAB_OPT_PDL) ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// SMs of the current device, asked for once.
inline int device_sms(int* sms) {
  static std::atomic<int> cached[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return KLAB_E_UNSUPPORTED;
  int n = cached[dev].load();
  if (!n) {
    err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (err != cudaSuccess) return err;
    cached[dev].store(n);
  }
  *sms = n;
  return 0;
}

}  // namespace klab
