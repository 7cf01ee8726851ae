// Launch helpers of the block operators: programmatic dependent launch and the
// number of SMs.
#pragma once

#include <cuda_runtime.h>

namespace vcattn {

// Let the next kernel of the stream start, and wait until the one before has
// completed (at once if this one was launched normally).
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// A kernel that may start while the one before it in the stream still runs
// (programmatic dependent launch; `after`: that one is of this call).  The
// kernels release the next one at their start, wait for the one before where
// they need its results, and otherwise at their end, so that a kernel's
// completion implies that of all before it.
template <typename K, typename... A>
cudaError_t launch_after(K kernel, dim3 grid, int threads, int smem, cudaStream_t st, bool after, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = after ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n > 0 ? n : 148;
}

}  // namespace vcattn
