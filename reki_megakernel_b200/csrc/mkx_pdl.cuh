// Programmatic dependent launch of the episode cache's kernels. A step of serving is a row of short kernels: each waits
// for the one before only where it first touches global memory, so that its launch and first instructions lie under
// the other's end (10 new rows of 128 episodes 48.1 -> 45.9 us, 8 single rows 10.5 -> 9.1 us, 4096 stored rows 12.3 ->
// 10.0 us, as passes behind one another). None of them lets the next one start before it ends: that next one's waiting
// blocks would only be in the way (placing 100,003 rows: 7.2 us so, 14.7 us with griddepcontrol.launch_dependents first).
#pragma once
#include <cuda_runtime.h>

#include "mkx_cache_host.h"

namespace mkx {

// Every thread, before its first access to global memory: the kernels before have ended, their stores are visible.
__device__ __forceinline__ void pdl_begin() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... Params, typename... Args>
inline bool pdl_launch(void (*kernel)(Params...), int grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return mkxc::cuda_ok(cudaLaunchKernelEx(&cfg, kernel, args...));
}

}  // namespace mkx
