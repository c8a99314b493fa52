// Kernels of one call that follow each other: each is brought to the GPU while the one before it still runs and waits inside for its end, so that its launch is
// not waited for. (Us: gradients of a table by 2000 x 64 places 12.6, so 11.6; 16384 x 1024 56.2, 52.9; 131072 x 2048 249.7, 247.2; clipping of 101770 values 5.5, 5.0.
// Let in before the other's end, where all its blocks have begun, the next one's blocks are in the way: 131072 x 128 52.7, so 63.3.) The first kernel of a
// call is launched as any other, so all of them come after everything ahead of the call; every kernel of a chain has threads that wait, so that the last
// one's end is the end of all.
//
// Data that the kernel before writes is never read by ld.global.nc (__ldg), which the compiler may move ahead of the wait.
#pragma once
#include <cuda_runtime.h>

#include <utility>

namespace ono {
// Until the kernel before has ended and its writes are seen (it waits for nobody but those before it; in a kernel launched as any other this is nothing).
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_behind(void (*kern)(P...), unsigned grid, int threads, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}
}  // namespace ono
