// Kernels of one call that follow each other: each is brought to the GPU while the one before it still runs and waits inside for its end, so that its launch is
// not waited for. (Us, from a stream: gradients of a table by 3000 x 64 places 27.6, so 18.5; 16384 x 1024 f32 76.9, 67.4; 131072 x 2048 258, 250; clipping of 40 x 3000
// values 8.2, 6.2, of 8 M 20.5, 18.5. In a graph the two are within two percent: what follows is known there.
// Let in before the other's end, where all its blocks have begun, the next one's blocks are in the way: 131072 x 128 52.7, so 63.3.) The first kernel of a
// call, also an only one, is launched as any other, so all of them come after everything ahead of the call; every kernel of a chain has threads that wait, so that the last
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
