// pdl.cuh -- kernels that begin while the one before them in the stream ends.
//
// A kernel of a decode step takes 3 to 10 us, of which 2 are spent between it
// and its neighbours: a product of 33 rows on 4096 channels of 11008 took 18.3 us
// in a row of them and takes 15.3, one row on 12288 of 4096 11.7 and 9.6.  Launched through launch_next() its blocks may start once
// all blocks of the kernel before have called begin_next() or ended; until
// after_before() has returned, which every thread calls, they touch nothing
// that an earlier kernel writes or reads: only a handle's own weights, which
// are written when it is created.  A kernel that is launched plainly waits for
// the end of the one before, as always.
#pragma once

#include <cuda_runtime.h>

namespace kl {

__device__ __forceinline__ void begin_next() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void after_before() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

template <class... P, class... A>
void launch_next(void (*kernel)(P...), dim3 grid, int threads, size_t shared, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace kl
