// Programmatic dependent launch for chains of short kernels: a kernel launched with launch_after() may start while the
// one before it in the stream drains, and waits in pdl_wait() until that one is complete and its writes are visible.
// Every kernel of a chain calls pdl_trigger() as it starts (the next kernel's CTAs come only when all of this one's are
// running or done), and every thread of a kernel launched this way calls pdl_wait() before it touches memory that the chain
// writes, and before it returns: so a kernel's completion means that all before it are complete.  What was complete before
// the chain began may be read ahead of the wait.  Most of the launch gap between two kernels of a chain
// goes that way; outside such a chain both instructions do nothing.
#pragma once

#include <cuda_runtime.h>

namespace mat {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... K, typename... A>
cudaError_t launch_after(void (*kernel)(K...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, (K)args...);
}

}  // namespace mat
