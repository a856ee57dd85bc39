// kmb_launch.cuh -- a kernel that follows another of the same call on the same stream may be launched while the first
// still runs (programmatic dependent launch): its blocks are set up in the meantime and wait, on the device, for
// the first to end.  The first calls pdl_release() at its start, the second pdl_wait() before it reads anything
// that the first writes.
#pragma once
#include <cuda_runtime.h>

namespace kmb {

__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// after = false: an ordinary launch
template <typename... P, typename... A>
cudaError_t launch(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool after, A... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = after ? 1 : 0;
    return cudaLaunchKernelEx(&c, kern, P(args)...);
}

}  // namespace kmb
