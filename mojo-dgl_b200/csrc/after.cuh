// Kernels of one call that follow one another: the next one's blocks may be set up
// while the last ones of the kernel before still run (programmatic dependent launch).
// Measured against plain launches: the expert plan's three kernels and the dispatch of
// 16384 x 4 x 2048 bf16 69.8 -> 65.6 us, layer norm's gradient of 16384 x 4096 bf16 82.6
// -> 81.3, segment_mm's of 190 rows 24.8 -> 23.6.
#pragma once

#include "common.cuh"

namespace bgl {

// In a kernel launched with launch_after: what the kernels before it wrote may be read,
// and what they read may be written, after this.
__device__ __forceinline__ void before_is_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Blocks of the kernel after this one may be started once every block has come here (or
// ended): they take no place that one of this kernel's blocks waits for.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A... args) {
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = s;
    c.attrs = &early;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

}  // namespace bgl
