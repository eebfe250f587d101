// Element types of the layer operators (layer norm, routing, dispatch and
// combine): float32, float64 and bfloat16 in memory; sums, statistics and
// gradients in float32 (bf16, float32) or float64.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace bgl {

template <typename T>
struct AccOf { using type = float; };
template <>
struct AccOf<double> { using type = double; };
template <typename T>
using Acc = typename AccOf<T>::type;

__device__ __forceinline__ float to_acc(float x) { return x; }
__device__ __forceinline__ double to_acc(double x) { return x; }
__device__ __forceinline__ float to_acc(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_acc(Acc<T> x);
template <>
__device__ __forceinline__ float from_acc<float>(float x) { return x; }
template <>
__device__ __forceinline__ double from_acc<double>(double x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// How rows are moved: by single values; in whole 16-byte pieces; or, where their
// length is no multiple of 16 bytes, in the aligned pieces inside them and the few
// values beside those one by one.  Which values that are is the same for all rows
// of one remainder modulo the values of a piece.
enum RowMode { kScalar = 0, kAligned = 1, kShifted = 2 };

template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the block (a multiple of 32 threads, at most 1024), on every
// thread; `smem` holds 32 values and is free for reuse after the call.
template <typename A>
__device__ __forceinline__ A block_sum(A v, A *smem) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    v = warp_sum(v);
    if (lane == 0) smem[warp] = v;
    __syncthreads();
    v = lane < warps ? smem[lane] : A(0);
    v = warp_sum(v);
    __syncthreads();
    return v;
}

inline size_t row_elem_size(int dtype) { return dtype == BGL_F64 ? 8 : dtype == BGL_F32 ? 4 : 2; }
inline bool row_dtype(int dtype) { return dtype == BGL_F32 || dtype == BGL_F64 || dtype == BGL_BF16; }

}  // namespace bgl
