// Elements of a storage type (fg_dtype) and reductions over a block, shared by the row operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fg_internal.cuh"

__device__ __forceinline__ float fg_widen(float x) { return x; }
__device__ __forceinline__ float fg_widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float fg_widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T fg_narrow(float x);
template <> __device__ __forceinline__ float fg_narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __half fg_narrow<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 fg_narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

inline uint32_t fg_dtype_size(int32_t dtype) { return dtype == FG_DTYPE_F32 ? 4 : 2; }
inline bool fg_dtype_known(int32_t dtype) { return dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16; }
// Does a tensor start at a whole element (NULL: yes)?
inline bool fg_at_element(const void* p, uint32_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// F<T>(args...) for the storage type.
#define FG_BY_DTYPE(dtype, F, ...) \
    ((dtype) == FG_DTYPE_F32 ? F<float>(__VA_ARGS__) : (dtype) == FG_DTYPE_F16 ? F<__half>(__VA_ARGS__) : F<__nv_bfloat16>(__VA_ARGS__))

__device__ __forceinline__ float fg_warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Two sums over a block of whole warps, in every thread; `red` is 64 floats, free again after the call's last barrier.
__device__ __forceinline__ float2 fg_block_sum2(float a, float b, float* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    a = fg_warp_sum(a);
    b = fg_warp_sum(b);
    if (lane == 0) { red[warp] = a; red[32 + warp] = b; }
    __syncthreads();
    a = fg_warp_sum(lane < nw ? red[lane] : 0.0f);
    b = fg_warp_sum(lane < nw ? red[32 + lane] : 0.0f);
    __syncthreads();
    return make_float2(a, b);
}
