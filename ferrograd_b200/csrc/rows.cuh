// Elements of a storage type (fg_dtype) and reductions over a block, shared by the row operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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
// A barrier over one of a block's groups of warps (0 to 14).
__device__ __forceinline__ void fg_group_barrier(int group, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory"); }
// Sixteen bytes on their way from memory to shared memory, past the L1; a thread waits for its own.
__device__ __forceinline__ void fg_copy_async(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// The first `bytes` of them, zeros behind.
__device__ __forceinline__ void fg_copy_async(uint32_t to, const void* from, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 fg_load_shared(uint32_t from) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
    return v;
}
__device__ __forceinline__ void fg_store_shared(uint32_t to, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void fg_copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>      // all but the last kLeft groups have arrived
__device__ __forceinline__ void fg_copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

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

// ---- two f32 operations in one instruction ----
__device__ __forceinline__ uint64_t fg_bits2(float2 a) { return (uint64_t)__float_as_uint(a.y) << 32 | __float_as_uint(a.x); }
__device__ __forceinline__ float2 fg_floats2(uint64_t a) { return make_float2(__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)(a >> 32))); }
__device__ __forceinline__ float2 fg_add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(fg_bits2(a)), "l"(fg_bits2(b)));
    return fg_floats2(r);
}
__device__ __forceinline__ float2 fg_mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(fg_bits2(a)), "l"(fg_bits2(b)));
    return fg_floats2(r);
}
__device__ __forceinline__ float2 fg_fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(fg_bits2(a)), "l"(fg_bits2(b)), "l"(fg_bits2(c)));
    return fg_floats2(r);
}

// ---- sixteen bytes of a row at a time ----
// A row whose tensors start on 16-byte boundaries and whose length is a whole number of packs is moved as it lies (kShift = false).  Any
// other row is moved in 16-byte words of memory too: a thread owns the same columns in every row and every tensor, and turns what it
// reads and writes by the row's distance from the boundary.
template <typename T>
struct FgPack {
    static constexpr int E = 16 / sizeof(T);
    static __device__ __forceinline__ void widen(const uint4& v, float (&x)[E]) {
        if constexpr (sizeof(T) == 4) {
            x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2 && !std::is_same_v<T, __half>) {
                    x[2 * i] = __uint_as_float(w[i] << 16);
                    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    x[2 * i] = f.x;
                    x[2 * i + 1] = f.y;
                }
            }
        }
    }
    static __device__ __forceinline__ void widen(const uint4& v, float2 (&x)[E / 2]) {
        float y[E];
        widen(v, y);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) x[i] = make_float2(y[2 * i], y[2 * i + 1]);
    }
    static __device__ __forceinline__ uint4 narrow(const float2 (&x)[E / 2]) {
        float y[E];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) { y[2 * i] = x[i].x; y[2 * i + 1] = x[i].y; }
        return narrow(y);
    }
    static __device__ __forceinline__ uint4 narrow(const float (&x)[E]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(x[i]);
            else if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// Bytes o to o + 16 of the 32 in a and b; o < 16 and even.
__device__ __forceinline__ uint4 fg_turn(const uint4& a, const uint4& b, uint32_t o) {
    const bool by8 = o & 8, by4 = o & 4;
    const uint32_t s[6] = {by8 ? a.z : a.x, by8 ? a.w : a.y, by8 ? b.x : a.z, by8 ? b.y : a.w, by8 ? b.z : b.x, by8 ? b.w : b.y};
    uint32_t t[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) t[i] = by4 ? s[i + 1] : s[i];
    const uint32_t by2 = (o & 2) * 8;
    return make_uint4(__funnelshift_r(t[0], t[1], by2), __funnelshift_r(t[1], t[2], by2), __funnelshift_r(t[2], t[3], by2), __funnelshift_r(t[3], t[4], by2));
}

// The pack at p, of which `left` elements (1 or more) belong to the row; [lo, hi) is the tensor.  What lies behind the row's end in the same
// pack is whatever follows it in the tensor: the caller leaves it out.  Only words that lie in the tensor whole are read as words.
template <typename T, bool kShift>
__device__ __forceinline__ uint4 fg_load_pack(const T* p, uint32_t left, const T* lo, const T* hi) {
    if constexpr (!kShift) return *reinterpret_cast<const uint4*>(p);
    else {
        const uint32_t o = reinterpret_cast<uintptr_t>(p) & 15u;
        const char* q = reinterpret_cast<const char*>(p) - o;
        if (q >= reinterpret_cast<const char*>(lo) && q + (o ? 32 : 16) <= reinterpret_cast<const char*>(hi)) {
            const uint4 a = *reinterpret_cast<const uint4*>(q), b = *reinterpret_cast<const uint4*>(q + (o ? 16 : 0));
            return fg_turn(a, b, o);
        }
        uint4 v = make_uint4(0, 0, 0, 0);
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < FgPack<T>::E; ++e)
            if ((uint32_t)e < left) {
                if constexpr (sizeof(T) == 4) w[e] = *reinterpret_cast<const uint32_t*>(p + e);
                else w[e / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p + e) << (16 * (e & 1));
            }
        v.x = w[0]; v.y = w[1]; v.z = w[2]; v.w = w[3];
        return v;
    }
}

// Writes the first `left` elements (0: none) of v at p.  All lanes of a warp call it, with consecutive packs of one row; all but the last
// that has any are whole.  Turned rows: a lane writes the 16-byte word that ends in its columns, from its own and its neighbour's
// elements; the ends of the warp's stretch go element by element.
template <typename T, bool kShift>
__device__ __forceinline__ void fg_store_pack(T* p, const uint4& v, uint32_t left) {
    constexpr uint32_t E = FgPack<T>::E;
    if constexpr (!kShift) {
        if (left) *reinterpret_cast<uint4*>(p) = v;
    } else {
        const uint32_t lane = threadIdx.x & 31, o = reinterpret_cast<uintptr_t>(p) & 15u;
        uint4 before;
        before.x = __shfl_up_sync(0xffffffffu, v.x, 1);
        before.y = __shfl_up_sync(0xffffffffu, v.y, 1);
        before.z = __shfl_up_sync(0xffffffffu, v.z, 1);
        before.w = __shfl_up_sync(0xffffffffu, v.w, 1);
        uint32_t next = __shfl_down_sync(0xffffffffu, left, 1);
        if (lane == 31) next = 0;
        const uint32_t head = E - o / sizeof(T);      // own elements in the word that the pack starts in
        if (o == 0) {
            if (left == E) { *reinterpret_cast<uint4*>(p) = v; return; }
        } else if (lane > 0 && left >= head) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(p) - o) = fg_turn(before, v, 16 - o);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (uint32_t e = 0; e < E; ++e)
            if (e < left && (o == 0 || (e < head ? lane == 0 || left < head : next < head))) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p + e) = w[e];
                else *reinterpret_cast<uint16_t*>(p + e) = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
            }
    }
}
// Can the rows of these tensors be moved as they lie?
inline bool fg_rows_lie_straight(uint64_t cols, uint32_t size, const void* a, const void* b, const void* c = nullptr, const void* d = nullptr) {
    return cols * size % 16 == 0 && fg_aligned16(a) && fg_aligned16(b) && fg_aligned16(c) && fg_aligned16(d);
}
