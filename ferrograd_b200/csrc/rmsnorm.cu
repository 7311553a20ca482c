// Root-mean-square norm over the rows of a matrix, with the addition of a residual before it, and its backward pass.
//
// Forward: h = x + residual, rounded to the storage type; y = h * rstd * gamma with rstd = 1 / sqrt(mean(h * h) + eps).  The 8-bit form writes
// y / s in e4m3 for each group of columns, s = largest |y| of the group / 448 (448: the largest number of e4m3).
// Backward, with n = h * rstd and g = dy * gamma: dh = dsum + rstd * (g - n * mean(g * n)), which is the gradient of x and of the residual;
// dgamma = column sums of dy * n.
#include <cuda_fp8.h>

#include "norm_rows.cuh"

namespace {

struct RmsArgs {
    const void *x, *residual, *gamma;
    void *sum, *y;
    float *rstd, *scale;
    uint32_t rows, cols, group, groups;      // columns that share a scale, and how many such groups a row has
    float eps;
};
struct RmsBwdArgs {
    const void *x, *dy, *gamma, *dsum;
    const float* rstd;
    void *dx, *dgamma;
    uint32_t rows, cols;
    int accumulate;
};
constexpr float kE4m3Max = 448.0f;

// y / s in e4m3, rounded from the f32 quotient; a group of zeros stays one.  The quotient is the product with 1 / s and a step that adds what is left of y times 1 / s (P. Markstein,
// Computation of elementary functions on the IBM RISC System/6000 processor, 1990): exact enough that no byte differs, where a quotient beside a border between bytes took the product alone over
// it.  s has to leave the remainder its bits, or y is divided, which for all of them took 16384 x 4096 bf16 from 97 us to 143.
__device__ __forceinline__ bool has_inverse(float s) { return s > 1e-25f && s < 1e37f; }
__device__ __forceinline__ float divided(float y, float s) { return s > 0.0f ? y / s : fabsf(y) * 0.0f; }      // (a zero of either sign is byte 0)
__device__ __forceinline__ uint8_t to_e4m3(float y, float s) {
    float q;
    if (has_inverse(s)) {
        const float by = 1.0f / s;
        q = y * by;
        q = __fmaf_rn(__fmaf_rn(-s, q, y), by, q);
    } else q = divided(y, s);
    return (uint8_t)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}
// 2 * P of them, four in a word.
template <int P>
__device__ __forceinline__ void put_e4m3(float (&y)[2 * P], float s, uint32_t (&w)[P / 2]) {
    if (has_inverse(s)) {
        const float by = 1.0f / s;
#pragma unroll
        for (int e = 0; e < 2 * P; e += 2) {
            const float2 x = make_float2(y[e], y[e + 1]), by2 = make_float2(by, by);
            float2 q = fg_mul2(x, by2);
            q = fg_fma2(fg_fma2(q, make_float2(-s, -s), x), by2, q);
            y[e] = q.x;
            y[e + 1] = q.y;
        }
    } else
#pragma unroll
        for (int e = 0; e < 2 * P; ++e) y[e] = divided(y[e], s);
#pragma unroll
    for (int i = 0; i < P / 2; ++i)
        w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[4 * i], y[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
               (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[4 * i + 2], y[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
}

// A row per group of threads (norm_rows.cuh), kRes: with a residual.  y in 8 bits (k8) is for rows that lie straight: a thread's pack belongs to one group of columns,
// whose largest |y| is found among `lanes` neighbouring lanes, or (lanes = 0) over the row.
template <typename C, bool kRes, bool k8>
__global__ void __launch_bounds__(kMaxThreads, C::kTight && C::N <= 16 ? 2 : 1) rms_held_kernel(const RmsArgs a, int threads, int lanes) {
    using T = typename C::T;
    constexpr int H = C::N / 2;
    extern __shared__ uint4 shared[];
    __shared__ float red[kMaxGroups][k8 ? 4 : 2][32];
    fg_grid_enter();
    const Group group(threads);
    const uint32_t groups = blockDim.x / threads, step = gridDim.x * groups;
    const uint32_t first = C::kApart ? group.index * gridDim.x + blockIdx.x : blockIdx.x * groups + group.index;
    C columns(group, a.cols, first, shared);
    const float inv_n = 1.0f / (float)a.cols;
    const T* const gamma = static_cast<const T*>(a.gamma);
    typename C::Kept gammas;
    if (gamma) columns.keep(gamma, gammas);
    const uint64_t stride = (uint64_t)step * a.cols, at = (uint64_t)first * a.cols;
    const T *x = static_cast<const T*>(a.x) + at, *res = kRes ? static_cast<const T*>(a.residual) + at : nullptr, *x_ahead = x, *res_ahead = res;
    T *sum = a.sum ? static_cast<T*>(a.sum) + at : nullptr, *y = k8 ? nullptr : static_cast<T*>(a.y) + at;
    uint8_t* y8 = k8 ? static_cast<uint8_t*>(a.y) + at : nullptr;
    uint64_t next = first;
    auto ask = [&] {
        if (next < a.rows) {
            columns.ask(0, x_ahead);
            if (kRes) columns.ask(1, res_ahead);
        }
        columns.asked();
        next += step;
        x_ahead += stride;
        if (kRes) res_ahead += stride;
    };
    if (C::kAhead)
#pragma unroll
        for (int i = 0; i < C::kStages; ++i) ask();
    int turn = 0;
    for (uint64_t r = first; r < a.rows; r += step, x += stride) {
        float2 v[H];
        columns.arrived();
        columns.get(0, x, v);
        if (kRes) {
            float2 u[H];
            columns.get(1, res, u);
            res += stride;
#pragma unroll
            for (int i = 0; i < H; ++i) {
                v[i] = fg_add2(v[i], u[i]);
                if (sizeof(T) == 2) v[i] = make_float2(fg_widen(fg_narrow<T>(v[i].x)), fg_widen(fg_narrow<T>(v[i].y)));
            }
        }
        columns.taken();
        if (C::kAhead) ask();
        if (sum) {
            columns.store(sum, v);
            sum += stride;
        }
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < H; ++i) s = fg_fma2(v[i], v[i], s);
        const float rstd = 1.0f / sqrtf(__fmaf_rn(group.sum(s.x + s.y, red[group.index][turn]), inv_n, a.eps));
        const float2 by = make_float2(rstd, rstd);
#pragma unroll
        for (int i = 0; i < H; ++i) v[i] = fg_mul2(v[i], by);
        if (gamma) {
            float2 g[H];
            columns.kept(gammas, gamma, g);
#pragma unroll
            for (int i = 0; i < H; ++i) v[i] = fg_mul2(v[i], g[i]);
        }
        if constexpr (!k8) {
            columns.store(y, v);
            y += stride;
        } else {
            constexpr int P = C::P, K = H / P;      // pairs of a pack, packs
            float most[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                most[k] = 0.0f;
#pragma unroll
                for (int e = 0; e < P; ++e) most[k] = fmaxf(most[k], fmaxf(fabsf(v[k * P + e].x), fabsf(v[k * P + e].y)));
            }
            if (lanes) {
                for (int o = lanes / 2; o > 0; o >>= 1)
#pragma unroll
                    for (int k = 0; k < K; ++k) most[k] = fmaxf(most[k], __shfl_xor_sync(0xffffffffu, most[k], o));
            } else {
#pragma unroll
                for (int k = 1; k < K; ++k) most[0] = fmaxf(most[0], most[k]);
                most[0] = group.max(most[0], red[group.index][2 + turn]);
#pragma unroll
                for (int k = 1; k < K; ++k) most[k] = most[0];
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!columns.has(k)) continue;
                const float scale = most[k] / kE4m3Max;
                const uint32_t c = (group.thread + k * threads) * (2 * P);      // the pack's first column
                if (lanes ? (group.lane & (lanes - 1)) == 0 : k == 0 && group.thread == 0) a.scale[r * a.groups + (lanes ? c / a.group : 0)] = scale;
                float q[2 * P];
#pragma unroll
                for (int e = 0; e < P; ++e) { q[2 * e] = v[k * P + e].x; q[2 * e + 1] = v[k * P + e].y; }
                uint32_t w[P / 2];
                put_e4m3<P>(q, scale, w);
                if constexpr (P == 4) *reinterpret_cast<uint2*>(y8 + c) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t*>(y8 + c) = w[0];
            }
            y8 += stride;
        }
        if (group.thread == 0 && a.rstd) a.rstd[r] = rstd;
        turn ^= 1;
    }
}

// e4m3 of rows that do not lie straight, or of groups that are more than a warp's packs: kWarps warps a row, a warp has kUnits stretches of 128 columns, a lane every
// 32nd of them, so groups of 32, 64, 128 and 256 columns are found within a warp.  Read once; elements, not words.
template <typename T, int kWarps, int kUnits, bool kRes>
__global__ void __launch_bounds__(256) rms8_ragged_kernel(const RmsArgs a) {
    constexpr int kPer = 8 / kWarps;      // rows of a block
    __shared__ float red[2][8];
    fg_grid_enter();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kWarps;
    const uint64_t r = (uint64_t)blockIdx.x * kPer + warp / kWarps;
    const bool there = r < a.rows;
    const uint64_t at = r * a.cols;
    const uint32_t first = part * (kUnits * 128) + lane;
    const T *const x = static_cast<const T*>(a.x) + at, *const res = kRes ? static_cast<const T*>(a.residual) + at : nullptr, *const gamma = static_cast<const T*>(a.gamma);
    float v[kUnits][4];
#pragma unroll
    for (int i = 0; i < kUnits * 4; ++i) {
        const uint32_t c = first + 32 * i;
        v[i / 4][i % 4] = there && c < a.cols ? fg_widen(x[c]) : 0.0f;
    }
    if (kRes)
#pragma unroll
        for (int i = 0; i < kUnits * 4; ++i) {
            const uint32_t c = first + 32 * i;
            if (there && c < a.cols) v[i / 4][i % 4] = fg_widen(fg_narrow<T>(v[i / 4][i % 4] + fg_widen(res[c])));
        }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kUnits * 4; ++i) s = __fmaf_rn(v[i / 4][i % 4], v[i / 4][i % 4], s);
    s = fg_warp_sum(s);
    if (kWarps > 1) {
        if (lane == 0) red[0][warp] = s;
        __syncthreads();
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += red[0][w];
    }
    const float rstd = 1.0f / sqrtf(s / (float)a.cols + a.eps);
    float most[kUnits][4];
#pragma unroll
    for (int i = 0; i < kUnits * 4; ++i) {
        const uint32_t c = first + 32 * i;
        if (there && c < a.cols) {
            if (a.sum) static_cast<T*>(a.sum)[at + c] = fg_narrow<T>(v[i / 4][i % 4]);
            v[i / 4][i % 4] *= rstd * (gamma ? fg_widen(gamma[c]) : 1.0f);
        }
        most[i / 4][i % 4] = fabsf(v[i / 4][i % 4]);
    }
    const bool whole = a.groups == 1;      // one scale a row
    if (whole || a.group >= 64)
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            most[u][0] = most[u][1] = fmaxf(most[u][0], most[u][1]);
            most[u][2] = most[u][3] = fmaxf(most[u][2], most[u][3]);
        }
    if (whole || a.group >= 128)
#pragma unroll
        for (int u = 0; u < kUnits; ++u) most[u][0] = most[u][1] = most[u][2] = most[u][3] = fmaxf(most[u][0], most[u][2]);
    if (whole || a.group == 256)
#pragma unroll
        for (int u = 0; u + 1 < kUnits; u += 2) {
            const float m = fmaxf(most[u][0], most[u + 1][0]);
#pragma unroll
            for (int e = 0; e < 4; ++e) most[u][e] = most[u + 1][e] = m;
        }
    if (whole) {
        float m = most[0][0];
#pragma unroll
        for (int u = 1; u < kUnits; ++u) m = fmaxf(m, most[u][0]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (kWarps > 1) {
            if (lane == 0) red[1][warp] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) m = fmaxf(m, red[1][w]);
        }
#pragma unroll
        for (int i = 0; i < kUnits * 4; ++i) most[i / 4][i % 4] = m;
    } else
#pragma unroll
        for (int i = 0; i < kUnits * 4; ++i)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most[i / 4][i % 4] = fmaxf(most[i / 4][i % 4], __shfl_xor_sync(0xffffffffu, most[i / 4][i % 4], o));
    uint8_t* const y = static_cast<uint8_t*>(a.y) + at;
#pragma unroll
    for (int i = 0; i < kUnits * 4; ++i) {
        const uint32_t c = first + 32 * i;
        if (!there || c >= a.cols) continue;
        const float scale = most[i / 4][i % 4] / kE4m3Max;
        y[c] = to_e4m3(v[i / 4][i % 4], scale);
        if (whole ? c == 0 : c % a.group == 0) a.scale[r * a.groups + (whole ? 0 : c / a.group)] = scale;
    }
    if (there && part == 0 && lane == 0 && a.rstd) a.rstd[r] = rstd;
}

// The backward pass the same way: kSum with what reaches h by other ways.  With the parameter's gradient (kParams) a thread sums its columns over the rows of its
// group, a block adds its groups and leaves one row of parts: [block][pitch].
template <typename C, bool kSum, bool kParams>
__global__ void __launch_bounds__(kMaxThreads, C::kTight && C::N <= 4 ? 2 : 1) rms_bwd_held_kernel(const RmsBwdArgs a, int threads, float* parts, uint32_t pitch) {
    using T = typename C::T;
    constexpr int H = C::N / 2;
    extern __shared__ uint4 shared[];      // the slots; at the end the groups' sums
    __shared__ float red[kMaxGroups][2][32];
    fg_grid_enter();
    const Group group(threads);
    const uint32_t groups = blockDim.x / threads, step = gridDim.x * groups;
    const uint32_t first = C::kApart ? group.index * gridDim.x + blockIdx.x : blockIdx.x * groups + group.index;
    C columns(group, a.cols, first, shared);
    const float inv_n = 1.0f / (float)a.cols;
    const T* const gamma = static_cast<const T*>(a.gamma);
    typename C::Kept gammas;
    if (gamma) columns.keep(gamma, gammas);
    const uint64_t stride = (uint64_t)step * a.cols, at = (uint64_t)first * a.cols;
    const T *x = static_cast<const T*>(a.x) + at, *dy = static_cast<const T*>(a.dy) + at, *ds = kSum ? static_cast<const T*>(a.dsum) + at : nullptr;
    const T *x_ahead = x, *dy_ahead = dy, *ds_ahead = ds;
    T* dx = a.dx ? static_cast<T*>(a.dx) + at : nullptr;
    uint64_t next = first;
    auto ask = [&] {
        if (next < a.rows) {
            columns.ask(0, x_ahead);
            columns.ask(1, dy_ahead);
            if (kSum) columns.ask(2, ds_ahead);
        }
        columns.asked();
        next += step;
        x_ahead += stride;
        dy_ahead += stride;
        if (kSum) ds_ahead += stride;
    };
    if (C::kAhead)
#pragma unroll
        for (int i = 0; i < C::kStages; ++i) ask();
    float rstd = first < a.rows ? a.rstd[first] : 0.0f;
    float2 dg[H];
#pragma unroll
    for (int i = 0; i < H; ++i) dg[i] = make_float2(0.0f, 0.0f);
    int turn = 0;
    for (uint64_t r = first; r < a.rows; r += step, x += stride, dy += stride) {
        float2 c[H], g[H], d[kSum ? H : 1];
        const float sd = rstd;
        const float2 by = make_float2(sd, sd);
        columns.arrived();
        columns.get(0, x, c);
        columns.get(1, dy, g);
        if constexpr (kSum) {
            columns.get(2, ds, d);
            ds += stride;
        }
        columns.taken();
        if (r + step < a.rows) rstd = a.rstd[r + step];
        if (C::kAhead) ask();
        if (kParams)
#pragma unroll
            for (int i = 0; i < H; ++i) dg[i] = fg_fma2(g[i], fg_mul2(c[i], by), dg[i]);      // (columns that are not there: dy is zero)
        if (dx) {
            if (gamma) {
                float2 gm[H];
                columns.kept(gammas, gamma, gm);
#pragma unroll
                for (int i = 0; i < H; ++i) g[i] = fg_mul2(g[i], gm[i]);
            }
            float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < H; ++i) s = fg_fma2(g[i], c[i], s);
            const float t = group.sum(s.x + s.y, red[group.index][turn]), u = -sd * sd * (sd * (t * inv_n));
            const float2 slope = make_float2(u, u);
#pragma unroll
            for (int i = 0; i < H; ++i) {
                g[i] = fg_fma2(g[i], by, fg_mul2(c[i], slope));
                if constexpr (kSum) g[i] = fg_add2(g[i], d[i]);
            }
            columns.store(dx, g);
            dx += stride;
        }
        turn ^= 1;
    }
    if constexpr (kParams) {
        float2* const sums = reinterpret_cast<float2*>(shared);      // the groups one after the other: [pair][thread]
        if (C::kAhead) fg_copies_wait<0>();
        for (uint32_t i = 0; i + 1 < groups; ++i) {
            __syncthreads();
            if (group.index == (int)i)
#pragma unroll
                for (int e = 0; e < H; ++e) {
                    float2* const p = sums + e * threads + group.thread;
                    *p = i ? fg_add2(*p, dg[e]) : dg[e];
                }
        }
        __syncthreads();
        if (group.index + 1 == (int)groups) {
            if (groups > 1)
#pragma unroll
                for (int e = 0; e < H; ++e) dg[e] = fg_add2(sums[e * threads + group.thread], dg[e]);
            columns.store_sums(parts + (uint64_t)blockIdx.x * pitch, dg);
        }
    }
}

// Adds the blocks' parts: 128 columns per block, a warp takes every 32nd part.  pitch is a multiple of 128.
template <typename T>
__global__ void __launch_bounds__(1024) rms_parts_kernel(const RmsBwdArgs a, const float* parts, uint32_t count, uint32_t pitch) {
    __shared__ float4 red[32][32];
    fg_grid_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t at = blockIdx.x * 128 + 4 * lane;
    T* const out = static_cast<T*>(a.dgamma);
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t i0 = warp; i0 < count; i0 += 32 * 8) {
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = i0 + 32 * j < count ? *reinterpret_cast<const float4*>(parts + (uint64_t)(i0 + 32 * j) * pitch + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 8; ++j) { s.x += v[j].x; s.y += v[j].y; s.z += v[j].z; s.w += v[j].w; }
    }
    red[warp][lane] = s;
    __syncthreads();
    if (threadIdx.x < 128) {
        const uint32_t c = blockIdx.x * 128 + threadIdx.x;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 32; ++w) sum += reinterpret_cast<const float*>(red[w])[threadIdx.x];
        if (c < a.cols) out[c] = fg_narrow<T>(a.accumulate ? fg_widen(out[c]) + sum : sum);
    }
}

// Any row: one block each, read once per sum.
template <typename T, bool k8>
__global__ void __launch_bounds__(256) rms_stream_kernel(const RmsArgs a) {
    __shared__ float red[64];
    fg_grid_enter();
    const T* const gamma = static_cast<const T*>(a.gamma);
    for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const uint64_t at = r * a.cols;
        const T *const x = static_cast<const T*>(a.x) + at, *const res = a.residual ? static_cast<const T*>(a.residual) + at : nullptr;
        T* const sum = a.sum ? static_cast<T*>(a.sum) + at : nullptr;
        auto h_at = [&](uint64_t c) { return res ? fg_widen(fg_narrow<T>(fg_widen(x[c]) + fg_widen(res[c]))) : fg_widen(x[c]); };
        float s = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += 256) {
            const float h = h_at(c);
            s = __fmaf_rn(h, h, s);
        }
        const float rstd = 1.0f / sqrtf(fg_block_sum2(s, 0.0f, red).x / (float)a.cols + a.eps);
        if (threadIdx.x == 0 && a.rstd) a.rstd[r] = rstd;
        auto y_of = [&](float h, uint64_t c) { return h * rstd * (gamma ? fg_widen(gamma[c]) : 1.0f); };
        if (!k8) {
            T* const y = static_cast<T*>(a.y) + at;
            for (uint64_t c = threadIdx.x; c < a.cols; c += 256) {      // (sum or y may be x or the residual)
                const float h = h_at(c);
                if (sum) sum[c] = fg_narrow<T>(h);
                y[c] = fg_narrow<T>(y_of(h, c));
            }
        } else {
            uint8_t* const y = static_cast<uint8_t*>(a.y) + at;
            const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            if (a.groups > 1) {
                for (uint32_t g = warp; g < a.groups; g += 8) {
                    const uint64_t c0 = (uint64_t)g * a.group, c1 = min((uint64_t)a.cols, c0 + a.group);
                    float most = 0.0f;
                    for (uint64_t c = c0 + lane; c < c1; c += 32) most = fmaxf(most, fabsf(y_of(h_at(c), c)));
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    const float scale = most / kE4m3Max;
                    for (uint64_t c = c0 + lane; c < c1; c += 32) {
                        const float h = h_at(c);
                        if (sum) sum[c] = fg_narrow<T>(h);
                        y[c] = to_e4m3(y_of(h, c), scale);
                    }
                    if (lane == 0) a.scale[r * a.groups + g] = scale;
                }
            } else {
                float most = 0.0f;
                for (uint64_t c = threadIdx.x; c < a.cols; c += 256) most = fmaxf(most, fabsf(y_of(h_at(c), c)));
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (lane == 0) red[warp] = most;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < 8; ++w) most = fmaxf(most, red[w]);
                __syncthreads();
                const float scale = most / kE4m3Max;
                for (uint64_t c = threadIdx.x; c < a.cols; c += 256) {
                    const float h = h_at(c);
                    if (sum) sum[c] = fg_narrow<T>(h);
                    y[c] = to_e4m3(y_of(h, c), scale);
                }
                if (threadIdx.x == 0) a.scale[r] = scale;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) rms_bwd_stream_kernel(const RmsBwdArgs a) {
    __shared__ float red[64];
    fg_grid_enter();
    const T* const gamma = static_cast<const T*>(a.gamma);
    for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const uint64_t at = r * a.cols;
        const T *const x = static_cast<const T*>(a.x) + at, *const dy = static_cast<const T*>(a.dy) + at, *const dsum = a.dsum ? static_cast<const T*>(a.dsum) + at : nullptr;
        T* const dx = static_cast<T*>(a.dx) + at;
        const float rstd = a.rstd[r];
        float s = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += 256) s = __fmaf_rn(fg_widen(dy[c]) * (gamma ? fg_widen(gamma[c]) : 1.0f), fg_widen(x[c]) * rstd, s);
        const float m = fg_block_sum2(s, 0.0f, red).x / (float)a.cols;
        for (uint64_t c = threadIdx.x; c < a.cols; c += 256) {
            const float g = fg_widen(dy[c]) * (gamma ? fg_widen(gamma[c]) : 1.0f), n = fg_widen(x[c]) * rstd;
            dx[c] = fg_narrow<T>(__fmaf_rn(rstd, __fmaf_rn(-n, m, g), dsum ? fg_widen(dsum[c]) : 0.0f));
        }
    }
}

// dgamma by columns, over chunks of rows: part is [chunks][cols].  A warp takes 32 columns, or as many packs of rows that lie straight, and every 8th row.
constexpr uint32_t kChunk = 256;
template <typename T, bool kPacked>
__global__ void __launch_bounds__(256) rms_columns_kernel(const RmsBwdArgs a, float* part) {
    constexpr int E = kPacked ? FgPack<T>::E : 1, kRows = 4;
    __shared__ float red[8][32][E];
    fg_grid_enter();
    const uint64_t c = ((uint64_t)blockIdx.x * 32 + threadIdx.x) * E;
    const uint32_t r0 = blockIdx.y * kChunk, r1 = min(a.rows, r0 + kChunk);
    const T *const x = static_cast<const T*>(a.x) + c, *const dy = static_cast<const T*>(a.dy) + c;
    float s[E] = {};
    if (c < a.cols)
        for (uint32_t r = r0 + threadIdx.y; r < r1; r += 8 * kRows) {
            float u[kRows][E], v[kRows][E], rstd[kRows];
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                const uint32_t row = r + 8 * j;
                const bool there = row < r1;
                rstd[j] = there ? a.rstd[row] : 0.0f;
                if constexpr (kPacked) {
                    FgPack<T>::widen(there ? *reinterpret_cast<const uint4*>(x + (uint64_t)row * a.cols) : make_uint4(0, 0, 0, 0), u[j]);
                    FgPack<T>::widen(there ? *reinterpret_cast<const uint4*>(dy + (uint64_t)row * a.cols) : make_uint4(0, 0, 0, 0), v[j]);
                } else {
                    u[j][0] = there ? fg_widen(x[(uint64_t)row * a.cols]) : 0.0f;
                    v[j][0] = there ? fg_widen(dy[(uint64_t)row * a.cols]) : 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < kRows; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] = __fmaf_rn(v[j][e], u[j][e] * rstd[j], s[e]);
        }
#pragma unroll
    for (int e = 0; e < E; ++e) red[threadIdx.y][threadIdx.x][e] = s[e];
    __syncthreads();
    if (threadIdx.y == 0 && c < a.cols)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) t += red[i][threadIdx.x][e];
            part[(uint64_t)blockIdx.y * a.cols + c + e] = t;
        }
}
template <typename T>
__global__ void __launch_bounds__(256) rms_fold_kernel(const RmsBwdArgs a, const float* part, uint32_t chunks) {
    fg_grid_enter();
    const uint64_t c = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    T* const out = static_cast<T*>(a.dgamma);
    float s = 0.0f;
    for (uint32_t i = 0; i < chunks; ++i) s += part[(uint64_t)i * a.cols + c];
    out[c] = fg_narrow<T>(a.accumulate ? fg_widen(out[c]) + s : s);
}

template <typename C, bool kRes, bool k8 = false>
int32_t launch_held(fg_ctx* ctx, const RmsArgs& a, HeldPlan p, int lanes = 0) {
    static std::atomic<uint64_t> done{0};
    const int32_t s = allow_shared(ctx, done, rms_held_kernel<C, kRes, k8>, p.bytes);
    if (s != FG_OK) return s;
    fg_launch(ctx, rms_held_kernel<C, kRes, k8>, p.grid, p.threads * p.groups, p.bytes, a, p.threads, lanes);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T, int kPacks, bool kRes, bool k8>
int32_t launch_straight(fg_ctx* ctx, const RmsArgs& a, HeldPlan p, int lanes) {
    constexpr int kTensors = kRes ? 2 : 1;
    return p.full ? launch_held<Straight<T, kPacks, true, kTensors>, kRes, k8>(ctx, a, p, lanes) : launch_held<Straight<T, kPacks, false, kTensors>, kRes, k8>(ctx, a, p, lanes);
}
// A thread holds 16 columns, more where the row is longer than a block's threads have so, fewer for few rows: held_plan() has what that was measured at.
template <typename T, bool kRes, bool k8>
int32_t fwd_straight(fg_ctx* ctx, const RmsArgs& a, int lanes, bool* took) {
    constexpr int usual = 16 / FgPack<T>::E;
    const HeldPlan p = held_plan(ctx, a.rows, a.cols / FgPack<T>::E, 1, usual, 8, kRes ? 2 : 1, 512);
    *took = p.threads != 0;
    if (!p.threads) return FG_OK;
    return p.units == 1 ? launch_straight<T, 1, kRes, k8>(ctx, a, p, lanes) : p.units == 2 ? launch_straight<T, 2, kRes, k8>(ctx, a, p, lanes)
           : p.units == 4 ? launch_straight<T, 4, kRes, k8>(ctx, a, p, lanes) : launch_straight<T, 8, kRes, k8>(ctx, a, p, lanes);
}
template <typename T, bool kRes>
int32_t fwd_ragged(fg_ctx* ctx, const RmsArgs& a, bool* took) {
    constexpr int usual = 16 / FgPack<T>::E, kTensors = kRes ? 2 : 1;
    *took = true;
    if (a.cols > 64 * sizeof(T) && fg_aligned16(a.x) && fg_aligned16(a.residual) && fg_aligned16(a.sum) && fg_aligned16(a.y)) {
        constexpr int most = 32 / FgPack<T>::E;      // a bit per column of a thread
        const HeldPlan p = shifted_plan<T>(ctx, a.rows, a.cols, 1, usual, most, kTensors);
        if (p.threads)
            return p.units == 1 ? launch_held<Shifted<T, 1, kTensors>, kRes>(ctx, a, p) : p.units == 2 ? launch_held<Shifted<T, 2, kTensors>, kRes>(ctx, a, p)
                   : p.units == 4 ? launch_held<Shifted<T, 4, kTensors>, kRes>(ctx, a, p) : launch_held<Shifted<T, most, kTensors>, kRes>(ctx, a, p);
    }
    const HeldPlan p = held_plan(ctx, a.rows, a.cols, 4, 8, 32, 0, 1024);
    if (p.threads)
        return p.units == 4 ? launch_held<Ragged<T, 4, kTensors>, kRes>(ctx, a, p) : p.units == 8 ? launch_held<Ragged<T, 8, kTensors>, kRes>(ctx, a, p)
               : p.units == 16 ? launch_held<Ragged<T, 16, kTensors>, kRes>(ctx, a, p) : launch_held<Ragged<T, 32, kTensors>, kRes>(ctx, a, p);
    *took = false;
    return FG_OK;
}
template <typename T, int kWarps, int kUnits>
int32_t ragged_e4m3(fg_ctx* ctx, const RmsArgs& a) {
    constexpr uint32_t kPer = 8 / kWarps;
    fg_launch(ctx, a.residual ? rms8_ragged_kernel<T, kWarps, kUnits, true> : rms8_ragged_kernel<T, kWarps, kUnits, false>, (unsigned)(((uint64_t)a.rows + kPer - 1) / kPer), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T>
int32_t rms_fwd(fg_ctx* ctx, const RmsArgs& a) {
    constexpr uint32_t E = FgPack<T>::E;
    const bool res = a.residual, straight = fg_rows_lie_straight(a.cols, sizeof(T), a.x, a.residual, a.gamma, a.sum);
    bool took = false;
    int32_t s = FG_OK;
    if (a.scale) {
        const uint32_t lanes = a.group == a.cols && a.groups == 1 ? 0 : a.group / E;      // 256 columns of f32 are two warps
        if (straight && reinterpret_cast<uintptr_t>(a.y) % E == 0 && lanes <= 32)
            s = res ? fwd_straight<T, true, true>(ctx, a, (int)lanes, &took) : fwd_straight<T, false, true>(ctx, a, (int)lanes, &took);
    } else if (straight && fg_aligned16(a.y)) s = res ? fwd_straight<T, true, false>(ctx, a, 0, &took) : fwd_straight<T, false, false>(ctx, a, 0, &took);
    else s = res ? fwd_ragged<T, true>(ctx, a, &took) : fwd_ragged<T, false>(ctx, a, &took);
    if (took) return s;
    // A row by one warp or eight, 4 to 32 elements a lane (64 spill: 4504 x 9394 f16 984 us, 172 read once per sum).
    if (a.scale) {
        if (a.cols <= 128 && a.group != 256) return ragged_e4m3<T, 1, 1>(ctx, a);
        if (a.cols <= 1024) return ragged_e4m3<T, 1, 8>(ctx, a);
        if (a.cols <= 4096) return ragged_e4m3<T, 8, 4>(ctx, a);
    }
    fg_launch(ctx, a.scale ? rms_stream_kernel<T, true> : rms_stream_kernel<T, false>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

template <typename C, bool kSum, bool kParams>
int32_t launch_bwd(fg_ctx* ctx, const RmsBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch) {
    const size_t sums = kParams && p.groups > 1 ? 4ull * C::N * p.threads : 0, bytes = p.bytes < sums ? sums : p.bytes;
    static std::atomic<uint64_t> done{0};
    const int32_t s = allow_shared(ctx, done, rms_bwd_held_kernel<C, kSum, kParams>, bytes);
    if (s != FG_OK) return s;
    fg_launch(ctx, rms_bwd_held_kernel<C, kSum, kParams>, p.grid, p.threads * p.groups, bytes, a, p.threads, parts, pitch);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <template <typename, int, int> class R, typename T, int kUnits>
int32_t launch_bwd_held(fg_ctx* ctx, const RmsBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch) {
    if (a.dsum && a.dx) return parts ? launch_bwd<R<T, kUnits, 3>, true, true>(ctx, a, p, parts, pitch) : launch_bwd<R<T, kUnits, 3>, true, false>(ctx, a, p, parts, pitch);
    return parts ? launch_bwd<R<T, kUnits, 2>, false, true>(ctx, a, p, parts, pitch) : launch_bwd<R<T, kUnits, 2>, false, false>(ctx, a, p, parts, pitch);
}
template <typename T, int kUnits, int kTensors> using StraightFull = Straight<T, kUnits, true, kTensors>;
template <typename T, int kUnits, int kTensors> using StraightPart = Straight<T, kUnits, false, kTensors>;
template <typename T, int kUnits>
int32_t launch_bwd_straight(fg_ctx* ctx, const RmsBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch) {
    return p.full ? launch_bwd_held<StraightFull, T, kUnits>(ctx, a, p, parts, pitch) : launch_bwd_held<StraightPart, T, kUnits>(ctx, a, p, parts, pitch);
}
template <typename T>
int32_t rms_bwd(fg_ctx* ctx, const RmsBwdArgs& a) {
    constexpr int usual = 16 / FgPack<T>::E;
    const int tensors = a.dsum && a.dx ? 3 : 2;
    const bool straight = fg_rows_lie_straight(a.cols, sizeof(T), a.x, a.dy, a.gamma, a.dx) && fg_aligned16(a.dsum);
    HeldPlan p{};
    if (straight) p = held_plan(ctx, a.rows, a.cols / FgPack<T>::E, 1, usual, usual, tensors, 512);
    else if (fg_aligned16(a.x) && fg_aligned16(a.dy) && fg_aligned16(a.dx) && fg_aligned16(a.dsum)) p = shifted_plan<T>(ctx, a.rows, a.cols, 1, usual, usual, tensors);
    const bool shifted = !straight && p.threads;
    if (!straight && !shifted) p = held_plan(ctx, a.rows, a.cols, 4, 4, 16, 0, 1024);
    if (p.threads) {
        float* parts = nullptr;
        const uint32_t pitch = (a.cols + 127) / 128 * 128;
        if (a.dgamma) {
            void* w;
            const int32_t s = fg_ws_alloc(ctx, 4ull * pitch * p.grid, &w);
            if (s != FG_OK) return s;
            parts = (float*)w;
        }
        int32_t s;
        if (straight) {
            if (p.units == 1) s = launch_bwd_straight<T, 1>(ctx, a, p, parts, pitch);
            else if (p.units == 2) s = launch_bwd_straight<T, 2>(ctx, a, p, parts, pitch);
            else s = launch_bwd_straight<T, usual>(ctx, a, p, parts, pitch);
        } else if (shifted) {
            if (p.units == 1) s = launch_bwd_held<Shifted, T, 1>(ctx, a, p, parts, pitch);
            else if (p.units == 2) s = launch_bwd_held<Shifted, T, 2>(ctx, a, p, parts, pitch);
            else s = launch_bwd_held<Shifted, T, usual>(ctx, a, p, parts, pitch);
        } else if (p.units == 4) s = launch_bwd_held<Ragged, T, 4>(ctx, a, p, parts, pitch);
        else if (p.units == 8) s = launch_bwd_held<Ragged, T, 8>(ctx, a, p, parts, pitch);
        else s = launch_bwd_held<Ragged, T, 16>(ctx, a, p, parts, pitch);
        if (s != FG_OK || !parts) return s;
        fg_launch(ctx, rms_parts_kernel<T>, pitch / 128, 1024, 0, a, (const float*)parts, (uint32_t)p.grid, pitch);
        FG_LAUNCHED(ctx);
        return FG_OK;
    }
    if (a.dgamma) {      // before dx, which may be dy, x or dsum
        const uint32_t chunks = (a.rows + kChunk - 1) / kChunk;
        void* w;
        const int32_t s = fg_ws_alloc(ctx, 4ull * chunks * a.cols, &w);
        if (s != FG_OK) return s;
        for (uint32_t c0 = 0; c0 < chunks; c0 += 65535) {
            RmsBwdArgs b = a;
            const uint64_t skip = (uint64_t)c0 * kChunk;
            b.x = static_cast<const T*>(a.x) + skip * a.cols;
            b.dy = static_cast<const T*>(a.dy) + skip * a.cols;
            b.rstd = a.rstd + skip;
            b.rows = a.rows - (uint32_t)skip;
            const uint32_t E = straight ? FgPack<T>::E : 1;
            fg_launch(ctx, straight ? rms_columns_kernel<T, true> : rms_columns_kernel<T, false>,
                      dim3((unsigned)(((uint64_t)a.cols + 32 * E - 1) / (32 * E)), chunks - c0 < 65535 ? chunks - c0 : 65535), dim3(32, 8), 0, b, (float*)w + (uint64_t)c0 * a.cols);
            FG_LAUNCHED(ctx);
        }
        fg_launch(ctx, rms_fold_kernel<T>, (unsigned)(((uint64_t)a.cols + 255) / 256), 256, 0, a, (const float*)w, chunks);
        FG_LAUNCHED(ctx);
    }
    if (!a.dx) return FG_OK;
    // dx alone leaves a thread room for 32 columns.
    const HeldPlan q = straight ? held_plan(ctx, a.rows, a.cols / FgPack<T>::E, 2 * usual, 2 * usual, 2 * usual, tensors, 512) : HeldPlan{};
    if (q.threads) return a.dsum ? launch_bwd<StraightPart<T, 2 * usual, 3>, true, false>(ctx, a, q, nullptr, 0) : launch_bwd<StraightPart<T, 2 * usual, 2>, false, false>(ctx, a, q, nullptr, 0);
    fg_launch(ctx, rms_bwd_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

// What the two forward forms ask of their arguments; y_size: bytes of an element of y.
int32_t check(fg_ctx* ctx, int32_t dtype, const RmsArgs& a, uint32_t y_size) {
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_rmsnorm_fwd: unknown dtype");
    FG_REQUIRE(ctx, a.cols >= 1, "fg_rmsnorm_fwd: cols must be >= 1");
    FG_REQUIRE(ctx, a.x && a.y, "fg_rmsnorm_fwd: NULL pointer");
    FG_REQUIRE(ctx, a.eps >= 1.17549435e-38f && a.eps <= 3.402823466e38f, "fg_rmsnorm_fwd: eps must be a normal number > 0");
    FG_REQUIRE(ctx, (uint64_t)a.rows * a.cols < (1ull << 40), "fg_rmsnorm_fwd: tensor too large");
    FG_REQUIRE(ctx, !a.sum || a.residual, "fg_rmsnorm_fwd: sum_out without a residual");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(a.x, size) && fg_at_element(a.residual, size) && fg_at_element(a.gamma, size) && fg_at_element(a.sum, size) &&
                        fg_at_element(a.y, y_size) && fg_at_element(a.rstd, 4) && fg_at_element(a.scale, 4), "fg_rmsnorm_fwd: a tensor does not start at an element");
    const uint64_t n = (uint64_t)a.rows * a.cols, bytes = n * size, line = (uint64_t)a.cols * size, column = 4ull * a.rows;
    // An output may be an input of the same type, element by element; sum and y are two tensors.
    const struct { const void* p; uint64_t n; bool matrix; } out[] = {{a.sum, bytes, true}, {a.y, n * y_size, !a.scale}, {a.rstd, column, false}, {a.scale, column * a.groups, false}};
    for (const auto& o : out) {
        FG_REQUIRE(ctx, (o.matrix && o.p == a.x) || !fg_ranges_meet(o.p, o.n, a.x, bytes), "fg_rmsnorm_fwd: an output overlaps x but is not x");
        FG_REQUIRE(ctx, (o.matrix && o.p == a.residual) || !fg_ranges_meet(o.p, o.n, a.residual, bytes), "fg_rmsnorm_fwd: an output overlaps the residual but is not it");
        FG_REQUIRE(ctx, !fg_ranges_meet(o.p, o.n, a.gamma, line), "fg_rmsnorm_fwd: an output overlaps gamma");
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j) FG_REQUIRE(ctx, !fg_ranges_meet(out[i].p, out[i].n, out[j].p, out[j].n), "fg_rmsnorm_fwd: outputs overlap");
    return FG_OK;
}

}  // namespace

extern "C" {

int32_t fg_rmsnorm_fwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* x, const void* residual, const void* gamma, float eps,
                       void* sum_out, void* y, float* rstd_out) {
    FG_ENTER(ctx);
    const RmsArgs a{x, residual, gamma, sum_out, y, rstd_out, nullptr, rows, cols, 0, 0, eps};
    const int32_t s = check(ctx, dtype, a, fg_dtype_size(dtype));
    if (s != FG_OK || rows == 0) return s;
    return FG_BY_DTYPE(dtype, rms_fwd, ctx, a);
}

int32_t fg_rmsnorm_fwd_e4m3(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* x, const void* residual, const void* gamma, float eps,
                            uint32_t group, void* sum_out, uint8_t* y, float* scale_out, float* rstd_out) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, group == 0 || group == 32 || group == 64 || group == 128 || group == 256, "fg_rmsnorm_fwd_e4m3: group must be 0, 32, 64, 128 or 256");
    FG_REQUIRE(ctx, scale_out, "fg_rmsnorm_fwd_e4m3: NULL pointer");
    const uint32_t each = group ? group : cols;
    const RmsArgs a{x, residual, gamma, sum_out, y, rstd_out, scale_out, rows, cols, each, each ? (uint32_t)(((uint64_t)cols + each - 1) / each) : 0, eps};
    const int32_t s = check(ctx, dtype, a, 1);
    if (s != FG_OK || rows == 0) return s;
    return FG_BY_DTYPE(dtype, rms_fwd, ctx, a);
}

int32_t fg_rmsnorm_bwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* x, const void* dy, const void* gamma, const float* rstd,
                       const void* dsum, void* dx, void* dgamma, int32_t accumulate_params) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_rmsnorm_bwd: unknown dtype");
    FG_REQUIRE(ctx, x && dy && rstd, "fg_rmsnorm_bwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1, "fg_rmsnorm_bwd: cols must be >= 1");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_rmsnorm_bwd: tensor too large");
    FG_REQUIRE(ctx, dx || dgamma, "fg_rmsnorm_bwd: no output");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(x, size) && fg_at_element(dy, size) && fg_at_element(gamma, size) && fg_at_element(dsum, size) && fg_at_element(dx, size) &&
                        fg_at_element(dgamma, size) && fg_at_element(rstd, 4), "fg_rmsnorm_bwd: a tensor does not start at an element");
    const uint64_t bytes = (uint64_t)rows * cols * size, line = (uint64_t)cols * size, column = 4ull * rows;
    for (const void* in : {x, dy, dsum})
        FG_REQUIRE(ctx, (dx == in || !fg_ranges_meet(dx, bytes, in, bytes)) && !fg_ranges_meet(dgamma, line, in, bytes),
                   "fg_rmsnorm_bwd: a gradient overlaps another tensor");
    FG_REQUIRE(ctx, !fg_ranges_meet(dx, bytes, gamma, line) && !fg_ranges_meet(dx, bytes, rstd, column) && !fg_ranges_meet(dgamma, line, gamma, line) &&
                        !fg_ranges_meet(dgamma, line, rstd, column) && !fg_ranges_meet(dgamma, line, dx, bytes), "fg_rmsnorm_bwd: a gradient overlaps another tensor");
    if (rows == 0) {      // an empty sum
        if (dgamma && !accumulate_params) FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(dgamma, 0, line, ctx->stream));
        return FG_OK;
    }
    return FG_BY_DTYPE(dtype, rms_bwd, ctx, RmsBwdArgs{x, dy, gamma, dsum, rstd, dx, dgamma, rows, cols, accumulate_params});
}

}  // extern "C"
