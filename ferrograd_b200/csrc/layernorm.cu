// Layer norm over the rows of a matrix, forward and backward.
//
// Forward: m = sum(x) / n; then, over d = x - m, r = sum(d) / n and q = sum(d * d) / n.  r is what rounding left of the mean, so the
// mean is m + r and the variance q - r * r: rows far from zero lose nothing to the subtraction.
// Backward, with h = (x - mean) * rstd and g = dy * gamma: dx = rstd * (g - mean(g) - h * mean(g * h)); dgamma and dbeta are column
// sums of dy * h and dy.
#include "rows.cuh"

namespace {

struct NormArgs {
    const void *x, *gamma, *beta;
    void* y;
    float *mean, *rstd;
    uint32_t rows, cols;
    float eps;
};
struct NormBwdArgs {
    const void *x, *dy, *gamma;
    const float *mean, *rstd;
    void *dx, *dgamma, *dbeta;
    uint32_t rows, cols;
    int accumulate_dx, accumulate_params;
};

// ---- rows that a group of threads holds ----
// A group of warps takes a row at a time, a thread the same columns of each: pack `thread`, `thread` + threads, ... of 16 bytes.  What comes
// from memory is asked for two or three rows ahead: rows that lie straight by asynchronous copies into slots of shared memory that belong
// to the thread alone, turned rows (kShift) as loads one row ahead.
__host__ __device__ constexpr int stages_of(int packs) { return packs >= 8 ? 3 : 4; }      // by the packs of all tensors in a stage: 512 threads fit
struct Group {
    int index, threads, thread, warps, warp, lane;      // of the block's groups; a group's threads; within the group
    __device__ __forceinline__ explicit Group(int threads_) : threads(threads_) {
        warps = threads >> 5;
        index = (threadIdx.x >> 5) / warps;
        thread = threadIdx.x - index * threads;
        warp = thread >> 5;
        lane = threadIdx.x & 31;
    }
    // Two sums over the group, in all of its threads.  `red` is the group's [64] floats, another one from one call to the next.
    __device__ __forceinline__ float2 sum(float a, float b, float* red) const {
        a = fg_warp_sum(a);
        b = fg_warp_sum(b);
        if (warps == 1) return make_float2(a, b);
        if (lane == 0) { red[warp] = a; red[32 + warp] = b; }
        fg_group_barrier(index, threads);
        a = fg_warp_sum(lane < warps ? red[lane] : 0.0f);
        b = fg_warp_sum(lane < warps ? red[32 + lane] : 0.0f);
        return make_float2(a, b);
    }
};
constexpr int kMaxGroups = 8;

template <typename T, int kPacks, bool kShift>
__global__ void __launch_bounds__(512) norm_held_kernel(const NormArgs a, int threads) {
    constexpr int E = FgPack<T>::E, P = E / 2, kStages = stages_of(kPacks);
    constexpr bool kHeldParams = kPacks <= 4;      // gamma and beta stay in registers
    extern __shared__ uint4 slots[];      // [stage][pack][thread]
    __shared__ float red[kMaxGroups][4][64];
    fg_grid_enter();
    const Group group(threads);
    const uint32_t groups = blockDim.x / threads, step = gridDim.x * groups, first = blockIdx.x * groups + group.index;
    const float n = (float)a.cols, inv_n = 1.0f / n;
    const T *const x = static_cast<const T*>(a.x), *const x_end = x + (uint64_t)a.rows * a.cols, *const gamma = static_cast<const T*>(a.gamma),
            *const beta = static_cast<const T*>(a.beta);
    uint32_t col[kPacks], left[kPacks];
    uint4 gammas[kHeldParams ? kPacks : 1], betas[kHeldParams ? kPacks : 1];
    auto load_params = [&](int k, uint4& g, uint4& b) {
        g = b = make_uint4(0, 0, 0, 0);
        if (gamma && left[k]) g = fg_load_pack<T, kShift>(gamma + col[k], left[k], gamma, gamma + a.cols);
        if (beta && left[k]) b = fg_load_pack<T, kShift>(beta + col[k], left[k], beta, beta + a.cols);
    };
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
        col[k] = (group.thread + k * threads) * E;
        left[k] = col[k] < a.cols ? min((uint32_t)E, a.cols - col[k]) : 0;
        if constexpr (kHeldParams) load_params(k, gammas[k], betas[k]);
    }
    uint4 ahead[kPacks];
    auto ask = [&](uint64_t r, int stage) {
        if (r < a.rows) {
            const T* const row = x + r * a.cols;
#pragma unroll
            for (int k = 0; k < kPacks; ++k)
                if (left[k]) {
                    if constexpr (kShift) ahead[k] = fg_load_pack<T, true>(row + col[k], left[k], x, x_end);
                    else fg_copy_async(&slots[(stage * kPacks + k) * blockDim.x + threadIdx.x], row + col[k]);
                }
        }
        if constexpr (!kShift) fg_copies_end();
    };
    if constexpr (kShift) ask(first, 0);
    else
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) ask(first + (uint64_t)i * step, i);
    int stage = 0, turn = 0;
    for (uint64_t r = first; r < a.rows; r += step) {
        float2 v[kPacks][P];
        if constexpr (!kShift) fg_copies_wait<kStages - 2>();
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (left[k]) {
                if constexpr (kShift) w = ahead[k];
                else w = slots[(stage * kPacks + k) * blockDim.x + threadIdx.x];
            }
            FgPack<T>::widen(w, v[k]);
            if (kShift && left[k] < E)
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    if (2 * e >= left[k]) v[k][e].x = 0.0f;
                    if (2 * e + 1 >= left[k]) v[k][e].y = 0.0f;
                }
#pragma unroll
            for (int e = 0; e < P; ++e) s = fg_add2(s, v[k][e]);
        }
        if constexpr (kShift) ask(r + step, 0);
        else ask(r + (uint64_t)(kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
        const float m = group.sum(s.x + s.y, 0.0f, red[group.index][turn]).x / n;
        const float2 less = make_float2(-m, -m);
        float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
#pragma unroll
            for (int e = 0; e < P; ++e) v[k][e] = fg_add2(v[k][e], less);
            if (left[k] < E)      // columns behind the row's end count for nothing
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    if (2 * e >= left[k]) v[k][e].x = 0.0f;
                    if (2 * e + 1 >= left[k]) v[k][e].y = 0.0f;
                }
#pragma unroll
            for (int e = 0; e < P; ++e) {
                s1 = fg_add2(s1, v[k][e]);
                s2 = fg_fma2(v[k][e], v[k][e], s2);
            }
        }
        const float2 t = group.sum(s1.x + s1.y, s2.x + s2.y, red[group.index][turn + 1]);
        const float rest = t.x * inv_n, rstd = 1.0f / sqrtf(fmaxf(__fmaf_rn(-rest, rest, t.y * inv_n), 0.0f) + a.eps);
        T* const out = static_cast<T*>(a.y) + r * a.cols;
        const float2 less_rest = make_float2(-rest, -rest), by = make_float2(rstd, rstd);
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            if (!kShift && !left[k]) continue;      // (turned rows are stored by whole warps)
            uint4 gw, bw;
            if constexpr (kHeldParams) { gw = gammas[k]; bw = betas[k]; }
            else load_params(k, gw, bw);
            float2 g[P], b[P];
            FgPack<T>::widen(gw, g);
            FgPack<T>::widen(bw, b);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float2 h = fg_mul2(fg_add2(v[k][e], less_rest), by);
                g[e] = gamma ? fg_fma2(h, g[e], b[e]) : fg_add2(h, b[e]);
            }
            fg_store_pack<T, kShift>(out + col[k], FgPack<T>::narrow(g), left[k]);
        }
        if (group.thread == 0) {
            if (a.mean) a.mean[r] = m + rest;
            if (a.rstd) a.rstd[r] = rstd;
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
        turn ^= 2;
    }
}

// The backward pass the same way, 16 columns at most per thread.  With the gradients of the parameters (kParams) a thread sums its columns
// over the rows of its group, a block adds its groups and leaves one row of parts: [block][2][pitch].
// With c = x - mean, dx = rstd * g + (-rstd * m1) + c * (-rstd^2 * m2), where m1 and m2 are the means of g and of g * h.
template <typename T, int kPacks, bool kShift, bool kParams>
__global__ void __launch_bounds__(512) norm_bwd_held_kernel(const NormBwdArgs a, int threads, float* parts, uint32_t pitch) {
    constexpr int E = FgPack<T>::E, P = E / 2, kStages = stages_of(2 * kPacks);
    extern __shared__ uint4 slots[];      // [stage][x, dy][pack][thread]; at the end the groups' sums
    __shared__ float red[kMaxGroups][2][64];
    fg_grid_enter();
    const Group group(threads);
    const uint32_t groups = blockDim.x / threads, step = gridDim.x * groups, first = blockIdx.x * groups + group.index;
    const float inv_n = 1.0f / (float)a.cols;
    const uint64_t size = (uint64_t)a.rows * a.cols;
    const T *const x = static_cast<const T*>(a.x), *const dy = static_cast<const T*>(a.dy), *const gamma = static_cast<const T*>(a.gamma);
    T* const dx = static_cast<T*>(a.dx);
    uint32_t col[kPacks], left[kPacks];
    uint4 gammas[kPacks];
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
        col[k] = (group.thread + k * threads) * E;
        left[k] = col[k] < a.cols ? min((uint32_t)E, a.cols - col[k]) : 0;
        gammas[k] = make_uint4(0, 0, 0, 0);
        if (gamma && left[k]) gammas[k] = fg_load_pack<T, kShift>(gamma + col[k], left[k], gamma, gamma + a.cols);
    }
    uint4 ahead[2][kPacks];
    float mean = 0.0f, rstd = 0.0f;
    auto ask = [&](uint64_t r, int stage) {
        if (r < a.rows) {
            const T *const x_row = x + r * a.cols, *const dy_row = dy + r * a.cols;
#pragma unroll
            for (int k = 0; k < kPacks; ++k)
                if (left[k]) {
                    if constexpr (kShift) {
                        ahead[0][k] = fg_load_pack<T, true>(x_row + col[k], left[k], x, x + size);
                        ahead[1][k] = fg_load_pack<T, true>(dy_row + col[k], left[k], dy, dy + size);
                    } else {
                        fg_copy_async(&slots[(stage * 2 * kPacks + k) * blockDim.x + threadIdx.x], x_row + col[k]);
                        fg_copy_async(&slots[((stage * 2 + 1) * kPacks + k) * blockDim.x + threadIdx.x], dy_row + col[k]);
                    }
                }
        }
        if constexpr (!kShift) fg_copies_end();
    };
    auto ask_row = [&](uint64_t r) {
        if (r < a.rows) { mean = a.mean[r]; rstd = a.rstd[r]; }
    };
    if constexpr (kShift) ask(first, 0);
    else
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) ask(first + (uint64_t)i * step, i);
    ask_row(first);
    float2 dg[kPacks][P], db[kPacks][P];
#pragma unroll
    for (int k = 0; k < kPacks; ++k)
#pragma unroll
        for (int e = 0; e < P; ++e) dg[k][e] = db[k][e] = make_float2(0.0f, 0.0f);
    int stage = 0, turn = 0;
    for (uint64_t r = first; r < a.rows; r += step) {
        float2 c[kPacks][P], g[kPacks][P];
        const float m = mean, sd = rstd;
        const float2 less = make_float2(-m, -m), by = make_float2(sd, sd);
        ask_row(r + step);
        if constexpr (!kShift) fg_copies_wait<kStages - 2>();
        float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            uint4 v = make_uint4(0, 0, 0, 0), w = v;
            if (left[k]) {
                if constexpr (kShift) { v = ahead[0][k]; w = ahead[1][k]; }
                else {
                    v = slots[(stage * 2 * kPacks + k) * blockDim.x + threadIdx.x];
                    w = slots[((stage * 2 + 1) * kPacks + k) * blockDim.x + threadIdx.x];
                }
            }
            FgPack<T>::widen(v, c[k]);
            FgPack<T>::widen(w, g[k]);
            float2 gm[P];
            FgPack<T>::widen(gammas[k], gm);
#pragma unroll
            for (int e = 0; e < P; ++e) c[k][e] = fg_add2(c[k][e], less);
            if (left[k] < E)      // columns behind the row's end count for nothing
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    if (2 * e >= left[k]) c[k][e].x = g[k][e].x = 0.0f;
                    if (2 * e + 1 >= left[k]) c[k][e].y = g[k][e].y = 0.0f;
                }
#pragma unroll
            for (int e = 0; e < P; ++e) {
                if (kParams) {
                    dg[k][e] = fg_fma2(g[k][e], fg_mul2(c[k][e], by), dg[k][e]);
                    db[k][e] = fg_add2(db[k][e], g[k][e]);
                }
                if (gamma) g[k][e] = fg_mul2(g[k][e], gm[e]);
                s1 = fg_add2(s1, g[k][e]);
                s2 = fg_fma2(g[k][e], c[k][e], s2);
            }
        }
        if constexpr (kShift) ask(r + step, 0);
        else ask(r + (uint64_t)(kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
        if (dx) {
            const float2 t = group.sum(s1.x + s1.y, s2.x + s2.y, red[group.index][turn]);
            const float u1 = -sd * (t.x * inv_n), u2 = -sd * sd * (sd * (t.y * inv_n));
            const float2 add = make_float2(u1, u1), slope = make_float2(u2, u2);
            T* const row = dx + r * a.cols;
#pragma unroll
            for (int k = 0; k < kPacks; ++k) {
                if (!kShift && !left[k]) continue;
#pragma unroll
                for (int e = 0; e < P; ++e) g[k][e] = fg_fma2(g[k][e], by, fg_fma2(c[k][e], slope, add));
                if (a.accumulate_dx) {
                    float2 old[P];
                    FgPack<T>::widen(left[k] ? fg_load_pack<T, kShift>(row + col[k], left[k], dx, dx + size) : make_uint4(0, 0, 0, 0), old);
                    if (kShift) __syncwarp();      // a lane writes words that others have read
#pragma unroll
                    for (int e = 0; e < P; ++e) g[k][e] = fg_add2(g[k][e], old[e]);
                }
                fg_store_pack<T, kShift>(row + col[k], FgPack<T>::narrow(g[k]), left[k]);
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
        turn ^= 1;
    }
    if constexpr (kParams) {
        // the groups one after the other, in shared memory: [2][pack][pair][thread]
        float2* const sums = reinterpret_cast<float2*>(slots);
        if constexpr (!kShift) fg_copies_wait<0>();
        for (uint32_t i = 0; i + 1 < groups; ++i) {
            __syncthreads();
            if (group.index == (int)i)
#pragma unroll
                for (int k = 0; k < kPacks; ++k)
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        float2 *const p = sums + (k * P + e) * threads + group.thread, *const q = p + kPacks * P * threads;
                        *p = i ? fg_add2(*p, dg[k][e]) : dg[k][e];
                        *q = i ? fg_add2(*q, db[k][e]) : db[k][e];
                    }
        }
        __syncthreads();
        if (group.index + 1 == (int)groups) {
            float* const mine = parts + (uint64_t)blockIdx.x * 2 * pitch;
#pragma unroll
            for (int k = 0; k < kPacks; ++k)
                if (left[k])
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const float2 *const p = sums + (k * P + e) * threads + group.thread, *const q = p + kPacks * P * threads;
                        *reinterpret_cast<float2*>(mine + col[k] + 2 * e) = groups > 1 ? fg_add2(*p, dg[k][e]) : dg[k][e];
                        *reinterpret_cast<float2*>(mine + pitch + col[k] + 2 * e) = groups > 1 ? fg_add2(*q, db[k][e]) : db[k][e];
                    }
        }
    }
}

// Adds the blocks' parts: 128 columns per block, a warp takes every 32nd part.  pitch is a multiple of 128.
template <typename T>
__global__ void __launch_bounds__(1024) norm_parts_kernel(const NormBwdArgs a, const float* parts, uint32_t count, uint32_t pitch) {
    __shared__ float4 red[32][32];
    fg_grid_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t at = blockIdx.x * 128 + 4 * lane;      // dgamma's columns, then dbeta's
    T* const out = static_cast<T*>(at < pitch ? a.dgamma : a.dbeta);
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t i0 = warp; i0 < count; i0 += 32 * 8) {
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = i0 + 32 * j < count ? *reinterpret_cast<const float4*>(parts + (uint64_t)(i0 + 32 * j) * 2 * pitch + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 8; ++j) { s.x += v[j].x; s.y += v[j].y; s.z += v[j].z; s.w += v[j].w; }
    }
    red[warp][lane] = s;
    __syncthreads();
    if (threadIdx.x < 128) {
        const uint32_t c = blockIdx.x * 128 + threadIdx.x - (at < pitch ? 0 : pitch);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 32; ++w) sum += reinterpret_cast<const float*>(red[w])[threadIdx.x];
        if (out && c < a.cols) out[c] = fg_narrow<T>(a.accumulate_params ? fg_widen(out[c]) + sum : sum);
    }
}

// Any row: one block each, the row read once per sum.
template <typename T>
__global__ void __launch_bounds__(256) norm_stream_kernel(const NormArgs a) {
    __shared__ float red[64];
    fg_grid_enter();
    const float n = (float)a.cols;
    const T *gamma = static_cast<const T*>(a.gamma), *beta = static_cast<const T*>(a.beta);
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + (uint64_t)r * a.cols;
        T* y = static_cast<T*>(a.y) + (uint64_t)r * a.cols;
        float s = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) s += fg_widen(x[c]);
        const float m = fg_block_sum2(s, 0.0f, red).x / n;
        float s1 = 0.0f, s2 = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float d = fg_widen(x[c]) - m;
            s1 += d;
            s2 = __fmaf_rn(d, d, s2);
        }
        const float2 t = fg_block_sum2(s1, s2, red);
        const float rest = t.x / n, rstd = 1.0f / sqrtf(fmaxf(__fmaf_rn(-rest, rest, t.y / n), 0.0f) + a.eps);
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float h = ((fg_widen(x[c]) - m) - rest) * rstd;
            y[c] = fg_narrow<T>(__fmaf_rn(h, gamma ? fg_widen(gamma[c]) : 1.0f, beta ? fg_widen(beta[c]) : 0.0f));
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = m + rest;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_bwd_stream_kernel(const NormBwdArgs a) {
    __shared__ float red[64];
    fg_grid_enter();
    const float n = (float)a.cols;
    const T* gamma = static_cast<const T*>(a.gamma);
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const uint64_t at = (uint64_t)r * a.cols;
        const T *x = static_cast<const T*>(a.x) + at, *dy = static_cast<const T*>(a.dy) + at;
        T* dx = static_cast<T*>(a.dx) + at;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float g = fg_widen(dy[c]) * (gamma ? fg_widen(gamma[c]) : 1.0f);
            s1 += g;
            s2 = __fmaf_rn(g, (fg_widen(x[c]) - mean) * rstd, s2);
        }
        const float2 t = fg_block_sum2(s1, s2, red);
        const float m1 = t.x / n, m2 = t.y / n;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float g = fg_widen(dy[c]) * (gamma ? fg_widen(gamma[c]) : 1.0f), h = (fg_widen(x[c]) - mean) * rstd;
            const float v = rstd * __fmaf_rn(-h, m2, g - m1);
            dx[c] = fg_narrow<T>(a.accumulate_dx ? fg_widen(dx[c]) + v : v);
        }
    }
}

// Column sums of dy * h and dy over a chunk of rows: 32 columns by 8 rows per block.  part: [2][chunks][cols].
constexpr uint32_t kChunk = 256;
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormBwdArgs a, float* part) {
    __shared__ float red[2][8][32];
    fg_grid_enter();
    const uint64_t c = (uint64_t)blockIdx.x * 32 + threadIdx.x, chunks = gridDim.y;
    const uint32_t r0 = blockIdx.y * kChunk, r1 = min(a.rows, r0 + kChunk);
    float s1 = 0.0f, s2 = 0.0f;
    if (c < a.cols)
        for (uint32_t r = r0 + threadIdx.y; r < r1; r += 8) {
            const float dy = fg_widen(static_cast<const T*>(a.dy)[(uint64_t)r * a.cols + c]);
            s1 = __fmaf_rn(dy, (fg_widen(static_cast<const T*>(a.x)[(uint64_t)r * a.cols + c]) - a.mean[r]) * a.rstd[r], s1);
            s2 += dy;
        }
    red[0][threadIdx.y][threadIdx.x] = s1;
    red[1][threadIdx.y][threadIdx.x] = s2;
    __syncthreads();
    if (threadIdx.y < 2 && c < a.cols) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += red[threadIdx.y][i][threadIdx.x];
        part[(threadIdx.y * chunks + blockIdx.y) * a.cols + c] = s;
    }
}
template <typename T>
__global__ void __launch_bounds__(256) norm_fold_kernel(const NormBwdArgs a, const float* part, uint32_t chunks) {
    fg_grid_enter();
    const uint64_t c = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    T* out = static_cast<T*>(blockIdx.y == 0 ? a.dgamma : a.dbeta);
    if (c >= a.cols || !out) return;
    part += (uint64_t)blockIdx.y * chunks * a.cols;
    float s = 0.0f;
    for (uint32_t i = 0; i < chunks; ++i) s += part[(uint64_t)i * a.cols + c];
    out[c] = fg_narrow<T>(a.accumulate_params ? fg_widen(out[c]) + s : s);
}

int rows_grid(const fg_ctx* ctx, uint32_t rows) { return (int)(rows < 8u * ctx->sm_count ? rows : 8u * ctx->sm_count); }

// How a kernel that holds rows is launched: packs per thread, the threads of a group, the groups of a block, its shared memory, the blocks.
struct HeldPlan { int packs, threads, groups; size_t bytes; int grid; };
// A block has 256 threads or, for a longer row, up to 512.  Threads hold up to `most` packs; of few rows, and where a warp is enough, one.
HeldPlan held_plan(const fg_ctx* ctx, uint32_t rows, uint32_t cols, uint32_t elements, int most, int slots) {
    const uint64_t packs = ((uint64_t)cols + elements - 1) / elements;
    HeldPlan p{1, 0, 1, 0, 0};
    while (p.packs < most && (packs > 512ull * p.packs || (p.packs < 4 && rows > 2u * ctx->sm_count && packs > 32ull * p.packs))) p.packs *= 2;
    if (packs > 512ull * p.packs) return p;      // threads = 0: no
    p.threads = (int)((packs + 32 * p.packs - 1) / (32 * p.packs) * 32);
    p.groups = 256 / p.threads < 1 ? 1 : 256 / p.threads;
    while (p.groups > 1 && (uint64_t)rows * 2 <= (uint64_t)p.groups * ctx->sm_count) p.groups /= 2;      // few rows: over the SMs first
    p.bytes = sizeof(uint4) * stages_of(slots * p.packs) * slots * p.packs * p.threads * p.groups;
    // What the SMs hold at once: 512 threads of 128 registers, 220 KB with the static part.
    const uint64_t by_threads = 512 / (p.threads * p.groups), by_memory = 220 * 1024 / (p.bytes + 9 * 1024), per_sm = by_threads < by_memory ? by_threads : by_memory;
    const uint64_t need = ((uint64_t)rows + p.groups - 1) / p.groups, cap = (uint64_t)ctx->sm_count * (per_sm ? per_sm : 1);
    p.grid = (int)(need < cap ? need : cap);
    return p;
}
template <typename K>
int32_t allow_shared(fg_ctx* ctx, K kernel, size_t bytes) {
    if (bytes > 32 * 1024) FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return FG_OK;
}

template <typename T, int kPacks, bool kShift>
int32_t launch_held(fg_ctx* ctx, const NormArgs& a, HeldPlan p) {
    const size_t bytes = p.bytes;
    const int32_t s = allow_shared(ctx, norm_held_kernel<T, kPacks, kShift>, bytes);
    if (s != FG_OK) return s;
    fg_launch(ctx, norm_held_kernel<T, kPacks, kShift>, p.grid, p.threads * p.groups, bytes, a, p.threads);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T, bool kShift>
int32_t choose_held(fg_ctx* ctx, const NormArgs& a, HeldPlan p) {
    return p.packs == 1 ? launch_held<T, 1, kShift>(ctx, a, p) : p.packs == 2 ? launch_held<T, 2, kShift>(ctx, a, p)
           : p.packs == 4 ? launch_held<T, 4, kShift>(ctx, a, p) : launch_held<T, 8, kShift>(ctx, a, p);
}
template <typename T>
int32_t norm_fwd(fg_ctx* ctx, const NormArgs& a) {
    const bool straight = fg_rows_lie_straight(a.cols, sizeof(T), a.x, a.y, a.gamma, a.beta);
    const HeldPlan p = held_plan(ctx, a.rows, a.cols, FgPack<T>::E, 8, straight ? 1 : 0);
    if (p.threads) return straight ? choose_held<T, false>(ctx, a, p) : choose_held<T, true>(ctx, a, p);
    fg_launch(ctx, norm_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

template <typename T, int kPacks, bool kShift, bool kParams>
int32_t launch_bwd_held(fg_ctx* ctx, const NormBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch) {
    const size_t sums = kParams && p.groups > 1 ? 8ull * FgPack<T>::E * kPacks * p.threads : 0, bytes = p.bytes < sums ? sums : p.bytes;
    const int32_t s = allow_shared(ctx, norm_bwd_held_kernel<T, kPacks, kShift, kParams>, bytes);
    if (s != FG_OK) return s;
    fg_launch(ctx, norm_bwd_held_kernel<T, kPacks, kShift, kParams>, p.grid, p.threads * p.groups, bytes, a, p.threads, parts, pitch);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T, int kPacks>
int32_t choose_bwd_held(fg_ctx* ctx, const NormBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch, bool straight) {
    if (parts) return straight ? launch_bwd_held<T, kPacks, false, true>(ctx, a, p, parts, pitch) : launch_bwd_held<T, kPacks, true, true>(ctx, a, p, parts, pitch);
    return straight ? launch_bwd_held<T, kPacks, false, false>(ctx, a, p, parts, pitch) : launch_bwd_held<T, kPacks, true, false>(ctx, a, p, parts, pitch);
}

template <typename T>
int32_t norm_bwd(fg_ctx* ctx, const NormBwdArgs& a) {
    const bool straight = fg_rows_lie_straight(a.cols, sizeof(T), a.x, a.dy, a.gamma, a.dx);
    const HeldPlan p = held_plan(ctx, a.rows, a.cols, FgPack<T>::E, sizeof(T) == 4 ? 4 : 2, straight ? 2 : 0);
    if (p.threads) {
        float* parts = nullptr;
        const uint32_t pitch = (a.cols + 127) / 128 * 128;
        if (a.dgamma || a.dbeta) {
            void* w;
            const int32_t s = fg_ws_alloc(ctx, 8ull * pitch * p.grid, &w);
            if (s != FG_OK) return s;
            parts = (float*)w;
        }
        int32_t s = FG_OK;
        if (p.packs == 1) s = choose_bwd_held<T, 1>(ctx, a, p, parts, pitch, straight);
        else if (p.packs == 2) s = choose_bwd_held<T, 2>(ctx, a, p, parts, pitch, straight);
        else if constexpr (sizeof(T) == 4) s = choose_bwd_held<T, 4>(ctx, a, p, parts, pitch, straight);
        if (s != FG_OK || !parts) return s;
        fg_launch(ctx, norm_parts_kernel<T>, pitch / 64, 1024, 0, a, (const float*)parts, (uint32_t)p.grid, pitch);
        FG_LAUNCHED(ctx);
        return FG_OK;
    }
    float* part = nullptr;
    const uint32_t chunks = (a.rows + kChunk - 1) / kChunk;
    if (a.dgamma || a.dbeta) {      // before dx, which may be dy or x
        void* w;
        const int32_t s = fg_ws_alloc(ctx, 8ull * chunks * a.cols, &w);
        if (s != FG_OK) return s;
        part = (float*)w;
        fg_launch(ctx, norm_columns_kernel<T>, dim3((a.cols + 31) / 32, chunks), dim3(32, 8), 0, a, part);
        FG_LAUNCHED(ctx);
        fg_launch(ctx, norm_fold_kernel<T>, dim3((a.cols + 255) / 256, 2), 256, 0, a, (const float*)part, chunks);
        FG_LAUNCHED(ctx);
    }
    if (a.dx) {
        fg_launch(ctx, norm_bwd_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
        FG_LAUNCHED(ctx);
    }
    return FG_OK;
}

}  // namespace

extern "C" {

int32_t fg_layernorm_fwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* x, const void* gamma, const void* beta,
                         float eps, void* y, float* mean_out, float* rstd_out) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_layernorm_fwd: unknown dtype");
    FG_REQUIRE(ctx, x && y, "fg_layernorm_fwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1, "fg_layernorm_fwd: cols must be >= 1");
    FG_REQUIRE(ctx, eps >= 0.0f && eps <= 3.402823466e38f, "fg_layernorm_fwd: eps must be a number >= 0");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_layernorm_fwd: tensor too large");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(x, size) && fg_at_element(y, size) && fg_at_element(gamma, size) && fg_at_element(beta, size) &&
                        fg_at_element(mean_out, 4) && fg_at_element(rstd_out, 4), "fg_layernorm_fwd: a tensor does not start at an element");
    const uint64_t bytes = (uint64_t)rows * cols * size;
    FG_REQUIRE(ctx, y == x || !fg_ranges_meet(x, bytes, y, bytes), "fg_layernorm_fwd: y overlaps x but is not x");
    if (rows == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, norm_fwd, ctx, NormArgs{x, gamma, beta, y, mean_out, rstd_out, rows, cols, eps});
}

int32_t fg_layernorm_bwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* x, const void* dy, const void* gamma,
                         const float* mean, const float* rstd, void* dx, void* dgamma, void* dbeta, int32_t accumulate_dx,
                         int32_t accumulate_params) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_layernorm_bwd: unknown dtype");
    FG_REQUIRE(ctx, x && dy && mean && rstd, "fg_layernorm_bwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1, "fg_layernorm_bwd: cols must be >= 1");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_layernorm_bwd: tensor too large");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(x, size) && fg_at_element(dy, size) && fg_at_element(gamma, size) && fg_at_element(dx, size) &&
                        fg_at_element(dgamma, size) && fg_at_element(dbeta, size) && fg_at_element(mean, 4) && fg_at_element(rstd, 4),
               "fg_layernorm_bwd: a tensor does not start at an element");
    FG_REQUIRE(ctx, !accumulate_dx || (dx != dy && dx != x), "fg_layernorm_bwd: accumulate_dx needs a dx of its own");
    const uint64_t bytes = (uint64_t)rows * cols * size;
    FG_REQUIRE(ctx, (dx == x || !fg_ranges_meet(x, bytes, dx, bytes)) && (dx == dy || !fg_ranges_meet(dy, bytes, dx, bytes)),
               "fg_layernorm_bwd: dx overlaps x or dy but is neither");
    if (rows == 0) {      // empty sums
        if (dgamma && !accumulate_params) FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(dgamma, 0, (uint64_t)cols * size, ctx->stream));
        if (dbeta && !accumulate_params) FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(dbeta, 0, (uint64_t)cols * size, ctx->stream));
        return FG_OK;
    }
    return FG_BY_DTYPE(dtype, norm_bwd, ctx,
                       NormBwdArgs{x, dy, gamma, mean, rstd, dx, dgamma, dbeta, rows, cols, accumulate_dx, accumulate_params});
}

}  // extern "C"
