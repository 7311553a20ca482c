// Root-mean-square norm over the rows of a matrix, with the addition of a residual before it, and its backward pass.
//
// Forward: h = x + residual, rounded to the storage type; y = h * rstd * gamma with rstd = 1 / sqrt(mean(h * h) + eps).  The 8-bit form writes
// y / s in e4m3 for each group of columns, s = largest |y| of the group / 448 (448: the largest number of e4m3).
// Backward, with n = h * rstd and g = dy * gamma: dh = dsum + rstd * (g - n * mean(g * n)), which is the gradient of x and of the residual;
// dgamma = column sums of dy * n.
#include <cuda_fp8.h>

#include <atomic>

#include "rows.cuh"

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

// y / s in e4m3; s that has no finite reciprocal divides.
__device__ __forceinline__ uint8_t to_e4m3(float y, float s) {
    const float v = s > 0.0f ? (s > 1e-37f ? y * (1.0f / s) : y / s) : y * 0.0f;
    return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// Any row: one block each.
template <typename T, bool k8>
__global__ void __launch_bounds__(256) rms_stream_kernel(const RmsArgs a) {
    __shared__ float red[64];
    fg_grid_enter();
    const T* const gamma = static_cast<const T*>(a.gamma);
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const uint64_t at = (uint64_t)r * a.cols;
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
                    if (lane == 0) a.scale[(uint64_t)r * a.groups + g] = scale;
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
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const uint64_t at = (uint64_t)r * a.cols;
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

// dgamma by columns, over chunks of rows: part is [chunks][cols].
constexpr uint32_t kChunk = 256;
template <typename T>
__global__ void __launch_bounds__(256) rms_columns_kernel(const RmsBwdArgs a, float* part) {
    __shared__ float red[8][32];
    fg_grid_enter();
    const uint64_t c = (uint64_t)blockIdx.x * 32 + threadIdx.x;
    const uint32_t r0 = blockIdx.y * kChunk, r1 = min(a.rows, r0 + kChunk);
    float s = 0.0f;
    if (c < a.cols)
        for (uint32_t r = r0 + threadIdx.y; r < r1; r += 8) {
            const uint64_t at = (uint64_t)r * a.cols + c;
            s = __fmaf_rn(fg_widen(static_cast<const T*>(a.dy)[at]), fg_widen(static_cast<const T*>(a.x)[at]) * a.rstd[r], s);
        }
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < a.cols) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
        part[(uint64_t)blockIdx.y * a.cols + c] = s;
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

int rows_grid(const fg_ctx* ctx, uint32_t rows) { return (int)(rows < 8u * ctx->sm_count ? rows : 8u * ctx->sm_count); }

template <typename T>
int32_t rms_fwd(fg_ctx* ctx, const RmsArgs& a) {
    fg_launch(ctx, a.scale ? rms_stream_kernel<T, true> : rms_stream_kernel<T, false>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T>
int32_t rms_bwd(fg_ctx* ctx, const RmsBwdArgs& a) {
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
            fg_launch(ctx, rms_columns_kernel<T>, dim3((unsigned)(((uint64_t)a.cols + 31) / 32), chunks - c0 < 65535 ? chunks - c0 : 65535), dim3(32, 8), 0, b,
                      (float*)w + (uint64_t)c0 * a.cols);
            FG_LAUNCHED(ctx);
        }
        fg_launch(ctx, rms_fold_kernel<T>, (unsigned)(((uint64_t)a.cols + 255) / 256), 256, 0, a, (const float*)w, chunks);
        FG_LAUNCHED(ctx);
    }
    if (!a.dx) return FG_OK;
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
