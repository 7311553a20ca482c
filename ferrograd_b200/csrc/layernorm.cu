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

template <typename T>
int32_t norm_fwd(fg_ctx* ctx, const NormArgs& a) {
    fg_launch(ctx, norm_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

template <typename T>
int32_t norm_bwd(fg_ctx* ctx, const NormBwdArgs& a) {
    float* part = nullptr;
    const uint32_t chunks = (a.rows + kChunk - 1) / kChunk;
    if (a.dgamma || a.dbeta) {      // before dx, which may be dy or x
        void* p;
        const int32_t s = fg_ws_alloc(ctx, 8ull * chunks * a.cols, &p);
        if (s != FG_OK) return s;
        part = (float*)p;
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
