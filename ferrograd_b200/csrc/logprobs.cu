// Log probabilities of given tokens, with the rows' entropies and largest entries, and the gradient of the logits.
//
// With z = scale * x, m the largest z of the row and l = sum(exp(z - m)): lse = m + log l, logprob = z[target] - lse and
// entropy = log l - sum(exp(z - m) * (z - m)) / l.  The gradient, of dlogprob and dentropy: dx_c = scale * (dlogprob * ([c == target] - p_c) -
// dentropy * p_c * (log p_c + entropy)) with p_c = exp(z_c - lse).
#include <atomic>

#include "rows.cuh"

namespace {

constexpr uint32_t kMaxTop = 64;

struct LogprobArgs {
    const void* x;
    const uint32_t* targets;
    uint32_t rows, cols, top;
    float scale;
    float *logprob, *entropy, *lse;
    uint32_t* top_ids;
    float* top_logprobs;
};
struct LogprobBwdArgs {
    const void* x;
    const uint32_t* targets;
    const float *lse, *entropy, *dlogprob, *dentropy;
    void* dx;
    uint32_t rows, cols;
    float scale;
};

// The largest z, the sum of weights and the sum of weights times distances of a part of a row.
struct Part {
    float m, l, e;
    // Another part.  sum w (z - top) = sum w (z - m) + l (m - top); a part whose weights vanish beside the other's adds nothing, whatever its distance.
    __device__ __forceinline__ void join(const Part& o) {
        const float top = fmaxf(m, o.m);
        if (top == -INFINITY) {      // no weight, unless it is NaN
            l += o.l;
            return;
        }
        const float d = m - top, od = o.m - top, w = __expf(d), ow = __expf(od);
        e = (w == 0.0f ? 0.0f : w * __fmaf_rn(l, d, e)) + (ow == 0.0f ? 0.0f : ow * __fmaf_rn(o.l, od, o.e));
        l = __fmaf_rn(l, w, o.l * ow);
        m = top;
    }
};
// NaN has to come out of the sums: a largest value that is NaN hides behind fmaxf.
__device__ __forceinline__ Part block_join(Part p, float* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Part q{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.l, o), __shfl_xor_sync(0xffffffffu, p.e, o)};
        p.join(q);
    }
    if (lane == 0) { red[warp] = p.m; red[32 + warp] = p.l; red[64 + warp] = p.e; }
    __syncthreads();
    p = lane < nw ? Part{red[lane], red[32 + lane], red[64 + lane]} : Part{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Part q{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.l, o), __shfl_xor_sync(0xffffffffu, p.e, o)};
        p.join(q);
    }
    __syncthreads();
    return p;
}

// Any row: one block each, read once for the largest, once for the sums and once for every entry asked for.
template <typename T>
__global__ void __launch_bounds__(256) logprob_stream_kernel(const LogprobArgs a) {
    __shared__ float red[96];
    __shared__ unsigned long long best[8];
    fg_grid_enter();
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + (uint64_t)r * a.cols;
        const uint32_t target = a.targets ? a.targets[r] : 0;
        if (target >= a.cols) {      // padding
            if (threadIdx.x == 0) {
                if (a.logprob) a.logprob[r] = 0.0f;
                if (a.entropy) a.entropy[r] = 0.0f;
                if (a.lse) a.lse[r] = 0.0f;
            }
            for (uint32_t i = threadIdx.x; i < a.top; i += 256) {
                a.top_ids[(uint64_t)r * a.top + i] = FG_NO_TOKEN;
                a.top_logprobs[(uint64_t)r * a.top + i] = -INFINITY;
            }
            continue;
        }
        float m = -INFINITY;
        for (uint32_t c = threadIdx.x; c < a.cols; c += 256) m = fmaxf(m, fg_widen(x[c]) * a.scale);
        float l = 0.0f, e = 0.0f;
        for (uint32_t c = threadIdx.x; c < a.cols; c += 256) {
            const float d = fg_widen(x[c]) * a.scale - (m == -INFINITY ? 0.0f : m), w = __expf(d);
            l += w;
            if (w != 0.0f) e = __fmaf_rn(w, d, e);      // (a weight of zero times -inf)
        }
        const Part p = block_join(Part{m, l, e}, red);
        const float log_l = logf(p.l), lse = p.m + log_l;
        if (threadIdx.x == 0) {
            if (a.logprob) a.logprob[r] = p.l == 0.0f ? -INFINITY : fg_widen(x[target]) * a.scale - p.m - log_l;
            if (a.entropy) a.entropy[r] = p.l == 0.0f ? 0.0f : log_l - p.e / p.l;
            if (a.lse) a.lse[r] = lse;
        }
        unsigned long long last = ~0ull;      // key of the entry before: larger keys come first, of equal values the lowest index
        for (uint32_t i = 0; i < a.top; ++i) {
            unsigned long long mine = 0;
            for (uint32_t c = threadIdx.x; c < a.cols; c += 256) {
                const float v = fg_widen(x[c]);
                if (!(v > -INFINITY)) continue;
                const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
                const unsigned long long key = (unsigned long long)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - c);
                if (key < last && key > mine) mine = key;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
                if (other > mine) mine = other;
            }
            if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = mine;
            __syncthreads();
            for (int w = 0; w < 8; ++w)
                if (best[w] > mine) mine = best[w];
            __syncthreads();
            if (threadIdx.x == 0) {
                const uint32_t c = 0xffffffffu - (uint32_t)mine;
                a.top_ids[(uint64_t)r * a.top + i] = mine ? c : FG_NO_TOKEN;
                a.top_logprobs[(uint64_t)r * a.top + i] = mine ? fg_widen(x[c]) * a.scale - p.m - log_l : -INFINITY;
            }
            last = mine;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) logprob_bwd_stream_kernel(const LogprobBwdArgs a) {
    fg_grid_enter();
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + (uint64_t)r * a.cols;
        T* const dx = static_cast<T*>(a.dx) + (uint64_t)r * a.cols;
        const uint32_t target = a.targets ? a.targets[r] : 0;
        const float lse = a.lse[r];
        if (target >= a.cols || lse == -INFINITY) {
            for (uint32_t c = threadIdx.x; c < a.cols; c += 256) dx[c] = fg_narrow<T>(0.0f);
            continue;
        }
        const float gl = a.dlogprob ? a.scale * a.dlogprob[r] : 0.0f, ge = a.dentropy ? a.scale * a.dentropy[r] : 0.0f;
        const float h = a.dentropy ? a.entropy[r] : 0.0f;
        for (uint32_t c = threadIdx.x; c < a.cols; c += 256) {
            const float logp = fg_widen(x[c]) * a.scale - lse, p = __expf(logp);
            float g = p == 0.0f ? 0.0f : p * __fmaf_rn(-ge, logp + h, -gl);
            if (c == target && a.targets) g += gl;
            dx[c] = fg_narrow<T>(g);
        }
    }
}

int rows_grid(const fg_ctx* ctx, uint32_t rows) { return (int)(rows < 8u * ctx->sm_count ? rows : 8u * ctx->sm_count); }

template <typename T>
int32_t logprobs_fwd(fg_ctx* ctx, const LogprobArgs& a) {
    fg_launch(ctx, logprob_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T>
int32_t logprobs_bwd(fg_ctx* ctx, const LogprobBwdArgs& a) {
    fg_launch(ctx, logprob_bwd_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

}  // namespace

extern "C" {

int32_t fg_logprobs_fwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* logits, const uint32_t* targets, float scale,
                        float* logprob_out, float* entropy_out, float* lse_out, uint32_t top, uint32_t* top_ids_out, float* top_logprobs_out) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_logprobs_fwd: unknown dtype");
    FG_REQUIRE(ctx, logits, "fg_logprobs_fwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1, "fg_logprobs_fwd: cols must be >= 1");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_logprobs_fwd: tensor too large");
    FG_REQUIRE(ctx, scale > 0.0f && scale <= 3.402823466e38f, "fg_logprobs_fwd: scale must be a number > 0");
    FG_REQUIRE(ctx, !logprob_out || targets, "fg_logprobs_fwd: logprob_out without targets");
    FG_REQUIRE(ctx, top <= kMaxTop && top <= cols, "fg_logprobs_fwd: top must be at most 64 and at most cols");
    FG_REQUIRE(ctx, !top || (top_ids_out && top_logprobs_out), "fg_logprobs_fwd: top without outputs");
    FG_REQUIRE(ctx, logprob_out || entropy_out || lse_out || top, "fg_logprobs_fwd: no output");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(logits, size) && fg_at_element(targets, 4) && fg_at_element(logprob_out, 4) && fg_at_element(entropy_out, 4) &&
                        fg_at_element(lse_out, 4) && fg_at_element(top_ids_out, 4) && fg_at_element(top_logprobs_out, 4),
               "fg_logprobs_fwd: a tensor does not start at an element");
    const uint64_t bytes = (uint64_t)rows * cols * size, column = 4ull * rows, table = column * top;
    const struct { const void* p; uint64_t n; } out[] = {{logprob_out, column}, {entropy_out, column}, {lse_out, column}, {top ? top_ids_out : nullptr, table}, {top ? top_logprobs_out : nullptr, table}};
    for (int i = 0; i < 5; ++i) {
        FG_REQUIRE(ctx, !fg_ranges_meet(out[i].p, out[i].n, logits, bytes) && !fg_ranges_meet(out[i].p, out[i].n, targets, column),
                   "fg_logprobs_fwd: an output overlaps another tensor");
        for (int j = 0; j < i; ++j) FG_REQUIRE(ctx, !fg_ranges_meet(out[i].p, out[i].n, out[j].p, out[j].n), "fg_logprobs_fwd: outputs overlap");
    }
    if (rows == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, logprobs_fwd, ctx, LogprobArgs{logits, targets, rows, cols, top, scale, logprob_out, entropy_out, lse_out, top_ids_out, top_logprobs_out});
}

int32_t fg_logprobs_bwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* logits, const uint32_t* targets, float scale,
                        const float* lse, const float* entropy, const float* dlogprob, const float* dentropy, void* dlogits) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_logprobs_bwd: unknown dtype");
    FG_REQUIRE(ctx, logits && lse && dlogits, "fg_logprobs_bwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1, "fg_logprobs_bwd: cols must be >= 1");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_logprobs_bwd: tensor too large");
    FG_REQUIRE(ctx, scale > 0.0f && scale <= 3.402823466e38f, "fg_logprobs_bwd: scale must be a number > 0");
    FG_REQUIRE(ctx, dlogprob || dentropy, "fg_logprobs_bwd: no gradient given");
    FG_REQUIRE(ctx, !dlogprob || targets, "fg_logprobs_bwd: dlogprob without targets");
    FG_REQUIRE(ctx, !dentropy || entropy, "fg_logprobs_bwd: dentropy without the entropies");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(logits, size) && fg_at_element(dlogits, size) && fg_at_element(targets, 4) && fg_at_element(lse, 4) && fg_at_element(entropy, 4) &&
                        fg_at_element(dlogprob, 4) && fg_at_element(dentropy, 4), "fg_logprobs_bwd: a tensor does not start at an element");
    const uint64_t bytes = (uint64_t)rows * cols * size, column = 4ull * rows;
    FG_REQUIRE(ctx, dlogits == logits || !fg_ranges_meet(dlogits, bytes, logits, bytes), "fg_logprobs_bwd: dlogits overlaps logits but is not them");
    for (const void* in : {(const void*)targets, (const void*)lse, (const void*)entropy, (const void*)dlogprob, (const void*)dentropy})
        FG_REQUIRE(ctx, !fg_ranges_meet(dlogits, bytes, in, column), "fg_logprobs_bwd: dlogits overlaps another tensor");
    if (rows == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, logprobs_bwd, ctx, LogprobBwdArgs{logits, targets, lse, entropy, dlogprob, dentropy, dlogits, rows, cols, scale});
}

}  // extern "C"
