// Embedding lookup with scaling, and the gradient of its table.
#include "rows.cuh"

namespace {

template <typename T>
__global__ void __launch_bounds__(256) embed_kernel(uint32_t tokens, uint32_t vocab, uint32_t dim, const uint32_t* ids, const T* table, float scale,
                                                    T* out) {
    fg_grid_enter();
    for (uint32_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        const uint32_t id = ids[t];
        const T* row = table + (uint64_t)id * dim;
        for (uint64_t c = threadIdx.x; c < dim; c += 256) out[(uint64_t)t * dim + c] = fg_narrow<T>(id < vocab ? scale * fg_widen(row[c]) : 0.0f);
    }
}

// One block for a row of the table and 256 columns: looks for its tokens in order.
template <typename T>
__global__ void __launch_bounds__(256) embed_bwd_scan_kernel(uint32_t tokens, uint32_t vocab, uint32_t dim, const uint32_t* ids, const T* dout, float scale,
                                                             T* dtable, int accumulate) {
    __shared__ uint32_t found[256];
    __shared__ int count;
    fg_grid_enter();
    const uint64_t c = (uint64_t)blockIdx.y * 256 + threadIdx.x;
    for (uint32_t v = blockIdx.x; v < vocab; v += gridDim.x) {
        float s = 0.0f;
        bool any = false;
        for (uint64_t t0 = 0; t0 < tokens; t0 += 256) {
            const uint64_t t = t0 + threadIdx.x;
            found[threadIdx.x] = t < tokens ? ids[t] : 0xffffffffu;
            if (!__syncthreads_or(found[threadIdx.x] == v)) continue;
            for (int i = 0; i < 256 && t0 + i < tokens; ++i)
                if (found[i] == v) {
                    any = true;
                    if (c < dim) s += fg_widen(dout[(t0 + i) * dim + c]);
                }
            __syncthreads();
        }
        if (c < dim && (any || !accumulate)) {
            T* p = dtable + (uint64_t)v * dim + c;
            *p = fg_narrow<T>(accumulate ? __fmaf_rn(scale, s, fg_widen(*p)) : scale * s);
        }
    }
}

struct EmbedArgs {
    uint32_t tokens, vocab, dim;
    const uint32_t* ids;
    const void* src;
    float scale;
    void* dst;
    int accumulate;
};

template <typename T>
int32_t embed_fwd(fg_ctx* ctx, const EmbedArgs& a) {
    const uint32_t cap = 8u * ctx->sm_count;
    fg_launch(ctx, embed_kernel<T>, a.tokens < cap ? a.tokens : cap, 256, 0, a.tokens, a.vocab, a.dim, a.ids, (const T*)a.src, a.scale, (T*)a.dst);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T>
int32_t embed_bwd(fg_ctx* ctx, const EmbedArgs& a) {
    const uint32_t cap = 8u * ctx->sm_count;
    fg_launch(ctx, embed_bwd_scan_kernel<T>, dim3(a.vocab < cap ? a.vocab : cap, (a.dim + 255) / 256), 256, 0, a.tokens, a.vocab, a.dim, a.ids,
              (const T*)a.src, a.scale, (T*)a.dst, a.accumulate);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

}  // namespace

extern "C" {

int32_t fg_embedding_fwd(fg_ctx* ctx, int32_t dtype, uint32_t tokens, uint32_t vocab, uint32_t dim, const uint32_t* ids, const void* table,
                         float scale, void* out) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_embedding_fwd: unknown dtype");
    FG_REQUIRE(ctx, ids && table && out, "fg_embedding_fwd: NULL pointer");
    FG_REQUIRE(ctx, vocab >= 1 && dim >= 1, "fg_embedding_fwd: vocab and dim must be >= 1");
    FG_REQUIRE(ctx, (uint64_t)tokens * dim < (1ull << 40) && (uint64_t)vocab * dim < (1ull << 40), "fg_embedding_fwd: tensor too large");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(ids, 4) && fg_at_element(table, size) && fg_at_element(out, size),
               "fg_embedding_fwd: a tensor does not start at an element");
    FG_REQUIRE(ctx, !fg_ranges_meet(table, (uint64_t)vocab * dim * size, out, (uint64_t)tokens * dim * size), "fg_embedding_fwd: out overlaps the table");
    if (tokens == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, embed_fwd, ctx, EmbedArgs{tokens, vocab, dim, ids, table, scale, out, 0});
}

int32_t fg_embedding_bwd(fg_ctx* ctx, int32_t dtype, uint32_t tokens, uint32_t vocab, uint32_t dim, const uint32_t* ids, const void* dout,
                         float scale, void* dtable, int32_t accumulate) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_embedding_bwd: unknown dtype");
    FG_REQUIRE(ctx, ids && dout && dtable, "fg_embedding_bwd: NULL pointer");
    FG_REQUIRE(ctx, vocab >= 1 && dim >= 1, "fg_embedding_bwd: vocab and dim must be >= 1");
    FG_REQUIRE(ctx, (uint64_t)tokens * dim < (1ull << 40) && (uint64_t)vocab * dim < (1ull << 40), "fg_embedding_bwd: tensor too large");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(ids, 4) && fg_at_element(dout, size) && fg_at_element(dtable, size),
               "fg_embedding_bwd: a tensor does not start at an element");
    FG_REQUIRE(ctx, !fg_ranges_meet(dtable, (uint64_t)vocab * dim * size, dout, (uint64_t)tokens * dim * size), "fg_embedding_bwd: dtable overlaps dout");
    if (tokens == 0) {      // empty sums
        if (!accumulate) FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(dtable, 0, (uint64_t)vocab * dim * size, ctx->stream));
        return FG_OK;
    }
    return FG_BY_DTYPE(dtype, embed_bwd, ctx, EmbedArgs{tokens, vocab, dim, ids, dout, scale, dtable, accumulate});
}

}  // extern "C"
