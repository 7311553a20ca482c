// Attention on the tensor cores: 16-bit tensors, head_dim a multiple of 8 up to 128, tensors and strides on 16-byte boundaries.
//
// A tile has 128 rows: all heads of a group by 128 / group queries, so keys are read once for the group, and a box of a tensor map
// {head_dim, heads, tokens} is a tile.  Operands are [rows][64] in shared memory with the 128-byte swizzle, two such halves for a head_dim over 64;
// columns behind head_dim are zeros, which the tensor map fills in.
#include <cuda.h>

#include <atomic>

#include "attention_tc.cuh"
#include "ptx_sm100.cuh"

using namespace fgptx;

namespace {

constexpr long long kWaitCycles = 2000000000LL;      // bound on every device-side wait (about 1 s)
constexpr int kRows = 128, kHalfBytes = 128 * 128;
constexpr uint32_t kTmemCols = 512;

template <typename T> constexpr uint32_t kFormat = std::is_same_v<T, __half> ? 0u : 1u;      // of the tensor cores' operands

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same_v<T, __half>) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t round_up(uint32_t a, uint32_t b) { return (a + b - 1) / b * b; }

// A warp's wait: true in all lanes, or an error is left behind for the host and the role ends.
__device__ __forceinline__ bool await(uint32_t bar, uint32_t parity, int* dev_status, int error) {
    if (__all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, kWaitCycles))) return true;
    if ((threadIdx.x & 31) == 0) atomicOr(dev_status, error);
    return false;
}

// ---- forward ----
// A block has two tiles of rows, one after the other in the sequence, that take turns: while the threads of one turn scores into weights, the tensor cores
// multiply for the other.  Warps 0 to 3 and 4 to 7 have a row of their tile per thread, warp 8 loads, warp 9 multiplies.
// Tensor memory: scores of tile s at column 128 s, where the weights then lie as the A operand of the product with v; sums of out at 256 + 128 s.
// Order of the products: S0(0) S1(0), then for each tile of keys j: PV0(j) S0(j+1) PV1(j) S1(j+1).  The scores of j + 1 come after PV(j) in this order, so they
// may take the weights' place, and whoever has seen them arrive knows that out holds everything up to j.
template <int DP>
struct FwdCfg {
    static constexpr int kTile = kHalfBytes * (DP / 64), kStages = DP == 128 ? 5 : 8, kThreads = 384;
    static constexpr int kBars = 2 + 2 * kStages + 7;
    static constexpr size_t kSmem = 1024 + (size_t)(2 + kStages) * kTile + 8 * kBars + 16;
};

template <typename T, int DP>
__global__ void __launch_bounds__(FwdCfg<DP>::kThreads, 1)
attn_tc_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ FgAttnArgs a, uint32_t tokens, uint32_t tiles) {
    using Cfg = FwdCfg<DP>;
    constexpr int S = Cfg::kStages;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t qs = base, ring = base + 2 * Cfg::kTile, bar0 = ring + S * Cfg::kTile;
    auto q_full = [&](uint32_t s) { return bar0 + 8 * s; };
    auto kv_full = [&](uint32_t i) { return bar0 + 8 * (2 + i); };
    auto kv_empty = [&](uint32_t i) { return bar0 + 8 * (2 + S + i); };
    auto s_full = [&](uint32_t s) { return bar0 + 8 * (2 + 2 * S + s); };
    auto p_full = [&](uint32_t s) { return bar0 + 8 * (4 + 2 * S + s); };
    auto o_full = [&](uint32_t s) { return bar0 + 8 * (6 + 2 * S + s); };
    const uint32_t drained = bar0 + 8 * (8 + 2 * S);
    __shared__ uint32_t tmem_slot;
    __shared__ int s_abort;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) { mbar_init(q_full(s), 1); mbar_init(s_full(s), 1); mbar_init(p_full(s), 128); mbar_init(o_full(s), 1); }
        for (int i = 0; i < S; ++i) { mbar_init(kv_full(i), 1); mbar_init(kv_empty(i), 1); }
        mbar_init(drained, 1);
        fence_mbar_init();
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(&tmem_slot), kTmemCols);
        tmem_relinquish();
    }
    fg_grid_enter();
    if (threadIdx.x == 0) s_abort = *reinterpret_cast<volatile int*>(a.dev_status);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    const bool go = __all_sync(0xffffffffu, s_abort == 0);

    const uint32_t kv = blockIdx.x % a.kv_heads;
    uint32_t tile;
    const int b = go ? fg_attn_find(a.q_starts, a.sequences, a.queries, 1, 2 * tokens, tiles - 1 - blockIdx.x / a.kv_heads, &tile) : -1;
    if (b >= 0) {
        const FgAttnSeq s(a, b);
        // (the numbering leaves gaps: a tile may lie behind its sequence's end)
        const uint64_t tok0_ = (uint64_t)tile * 2 * tokens;
        const uint32_t tok0 = tok0_ < s.nq ? (uint32_t)tok0_ : s.nq, left = s.nq - tok0;
        const uint32_t tok_0 = min(tokens, left), tok_1 = left > tokens ? min(tokens, left - tokens) : 0;
        // Keys that the tile's last query sees, and tiles of them.
        const uint32_t hi_0 = tok_0 ? s.seen(a, tok0 + tok_0 - 1) : 0, hi_1 = tok_1 ? s.seen(a, tok0 + tokens + tok_1 - 1) : 0;
        const uint32_t n_0 = (hi_0 + kRows - 1) / kRows, n_1 = (hi_1 + kRows - 1) / kRows, n_all = max(n_0, n_1);
        const uint32_t fmt = kFormat<T>, dim16 = round_up(a.dim, 16);

        if (warp >= 8) reg_release<40>();      // (all four warps of the group)
        if (warp == 8) {
            // ---- loads ----
            const uint32_t q_bytes = DP / 64 * 128 * tokens * a.group;
            auto load_q = [&](uint32_t t) {
                mbar_expect_tx(q_full(t), q_bytes);
#pragma unroll
                for (int h = 0; h < DP / 64; ++h)
                    tma_load_3d(qs + t * Cfg::kTile + h * kHalfBytes, &tm_q, q_full(t), 64 * h, (int)(kv * a.group), (int)(s.q0 + tok0 + t * tokens));
            };
            uint32_t g = 0;
            for (uint32_t i = 0; i < 2 * n_all; ++i, ++g) {
                const uint32_t st = g % S;
                if (!await(kv_empty(st), ((g / S) & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
                if (elect_one()) {
                    if (i == 0 && n_0) load_q(0);
                    mbar_expect_tx(kv_full(st), Cfg::kTile);
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h)
                        tma_load_3d(ring + st * Cfg::kTile + h * kHalfBytes, i & 1 ? &tm_v : &tm_k, kv_full(st), 64 * h, (int)kv, (int)(s.k0 + i / 2 * kRows));
                    if (i == 0 && n_1) load_q(1);
                }
                __syncwarp();
            }
            // Nothing of this block is on its way when it ends, whatever became of the other roles.
            for (uint32_t i = g > (uint32_t)S ? g - S : 0; i < g; ++i)
                if (!await(kv_full(i % S), (i / S) & 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
            for (uint32_t t = 0; g && t < 2; ++t)
                if (t ? n_1 : n_0) await(q_full(t), 0, a.dev_status, FG_DEVERR_TMA_WAIT);
        } else if (warp == 9) {
            // ---- products ----
            const uint32_t o_desc = make_idesc(fmt, 128, dim16) | kIdescBMnMajor, steps = dim16 / 16;
            bool ok = true;
            auto scores = [&](uint32_t t, uint32_t j, uint32_t st) {
                const uint32_t cols = round_up(min((uint32_t)kRows, (t ? hi_1 : hi_0) - j * kRows), 16);
                const uint32_t id = make_idesc(fmt, 128, cols);
                const uint64_t q_d = make_desc_kmajor<128>(qs + t * Cfg::kTile), k_d = make_desc_kmajor<128>(ring + st * Cfg::kTile);
                for (uint32_t c = 0; c < steps; ++c) {
                    const uint64_t at = (uint64_t)((c & 3) * 2 + (c >> 2) * (kHalfBytes >> 4));
                    mma_f16(tmem + t * 128, q_d + at, k_d + at, id, c != 0);
                }
                mma_commit(s_full(t));
            };
            uint32_t g = 0;      // position in the ring: k0 v0 k1 v1 ..
            if (n_all) {
                ok = await(kv_full(0), 0, a.dev_status, FG_DEVERR_MMA_WAIT);
                for (uint32_t t = 0; ok && t < 2; ++t) {
                    if (!(t ? n_1 : n_0)) continue;
                    ok = await(q_full(t), 0, a.dev_status, FG_DEVERR_MMA_WAIT);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) scores(t, 0, 0);
                    __syncwarp();
                }
                if (ok && elect_one()) mma_commit(kv_empty(0));
                __syncwarp();
                g = 1;
            }
            for (uint32_t j = 0; ok && j < n_all; ++j, g += 2) {
                const uint32_t vs = g % S, ks = (g + 1) % S;
                const bool more = j + 1 < n_all;
                if (!await(kv_full(vs), (g / S) & 1, a.dev_status, FG_DEVERR_MMA_WAIT)) break;
                // The rows of v behind the sequence's end have a weight of zero, but what stands there may be NaN: zeros for those that the last step multiplies.
                const uint32_t left = s.nk - j * kRows;
                if (left < kRows && (left & 15)) {
                    const uint32_t end = round_up(left, 16);
                    for (uint32_t i = left * 8 + lane; i < end * 8; i += 32)
#pragma unroll
                        for (int h = 0; h < DP / 64; ++h) fg_store_shared(ring + vs * Cfg::kTile + h * kHalfBytes + i * 16, make_uint4(0, 0, 0, 0));
                    fence_proxy_async();
                    __syncwarp();
                }
                if (more && !await(kv_full(ks), ((g + 1) / S) & 1, a.dev_status, FG_DEVERR_MMA_WAIT)) break;
                for (uint32_t t = 0; t < 2; ++t) {
                    if (j < (t ? n_1 : n_0)) {
                        ok = await(p_full(t), j & 1, a.dev_status, FG_DEVERR_MMA_WAIT);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t key_steps = (min((uint32_t)kRows, (t ? hi_1 : hi_0) - j * kRows) + 15) / 16;
                            const uint64_t v_d = make_desc_mnmajor(ring + vs * Cfg::kTile, kHalfBytes, 1024, 2);
                            for (uint32_t c = 0; c < key_steps; ++c) mma_f16_ta(tmem + 256 + t * 128, tmem + t * 128 + c * 8, v_d + (uint64_t)(c * 128), o_desc, j | c);
                            if (j + 1 < (t ? n_1 : n_0)) scores(t, j + 1, ks);
                            else mma_commit(o_full(t));
                        }
                        __syncwarp();
                    }
                    if (t == 1 && elect_one()) {
                        mma_commit(kv_empty(vs));
                        if (more) mma_commit(kv_empty(ks));
                    }
                    __syncwarp();
                }
            }
            // (a product may still run where a wait ran out)
            if (elect_one()) mma_commit(drained);
            __syncwarp();
            await(drained, 0, a.dev_status, FG_DEVERR_MMA_WAIT);
        } else if (warp < 8) {
            // ---- weights: a row per thread ----
            reg_acquire<232>();
            const uint32_t t = warp >> 2, r = threadIdx.x & 127, i = tok0 + t * tokens + r / a.group, head = kv * a.group + r % a.group;
            const bool there = r / a.group < (t ? tok_1 : tok_0);
            const uint32_t seen = there ? s.seen(a, i) : 0;
            const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21), t_s = lanes + t * 128, t_o = lanes + 256 + t * 128;
            const float by = a.scale * kFgLog2e;
            float top = -INFINITY;
            float2 sum = make_float2(0.0f, 0.0f);
            bool ok = true;
            for (uint32_t j = 0; j < (t ? n_1 : n_0); ++j) {
                if (!(ok = await(s_full(t), j & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                tc_fence_after();
                uint32_t w[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_s + c * 32, w[c]);
                tmem_ld_wait();
                const uint32_t end = j * kRows < seen ? seen - j * kRows : 0;
                if (__any_sync(0xffffffffu, end < kRows)) {
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if ((uint32_t)c >= end) w[c / 32][c % 32] = __float_as_uint(-INFINITY);
                }
                float most = -INFINITY, m1 = -INFINITY;
#pragma unroll
                for (int c = 0; c < 128; c += 4) {
                    most = max3(most, __uint_as_float(w[c / 32][c % 32]), __uint_as_float(w[c / 32][c % 32 + 1]));
                    m1 = max3(m1, __uint_as_float(w[c / 32][c % 32 + 2]), __uint_as_float(w[c / 32][c % 32 + 3]));
                }
                most = fmaxf(most, m1) * by;
                // The base of the exponents follows the largest score only when that has grown by more than 8: weights stay below 2^8, and out is
                // seldom gone over again.
                if (j == 0) top = most;
                else if (__any_sync(0xffffffffu, most > top + 8.0f)) {
                    const float next = fmaxf(top, most), f = next == -INFINITY ? 1.0f : fg_ex2_fast(top - next);
                    top = next;
                    sum = make_float2(sum.x * f, sum.y * f);
#pragma unroll
                    for (int c = 0; c < DP; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32(t_o + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_32x32(t_o + c, o);
                    }
                }
                const float less = top == -INFINITY ? 0.0f : -top;
                const float2 by2 = make_float2(by, by), less2 = make_float2(less, less);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t p[32];
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        const int at = h * 64 + 2 * c;
                        float2 x = make_float2(__uint_as_float(w[at / 32][at % 32]), __uint_as_float(w[at / 32][at % 32 + 1]));
                        x = fg_fma2(x, by2, less2);
                        x = make_float2(fg_ex2_fast(x.x), fg_ex2_fast(x.y));
                        sum = fg_add2(sum, x);
                        p[c] = pack2<T>(x.x, x.y);
                    }
                    tmem_st_32x32(t_s + h * 32, p);
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(p_full(t));
            }
            const float total = sum.x + sum.y;
            if (ok && (t ? n_1 : n_0)) ok = await(o_full(t), 0, a.dev_status, FG_DEVERR_EPI_WAIT);
            if (ok && (t ? tok_1 : tok_0)) {
                tc_fence_after();
                const uint32_t row = s.q0 + i;
                const float f = total == 0.0f ? 0.0f : 1.0f / total;
                T* const out = static_cast<T*>(a.out) + ((uint64_t)row * a.heads + head) * a.dim;
#pragma unroll
                for (int c = 0; c < DP; c += 32) {
                    uint32_t o[32];
                    if ((t ? n_1 : n_0)) {      // a tile that sees nothing has no sums
                        tmem_ld_32x32(t_o + c, o);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (total != 0.0f) {
                            v.x = pack2<T>(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f);
                            v.y = pack2<T>(__uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
                            v.z = pack2<T>(__uint_as_float(o[e + 4]) * f, __uint_as_float(o[e + 5]) * f);
                            v.w = pack2<T>(__uint_as_float(o[e + 6]) * f, __uint_as_float(o[e + 7]) * f);
                        }
                        if (there && (uint32_t)(c + e) < a.dim) *reinterpret_cast<uint4*>(out + c + e) = v;
                    }
                }
                if (there && a.lse) a.lse[(uint64_t)head * a.queries + row] = (top + __log2f(total)) * kFgLn2;
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// ---- host ----
typedef CUresult (*pfn_encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Tokens of `heads` heads of `dim`, `stride` elements apart; boxes of 64 columns by box_heads by box_tokens.
int32_t make_map(fg_ctx* ctx, CUtensorMap* out, const void* p, bool half, uint32_t dim, uint32_t heads, uint32_t tokens, uint64_t stride, uint32_t box_heads,
                 uint32_t box_tokens) {
    cuuint64_t dims[3] = {dim, heads, tokens};
    cuuint64_t strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)stride * 2};
    cuuint32_t box[3] = {64, box_heads, box_tokens}, each[3] = {1, 1, 1};
    const CUresult r = ((pfn_encode)ctx->tmap_encode)(out, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims,
                                                      strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        snprintf(ctx->err, sizeof(ctx->err), "attention: cuTensorMapEncodeTiled failed with code %d", (int)r);
        return FG_ERR_INTERNAL;
    }
    return FG_OK;
}
// The most shared memory that a kernel is given, once per kernel (`done`) and device.
template <typename K>
int32_t allow_shared(fg_ctx* ctx, std::atomic<uint64_t>& done, K kernel, size_t bytes) {
    if (done.load(std::memory_order_acquire) >> (ctx->device & 63) & 1ull) return FG_OK;
    FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done.fetch_or(1ull << (ctx->device & 63), std::memory_order_release);
    return FG_OK;
}
template <typename T, int DP>
int32_t fwd_launch(fg_ctx* ctx, const FgAttnArgs& a) {
    using Cfg = FwdCfg<DP>;
    constexpr bool half = std::is_same_v<T, __half>;
    static std::atomic<uint64_t> done{0};
    int32_t s = allow_shared(ctx, done, attn_tc_fwd_kernel<T, DP>, Cfg::kSmem);
    if (s != FG_OK) return s;
    const uint32_t tokens = kRows / a.group;
    CUtensorMap q, k, v;
    if ((s = make_map(ctx, &q, a.q, half, a.dim, a.heads, a.queries, a.q_stride, a.group, tokens)) != FG_OK) return s;
    if ((s = make_map(ctx, &k, a.k, half, a.dim, a.kv_heads, a.keys, a.k_stride, 1, kRows)) != FG_OK) return s;
    if ((s = make_map(ctx, &v, a.v, half, a.dim, a.kv_heads, a.keys, a.v_stride, 1, kRows)) != FG_OK) return s;
    const uint64_t tiles = fg_attn_tiles(a.sequences, a.queries, 1, 2 * tokens);
    if (tiles * a.kv_heads >= 1ull << 31) return fg_fail(ctx, FG_ERR_INVALID_ARGUMENT, "attention: tensor too large");
    fg_launch(ctx, attn_tc_fwd_kernel<T, DP>, (unsigned)(tiles * a.kv_heads), Cfg::kThreads, Cfg::kSmem, q, k, v, a, tokens, (uint32_t)tiles);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

}  // namespace

bool fg_attn_tc_suits(const fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a) {
    if (dtype == FG_DTYPE_F32 || !ctx->tmap_encode || a.dim % 8 || a.dim > 128 || a.group > (uint32_t)kRows || !(a.scale > 0.0f) || !a.keys) return false;
    const uint64_t strides = a.q_stride | a.k_stride | a.v_stride;
    return strides % 8 == 0 && fg_aligned16(a.q) && fg_aligned16(a.k) && fg_aligned16(a.v) && fg_aligned16(a.out) && fg_aligned16(a.dout) && fg_aligned16(a.dq) &&
           fg_aligned16(a.dk) && fg_aligned16(a.dv);
}
int32_t fg_attn_tc_fwd(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a) {
    if (dtype == FG_DTYPE_F16) return a.dim <= 64 ? fwd_launch<__half, 64>(ctx, a) : fwd_launch<__half, 128>(ctx, a);
    return a.dim <= 64 ? fwd_launch<__nv_bfloat16, 64>(ctx, a) : fwd_launch<__nv_bfloat16, 128>(ctx, a);
}
