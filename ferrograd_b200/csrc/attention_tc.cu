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
// A block has two tiles of rows, one behind the other in the sequence, that take turns: while the threads of one turn scores into weights, the tensor cores
// multiply for the other.  Warps 0 to 3 and 4 to 7 have a row of their tile per thread, warp 8 loads, warp 9 multiplies.  A block
// stays on its SM and takes one pair of tiles after the other from a counter, longest first, so that loads and the first products of the next pair
// run while the last sums of this one are written.
// Tensor memory: scores of tile t at column 128 t, where the weights then lie as the A operand of the product with v; sums of out at 256 + 128 t.
// Order of the products: S0(0) S1(0), then for each tile of keys j: PV0(j) S0(j+1) PV1(j) S1(j+1).  The scores of j + 1 come after PV(j) in this order, so they
// may take the weights' place, and whoever has seen them arrive knows that out holds everything up to j.
// A pair of tiles (more = 0: none is left): queries of each tile, keys that its last query sees, tiles of them.
struct FwdWork { uint32_t more, kv, q0, nq, k0, nk, tok0, tok_0, tok_1, hi_0, hi_1, n_0, n_1; };
// F(field) for each.
#define FG_FWD_WORK(F) F(more) F(kv) F(q0) F(nq) F(k0) F(nk) F(tok0) F(tok_0) F(tok_1) F(hi_0) F(hi_1) F(n_0) F(n_1)
template <int DP>
struct FwdCfg {
    static constexpr int kTile = kHalfBytes * (DP / 64), kStages = DP == 128 ? 5 : 8, kThreads = 384, kSlots = 2;
    static constexpr int kBars = 2 * kStages + 2 * 6 + 2 * kSlots + 1;
    static constexpr size_t kUsed = (size_t)(2 + kStages) * kTile + 8 * kBars + sizeof(FwdWork) * kSlots + 16, kSmem = kUsed + 1024;
};

template <typename T, int DP>
__global__ void __launch_bounds__(FwdCfg<DP>::kThreads, 1)
attn_tc_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ FgAttnArgs a, uint32_t tokens, uint32_t tiles, unsigned* counter) {
    using Cfg = FwdCfg<DP>;
    constexpr int S = Cfg::kStages, W = Cfg::kSlots;
    extern __shared__ __align__(1024) unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    const uint32_t qs = base, ring = base + 2 * Cfg::kTile, bar0 = ring + S * Cfg::kTile;
    auto kv_full = [&](uint32_t i) { return bar0 + 8 * i; };
    auto kv_empty = [&](uint32_t i) { return bar0 + 8 * (S + i); };
    auto tile_bar = [&](uint32_t which, uint32_t t) { return bar0 + 8 * (2 * S + 2 * which + t); };
    auto q_full = [&](uint32_t t) { return tile_bar(0, t); };
    auto q_empty = [&](uint32_t t) { return tile_bar(1, t); };
    auto s_full = [&](uint32_t t) { return tile_bar(2, t); };
    auto p_full = [&](uint32_t t) { return tile_bar(3, t); };
    auto o_full = [&](uint32_t t) { return tile_bar(4, t); };
    auto o_empty = [&](uint32_t t) { return tile_bar(5, t); };
    auto work_full = [&](uint32_t i) { return bar0 + 8 * (2 * S + 12 + i); };
    auto work_empty = [&](uint32_t i) { return bar0 + 8 * (2 * S + 12 + W + i); };
    const uint32_t drained = bar0 + 8 * (2 * S + 12 + 2 * W);
    unsigned char* const tail = raw + (bar0 + 8 * Cfg::kBars - smem_u32(raw));
    volatile uint32_t* const slot = reinterpret_cast<volatile uint32_t*>(tail);      // the tensor memory's address, a flag
    volatile FwdWork* const works = reinterpret_cast<volatile FwdWork*>(tail + 16);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(kv_full(i), 1); mbar_init(kv_empty(i), 1); }
        for (int t = 0; t < 2; ++t) {
            mbar_init(q_full(t), 1); mbar_init(q_empty(t), 1); mbar_init(s_full(t), 1);
            mbar_init(p_full(t), 128); mbar_init(o_full(t), 1); mbar_init(o_empty(t), 128);
        }
        for (int i = 0; i < W; ++i) { mbar_init(work_full(i), 1); mbar_init(work_empty(i), 9); }
        mbar_init(drained, 1);
        fence_mbar_init();
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
    }
    if (warp == 9) {
        tmem_alloc(bar0 + 8 * Cfg::kBars, kTmemCols);
        tmem_relinquish();
    }
    fg_grid_enter();
    if (threadIdx.x == 0) slot[1] = (uint32_t)*reinterpret_cast<volatile int*>(a.dev_status);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, slot[0], 0);
    const bool go = __all_sync(0xffffffffu, slot[1] == 0);

    // The next pair of tiles, for the warps that work on it (false: none, or a wait ran out).
    uint32_t taken = 0;
    auto next = [&](FwdWork& w, bool& ok) {
        if (!(ok = await(work_full(taken % W), (taken / W) & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) return false;
        volatile const FwdWork& from = works[taken % W];
#define FG_TAKE(field) w.field = from.field;
        FG_FWD_WORK(FG_TAKE)
#undef FG_TAKE
        __syncwarp();
        if (lane == 0) mbar_arrive(work_empty(taken % W));
        ++taken;
        return w.more != 0;
    };
    const uint32_t fmt = kFormat<T>, dim16 = round_up(a.dim, 16);
    if (go) {
        if (warp >= 8) reg_release<56>();      // (all four warps of the group)
        if (warp == 8) {
            // ---- work and loads: the next pair of tiles is taken when the last load of this one is under way ----
            const uint32_t all = tiles * a.kv_heads, q_bytes = DP / 64 * 128 * tokens * a.group;
            uint32_t g = 0, q_loads[2] = {0, 0};      // tiles of keys and values, tiles of queries so far
            bool ok = true;
            for (uint32_t count = 0; ok; ++count) {
                FwdWork w = {};
                for (;;) {      // tiles are numbered with gaps, which are passed over here
                    uint32_t item = 0;
                    if (lane == 0) item = atomicInc(counter, all + gridDim.x - 1);      // (each block takes one too many: the last one leaves zero)
                    item = __shfl_sync(0xffffffffu, item, 0);
                    w.more = item < all;
                    if (!w.more) break;
                    w.kv = item % a.kv_heads;
                    uint32_t tile;
                    const int b = fg_attn_find(a.q_starts, a.sequences, a.queries, 1, 2 * tokens, tiles - 1 - item / a.kv_heads, &tile);
                    if (b < 0) continue;
                    const FgAttnSeq s(a, b);
                    const uint64_t tok0 = (uint64_t)tile * 2 * tokens;
                    if (tok0 >= s.nq) continue;
                    w.q0 = s.q0; w.nq = s.nq; w.k0 = s.k0; w.nk = s.nk;
                    w.tok0 = (uint32_t)tok0;
                    const uint32_t left = s.nq - w.tok0;
                    w.tok_0 = min(tokens, left);
                    w.tok_1 = left > tokens ? min(tokens, left - tokens) : 0;
                    w.hi_0 = s.seen(a, w.tok0 + w.tok_0 - 1);
                    w.hi_1 = w.tok_1 ? s.seen(a, w.tok0 + tokens + w.tok_1 - 1) : 0;
                    w.n_0 = (w.hi_0 + kRows - 1) / kRows;
                    w.n_1 = (w.hi_1 + kRows - 1) / kRows;
                    break;
                }
                if (!(ok = await(work_empty(count % W), ((count / W) & 1) ^ 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                if (lane == 0) {
                    volatile FwdWork& to = works[count % W];
#define FG_LEAVE(field) to.field = w.field;
                    FG_FWD_WORK(FG_LEAVE)
#undef FG_LEAVE
                    mbar_arrive(work_full(count % W));
                }
                __syncwarp();
                if (!w.more) break;
                const uint32_t n_all = max(w.n_0, w.n_1);
                for (uint32_t i = 0; i < 2 * n_all; ++i, ++g) {
                    const uint32_t st = g % S;
                    if (!(ok = await(kv_empty(st), ((g / S) & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT))) break;
                    if (elect_one()) {
                        mbar_expect_tx(kv_full(st), Cfg::kTile);
#pragma unroll
                        for (int h = 0; h < DP / 64; ++h)
                            tma_load_3d(ring + st * Cfg::kTile + h * kHalfBytes, i & 1 ? &tm_v : &tm_k, kv_full(st), 64 * h, (int)w.kv, (int)(w.k0 + i / 2 * kRows));
                    }
                    __syncwarp();
                    if (i) continue;
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t) {
                        if (!(t ? w.n_1 : w.n_0) || !ok) continue;
                        if (!(ok = await(q_empty(t), (q_loads[t] & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT))) continue;
                        if (elect_one()) {
                            mbar_expect_tx(q_full(t), q_bytes);
#pragma unroll
                            for (int h = 0; h < DP / 64; ++h)
                                tma_load_3d(qs + t * Cfg::kTile + h * kHalfBytes, &tm_q, q_full(t), 64 * h, (int)(w.kv * a.group), (int)(w.q0 + w.tok0 + t * tokens));
                        }
                        __syncwarp();
                        ++q_loads[t];
                    }
                    if (!ok) { ++g; break; }
                }
            }
            // Nothing of this block is on its way when it ends, whatever became of the other roles.
            for (uint32_t i = g > (uint32_t)S ? g - S : 0; i < g; ++i)
                if (!await(kv_full(i % S), (i / S) & 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
#pragma unroll
            for (uint32_t t = 0; t < 2; ++t)
                if (q_loads[t]) await(q_full(t), (q_loads[t] - 1) & 1, a.dev_status, FG_DEVERR_TMA_WAIT);
        } else if (warp == 9) {
            // ---- products ----
            const uint32_t o_desc = make_idesc(fmt, 128, dim16) | kIdescBMnMajor, steps = dim16 / 16;
            uint32_t g = 0, p_seen[2] = {0, 0}, pairs[2] = {0, 0};      // position in the ring (k0 v0 k1 v1 ..), weights so far, tiles of rows so far
            FwdWork w = {};
            bool ok;
            const bool whole = dim16 == DP;      // (unrolled: an instruction per product and few beside it)
            auto scores = [&](uint32_t t, uint32_t j, uint32_t st) {
                const uint32_t cols = round_up(min((uint32_t)kRows, (t ? w.hi_1 : w.hi_0) - j * kRows), 16);
                const uint32_t id = make_idesc(fmt, 128, cols);
                const uint64_t q_d = make_desc_kmajor<128>(qs + t * Cfg::kTile), k_d = make_desc_kmajor<128>(ring + st * Cfg::kTile);
                if (whole) {
#pragma unroll
                    for (uint32_t c = 0; c < DP / 16; ++c) {
                        const uint64_t at = (uint64_t)((c & 3) * 2 + (c >> 2) * (kHalfBytes >> 4));
                        mma_f16(tmem + t * 128, q_d + at, k_d + at, id, c != 0);
                    }
                } else
                    for (uint32_t c = 0; c < steps; ++c) {
                        const uint64_t at = (uint64_t)((c & 3) * 2 + (c >> 2) * (kHalfBytes >> 4));
                        mma_f16(tmem + t * 128, q_d + at, k_d + at, id, c != 0);
                    }
                mma_commit(s_full(t));
                if (j + 1 == (t ? w.n_1 : w.n_0)) mma_commit(q_empty(t));
            };
            while (next(w, ok)) {
                const uint32_t n_all = max(w.n_0, w.n_1);
                if (!n_all) continue;
                if (!(ok = await(kv_full(g % S), (g / S) & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) break;
#pragma unroll
                for (uint32_t t = 0; t < 2; ++t) {
                    if (!(t ? w.n_1 : w.n_0) || !ok) continue;
                    if (!(ok = await(q_full(t), pairs[t] & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) continue;
                    tc_fence_after();
                    if (elect_one()) scores(t, 0, g % S);
                    __syncwarp();
                }
                // Before the first products into out: the sums of the tiles before have been read.  (Waited for inside of the loop, by a test of j, this
                // took a tenth of the kernel's time: the products' operands no longer stayed in uniform registers.)
#pragma unroll
                for (uint32_t t = 0; t < 2; ++t)
                    if (ok && (t ? w.n_1 : w.n_0)) ok = await(o_empty(t), (pairs[t] & 1) ^ 1, a.dev_status, FG_DEVERR_MMA_WAIT);
                if (!ok) break;
                if (elect_one()) mma_commit(kv_empty(g % S));
                __syncwarp();
                ++g;
                for (uint32_t j = 0; ok && j < n_all; ++j, g += j < n_all ? 2 : 1) {
                    const uint32_t vs = g % S, ks = (g + 1) % S;
                    const bool more = j + 1 < n_all;
                    if (!(ok = await(kv_full(vs), (g / S) & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) break;
                    // The rows of v behind the sequence's end have a weight of zero, but what stands there may be NaN: zeros for those that the last step multiplies.
                    const uint32_t left = w.nk - j * kRows;
                    if (left < kRows && (left & 15)) {
                        const uint32_t end = round_up(left, 16);
                        for (uint32_t i = left * 8 + lane; i < end * 8; i += 32)
#pragma unroll
                            for (int h = 0; h < DP / 64; ++h) fg_store_shared(ring + vs * Cfg::kTile + h * kHalfBytes + i * 16, make_uint4(0, 0, 0, 0));
                        fence_proxy_async();
                        __syncwarp();
                    }
                    if (more && !(ok = await(kv_full(ks), ((g + 1) / S) & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) break;
#pragma unroll
                    for (uint32_t t = 0; t < 2; ++t) {
                        if (ok && j < (t ? w.n_1 : w.n_0)) {
                            ok = await(p_full(t), p_seen[t] & 1, a.dev_status, FG_DEVERR_MMA_WAIT);
                            ++p_seen[t];
                            if (ok) {
                                tc_fence_after();
                                if (elect_one()) {
                                    const uint32_t key_steps = (min((uint32_t)kRows, (t ? w.hi_1 : w.hi_0) - j * kRows) + 15) / 16;
                                    const uint64_t v_d = make_desc_mnmajor(ring + vs * Cfg::kTile, kHalfBytes, 1024, 2);
                                    if (key_steps == 8) {
#pragma unroll
                                        for (uint32_t c = 0; c < 8; ++c) mma_f16_ta(tmem + 256 + t * 128, tmem + t * 128 + c * 8, v_d + (uint64_t)(c * 128), o_desc, j | c);
                                    } else
                                        for (uint32_t c = 0; c < key_steps; ++c) mma_f16_ta(tmem + 256 + t * 128, tmem + t * 128 + c * 8, v_d + (uint64_t)(c * 128), o_desc, j | c);
                                    if (j + 1 < (t ? w.n_1 : w.n_0)) scores(t, j + 1, ks);
                                    else mma_commit(o_full(t));
                                }
                                __syncwarp();
                            }
                        }
                        if (t == 1 && ok && elect_one()) {
                            mma_commit(kv_empty(vs));
                            if (more) mma_commit(kv_empty(ks));
                        }
                        __syncwarp();
                    }
                }
                if (!ok) break;
#pragma unroll
                for (uint32_t t = 0; t < 2; ++t) pairs[t] += (t ? w.n_1 : w.n_0) != 0;
            }
            // (a product may still run where a wait ran out)
            if (elect_one()) mma_commit(drained);
            __syncwarp();
            await(drained, 0, a.dev_status, FG_DEVERR_MMA_WAIT);
        } else if (warp < 8) {
            // ---- weights: a row per thread ----
            reg_acquire<224>();
            const uint32_t t = warp >> 2, r = threadIdx.x & 127, row_tok = r / a.group, row_head = r % a.group;
            const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21), t_s = lanes + t * 128, t_o = lanes + 256 + t * 128;
            const float by = a.scale * kFgLog2e;
            uint32_t steps = 0, pairs = 0;      // tiles of keys, tiles of rows so far
            FwdWork w = {};
            bool ok;
            while (next(w, ok)) {
                const uint32_t n = t ? w.n_1 : w.n_0, n_tok = t ? w.tok_1 : w.tok_0;
                const uint32_t i = w.tok0 + t * tokens + row_tok, head = w.kv * a.group + row_head;
                const bool there = row_tok < n_tok;
                uint32_t seen = 0;
                if (there) {
                    const int64_t last = a.causal ? (int64_t)i + 1 + (int64_t)w.nk - (int64_t)w.nq : (int64_t)w.nk;
                    seen = last < 0 ? 0 : (uint32_t)last;
                }
                float top = -INFINITY;
                float2 sum = make_float2(0.0f, 0.0f);
                for (uint32_t j = 0; j < n; ++j, ++steps) {
                    if (!(ok = await(s_full(t), steps & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                    tc_fence_after();
                    uint32_t x[4][32];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_s + c * 32, x[c]);
                    tmem_ld_wait();
                    const uint32_t end = j * kRows < seen ? seen - j * kRows : 0;
                    if (__any_sync(0xffffffffu, end < kRows)) {
#pragma unroll
                        for (int c = 0; c < 128; ++c)
                            if ((uint32_t)c >= end) x[c / 32][c % 32] = __float_as_uint(-INFINITY);
                    }
                    float most = -INFINITY, m1 = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 128; c += 4) {
                        most = max3(most, __uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1]));
                        m1 = max3(m1, __uint_as_float(x[c / 32][c % 32 + 2]), __uint_as_float(x[c / 32][c % 32 + 3]));
                    }
                    most = fmaxf(most, m1) * by;
                    // The base of the exponents follows the largest score only when that has grown by more than 8: weights stay below 2^8, and out is
                    // seldom gone over again.
                    if (j == 0) top = most;
                    else if (__any_sync(0xffffffffu, most > top + 8.0f)) {
                        const float up = fmaxf(top, most), f = up == -INFINITY ? 1.0f : fg_ex2_fast(top - up);
                        top = up;
                        sum = make_float2(sum.x * f, sum.y * f);
#pragma unroll
                        for (int c = 0; c < DP; c += 16) {
                            uint32_t o[16];
                            tmem_ld_32x16(t_o + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st_32x16(t_o + c, o);
                        }
                    }
                    const float less = top == -INFINITY ? 0.0f : -top;
                    const float2 by2 = make_float2(by, by), less2 = make_float2(less, less);
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        uint32_t p[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            float2 e = make_float2(__uint_as_float(x[h][2 * c]), __uint_as_float(x[h][2 * c + 1]));
                            e = fg_fma2(e, by2, less2);
                            e = make_float2(fg_ex2_fast(e.x), fg_ex2_fast(e.y));
                            sum = fg_add2(sum, e);
                            p[c] = pack2<T>(e.x, e.y);
                        }
                        tmem_st_32x16(t_s + h * 16, p);
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    mbar_arrive(p_full(t));
                }
                const float total = sum.x + sum.y;
                if (ok && n) ok = await(o_full(t), pairs & 1, a.dev_status, FG_DEVERR_EPI_WAIT);
                if (!ok) break;
                if (n_tok) {
                    tc_fence_after();
                    const uint32_t row = w.q0 + i;
                    const float f = total == 0.0f ? 0.0f : 1.0f / total;
                    T* const out = static_cast<T*>(a.out) + ((uint64_t)row * a.heads + head) * a.dim;
#pragma unroll
                    for (int c = 0; c < DP; c += 32) {
                        uint32_t o[32];
                        if (n) {      // a tile that sees nothing has no sums
                            tmem_ld_32x32(t_o + c, o);
                            tmem_ld_wait();
                            if (c + 32 == DP) {
                                tc_fence_before();
                                mbar_arrive(o_empty(t));
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint4 v = make_uint4(0, 0, 0, 0);
                            uint32_t* const u = o + e;
                            if (total != 0.0f) {
                                v.x = pack2<T>(__uint_as_float(u[0]) * f, __uint_as_float(u[1]) * f);
                                v.y = pack2<T>(__uint_as_float(u[2]) * f, __uint_as_float(u[3]) * f);
                                v.z = pack2<T>(__uint_as_float(u[4]) * f, __uint_as_float(u[5]) * f);
                                v.w = pack2<T>(__uint_as_float(u[6]) * f, __uint_as_float(u[7]) * f);
                            }
                            if (there && (uint32_t)(c + e) < a.dim) *reinterpret_cast<uint4*>(out + c + e) = v;
                        }
                    }
                    if (there && a.lse) a.lse[(uint64_t)head * a.queries + row] = (top + __log2f(total)) * kFgLn2;
                }
                pairs += n != 0;
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

// ---- few rows: generated tokens over a cache ----
// What bounds this is the reading of the keys, so a block keeps 96 KB of them on their way, and 16 rows at a time ((query, head of the group) pairs) are
// multiplied by the warps' own instructions.  A block has one share of a sequence's keys and one head of k and v.  Of its four warps kW have 16 rows each
// (as many as a sequence has on average), the others the same rows against other keys of a stage; they are joined at the end.
__device__ __forceinline__ void load_matrices(uint32_t from, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(from) : "memory");
}
__device__ __forceinline__ void load_matrices_turned(uint32_t from, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(from) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int DP>
struct FewCfg {
    static constexpr int kKeys = 64, kHalf = kKeys * 128, kTile = kHalf * (DP / 64), kStages = 3 * 128 / DP, kThreads = 128;
    static constexpr size_t kSmem = 1024 + (size_t)2 * kStages * kTile;
};
template <typename T, int DP, int kW>
__global__ void __launch_bounds__(128)
attn_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FgAttnArgs a) {
    using Cfg = FewCfg<DP>;
    constexpr int S = Cfg::kStages, kOwn = 16 * kW, kCols = kOwn / 8;      // keys of a stage that a warp has
    extern __shared__ __align__(1024) unsigned char raw[];
    __shared__ unsigned long long bars[S];
    __shared__ float2 stat[4][16];
    __shared__ int s_stop;
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u, bar0 = smem_u32(bars);
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp / kW;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) mbar_init(bar0 + 8 * i, 1);
        fence_mbar_init();
    }
    fg_grid_enter();
    if (threadIdx.x == 0) s_stop = *reinterpret_cast<volatile int*>(a.dev_status);
    __syncthreads();
    const uint32_t kv = blockIdx.x % a.kv_heads, z = blockIdx.x / a.kv_heads % a.splits, b = blockIdx.x / a.kv_heads / a.splits;
    const FgAttnSeq s(a, b);
    uint32_t lo, hi_share;
    if (s_stop || !s.nq || !s.share(a, z, &lo, &hi_share)) return;
    const uint64_t rows = (uint64_t)s.nq * a.group;
    const uint32_t steps = (a.dim + 15) / 16;
    const float by = a.scale * kFgLog2e;
    uint32_t g = 0;      // stages so far
    for (uint64_t r0 = 0; r0 < rows; r0 += 16 * kW) {
        const uint32_t n_row = (uint32_t)min((uint64_t)(16 * kW), rows - r0);
        const uint32_t hi = min(hi_share, s.seen(a, (uint32_t)((r0 + n_row - 1) / a.group)));
        const uint32_t n = hi > lo ? (hi - lo + Cfg::kKeys - 1) / Cfg::kKeys : 0;
        auto ask = [&](uint32_t i) {      // by one thread
            const uint32_t st = (g + i) % S, bar = bar0 + 8 * st, to = base + 2 * st * Cfg::kTile;
            mbar_expect_tx(bar, 2 * Cfg::kTile);
#pragma unroll
            for (int h = 0; h < DP / 64; ++h) {
                tma_load_3d(to + h * Cfg::kHalf, &tm_k, bar, 64 * h, (int)kv, (int)(s.k0 + lo + i * Cfg::kKeys));
                tma_load_3d(to + Cfg::kTile + h * Cfg::kHalf, &tm_v, bar, 64 * h, (int)kv, (int)(s.k0 + lo + i * Cfg::kKeys));
            }
        };
        if (threadIdx.x == 0)
            for (uint32_t i = 0; i < n && i < (uint32_t)S; ++i) ask(i);
        // Rows of this thread: lane / 4 and 8 more, of the warp's 16.
        uint32_t q[DP / 16][4], seen[2];
        const uint32_t own = (warp % kW) * 16 + lane / 4;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t r = own + 8 * e;
            const bool there = r < n_row;
            const uint32_t i = there ? (uint32_t)((r0 + r) / a.group) : 0, h = there ? (uint32_t)((r0 + r) % a.group) : 0;
            seen[e] = there ? min(hi, s.seen(a, i)) : 0;
            const T* const row = static_cast<const T*>(a.q) + (uint64_t)(s.q0 + i) * a.q_stride + (uint64_t)(kv * a.group + h) * a.dim;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    const uint32_t d = 16 * c + 8 * f + 2 * (lane % 4);
                    q[c][2 * f + e] = there && d < a.dim ? *reinterpret_cast<const uint32_t*>(row + d) : 0;
                }
        }
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f}, o[DP / 8][4];
#pragma unroll
        for (int c = 0; c < DP / 8; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] = 0.0f;
        for (uint32_t i = 0; i < n; ++i) {
            const uint32_t st = (g + i) % S, ks = base + 2 * st * Cfg::kTile, vs = ks + Cfg::kTile, j0 = lo + i * Cfg::kKeys;
            if (!mbar_wait_bounded(bar0 + 8 * st, ((g + i) / S) & 1, kWaitCycles)) {
                atomicOr(a.dev_status, FG_DEVERR_TMA_WAIT);
                s_stop = 1;
            }
            if (j0 + Cfg::kKeys > s.nk) {      // v behind the sequence's end has a weight of zero, but need not be a number
                const uint32_t from = s.nk - j0;
                for (uint32_t w = from * 8 + threadIdx.x; w < Cfg::kKeys * 8; w += 128)
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h) fg_store_shared(vs + h * Cfg::kHalf + w * 16, make_uint4(0, 0, 0, 0));
                __syncthreads();
            }
            float p[kCols][4];
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[c][e] = 0.0f;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                if ((uint32_t)c >= steps) break;
#pragma unroll
                for (int t = 0; t < kCols; t += 2) {
                    uint32_t m[4];
                    const uint32_t key = part * kOwn + 8 * t + (lane & 7) + (lane >> 4) * 8, chunk = 2 * (c & 3) + (lane >> 3 & 1);
                    load_matrices(ks + (c >> 2) * Cfg::kHalf + key * 128 + ((chunk ^ (key & 7)) << 4), m);
                    mma_16x8x16<T>(p[t], q[c], m[0], m[1]);
                    mma_16x8x16<T>(p[t + 1], q[c], m[2], m[3]);
                }
            }
            float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t key = j0 + part * kOwn + 8 * c + 2 * (lane % 4) + (e & 1);
                    p[c][e] = key < seen[e >> 1] ? p[c][e] * by : -INFINITY;
                    most[e >> 1] = fmaxf(most[e >> 1], p[c][e]);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], 1));
                most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], 2));
            }
            if (__any_sync(0xffffffffu, most[0] > top[0] + 8.0f || most[1] > top[1] + 8.0f)) {      // (as in the kernel above)
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float next = fmaxf(top[e], most[e]);
                    f[e] = next == -INFINITY ? 1.0f : fg_ex2_fast(top[e] - next);
                    top[e] = next;
                    sum[e] *= f[e];
                }
#pragma unroll
                for (int c = 0; c < DP / 8; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[c][e] *= f[e >> 1];
            }
            const float less[2] = {top[0] == -INFINITY ? 0.0f : top[0], top[1] == -INFINITY ? 0.0f : top[1]};
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[c][e] = fg_ex2_fast(p[c][e] - less[e >> 1]);
                    sum[e >> 1] += p[c][e];
                }
#pragma unroll
            for (int t = 0; t < kCols; t += 2) {
                const uint32_t w[4] = {pack2<T>(p[t][0], p[t][1]), pack2<T>(p[t][2], p[t][3]), pack2<T>(p[t + 1][0], p[t + 1][1]), pack2<T>(p[t + 1][2], p[t + 1][3])};
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    if ((uint32_t)c >= steps) break;
                    uint32_t m[4];
                    const uint32_t key = part * kOwn + 8 * t + (lane & 15), chunk = 2 * (c & 3) + (lane >> 4);
                    load_matrices_turned(vs + (c >> 2) * Cfg::kHalf + key * 128 + ((chunk ^ (key & 7)) << 4), m);
                    mma_16x8x16<T>(o[2 * c], w, m[0], m[1]);
                    mma_16x8x16<T>(o[2 * c + 1], w, m[2], m[3]);
                }
            }
            __syncthreads();      // the stage is free
            if (s_stop) {      // a wait ran out: nothing is on its way when the block ends
                for (uint32_t l = i; l < n && l < i + S; ++l) mbar_wait_bounded(bar0 + 8 * ((g + l) % S), ((g + l) / S) & 1, kWaitCycles);
                return;
            }
            if (threadIdx.x == 0 && i + S < n) ask(i + S);
        }
        g += n;
        // The warps' sums, over those that had the same rows.
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
            sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
            if (lane % 4 == 0) stat[warp][lane / 4 + 8 * e] = make_float2(top[e], sum[e]);
        }
        __syncthreads();
        float* const sums = reinterpret_cast<float*>(raw + (base - smem_u32(raw)));      // [4][16][DP + 4], where the stages were
        constexpr int kPitch = DP + 4;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float all = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4 / kW; ++w) all = fmaxf(all, stat[w * kW + warp % kW][lane / 4 + 8 * e].x);
            const float f = fg_ex2_fast(top[e] - (all == -INFINITY ? 0.0f : all));
#pragma unroll
            for (int c = 0; c < DP / 8; ++c)
                *reinterpret_cast<float2*>(sums + (warp * 16 + lane / 4 + 8 * e) * kPitch + 8 * c + 2 * (lane % 4)) = make_float2(o[c][2 * e] * f, o[c][2 * e + 1] * f);
        }
        __syncthreads();
        for (uint32_t r = warp; r < n_row; r += 4) {
            const uint32_t w0 = r / 16, in = r % 16;
            float all = -INFINITY, total = 0.0f;
#pragma unroll
            for (int w = 0; w < 4 / kW; ++w) all = fmaxf(all, stat[w * kW + w0][in].x);
            // (A part without a largest score has a sum of zero, or none where its scores are no numbers, which the row's then is not either.)
            const float base_all = all == -INFINITY ? 0.0f : all;
#pragma unroll
            for (int w = 0; w < 4 / kW; ++w) {
                const float2 st = stat[w * kW + w0][in];
                total = __fmaf_rn(fg_ex2_fast(st.x - base_all), st.y, total);
            }
            const uint32_t row = s.q0 + (uint32_t)((r0 + r) / a.group), head = kv * a.group + (uint32_t)((r0 + r) % a.group);
            const uint64_t line = (uint64_t)row * a.heads + head;
            const float f = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                const uint32_t d = 32 * c + lane;
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < 4 / kW; ++w) v += sums[((w * kW + w0) * 16 + in) * kPitch + d];
                if (d < a.dim) {
                    if (a.splits > 1) a.part_out[((uint64_t)z * a.queries * a.heads + line) * a.dim + d] = v;
                    else static_cast<T*>(a.out)[line * a.dim + d] = fg_narrow<T>(v * f);
                }
            }
            if (lane == 0) {
                if (a.splits > 1) a.part_stat[(uint64_t)z * a.queries * a.heads + line] = make_float2(all, total);
                else if (a.lse) a.lse[(uint64_t)head * a.queries + row] = (all + __log2f(total)) * kFgLn2;
            }
        }
        fence_proxy_async();      // the stages are loaded again
        __syncthreads();
    }
}

// ---- backward ----
// Both kinds of tile have a row (of dq) or a key (of dk, dv) per lane, two groups of four warps with half of the columns each, warp 8 loads, warp 9
// multiplies.  Weights are made again from lse.  What a tile's threads leave in tensor memory as an A operand takes the place of what they
// read: columns c / 2 behind the group's first.
//
// dq, by tiles of rows (their q and dout stay): for each tile of keys S = q k', dP = dout v', dS = P (dP - delta), dq += dS k.  Scores have two places, so
// S(j + 1) is there when the weights of j + 1 are wanted: dP(j + 1) dq(j) S(j + 2) are multiplied while the threads work on j + 1.
// dk and dv, by tiles of keys (their k and v stay): for each tile of rows S' = k q', dP' = v dout', dv += P' dout, dk += dS' q, in the order dv(i) S(i + 1)
// dk(i) dP(i + 1): the weights of i + 1 are made while dk(i) and dP(i + 1) are multiplied, dS(i + 1) during dv(i + 1) and S(i + 2).
// 7 products where one kernel that adds dq in memory would have 5, but no sum depends on who comes first, and nothing is read and written again.
template <int DP>
struct BwdCfg {
    static constexpr int kTile = kHalfBytes * (DP / 64), kTwice = DP == 128 ? 3 : 4, kOnce = DP == 128 ? 2 : 3, kThreads = 384;
    static constexpr int kBars = 1 + 2 * kTwice + 2 * kOnce + 2 + 1 + 2 + 1 + 2 + 2 + 1;
    // the two tensors that stay, the rings, lse and delta of two tiles of rows, barriers, the tensor memory's address and a flag
    static constexpr size_t kUsed = (size_t)(2 + kTwice + kOnce) * kTile + 2 * 2 * kRows * 4 + 8 * kBars + 16;
    static constexpr size_t kSmem = kUsed + (kUsed + 1024 <= 227 * 1024 ? 1024 : 227 * 1024 - kUsed);
};
// The f16 operands' factor: a power of two that brings the largest gradient of a score near 2^13, if dout and v are as large as they can be in sequence b's heads that share
// kv's.  (One for the whole call left gradients that are 10^5 times smaller than another sequence's two or three bits.)
__device__ __forceinline__ float gradient_factor(const FgAttnArgs& a, uint32_t b, uint32_t kv) {
    const uint32_t* const most = a.most + 2 * ((uint64_t)b * a.kv_heads + kv);
    const float m = __uint_as_float(most[0]) * __uint_as_float(most[1]) * (float)a.dim;
    if (!(m > 0.0f && m < INFINITY)) return 1.0f;
    const int e = 13 - ilogbf(m);
    return ldexpf(1.0f, e > 60 ? 60 : e < -60 ? -60 : e);
}
// What both kernels begin and end with.
template <int DP>
struct BwdBlock {
    using Cfg = BwdCfg<DP>;
    uint32_t base, bar0, tmem;
    bool go;
    int warp, lane;
    __device__ __forceinline__ uint32_t stay(uint32_t i) const { return base + i * Cfg::kTile; }                              // the tensors that stay
    __device__ __forceinline__ uint32_t twice(uint32_t i) const { return base + (2 + i) * Cfg::kTile; }                       // the ring of what two products read
    __device__ __forceinline__ uint32_t once(uint32_t i) const { return base + (2 + Cfg::kTwice + i) * Cfg::kTile; }          // the other
    __device__ __forceinline__ uint32_t stats(uint32_t i) const { return base + (2 + Cfg::kTwice + Cfg::kOnce) * Cfg::kTile + i * (2 * kRows * 4); }
    __device__ __forceinline__ uint32_t stay_full() const { return bar0; }
    __device__ __forceinline__ uint32_t twice_full(uint32_t i) const { return bar0 + 8 * (1 + i); }
    __device__ __forceinline__ uint32_t twice_empty(uint32_t i) const { return bar0 + 8 * (1 + Cfg::kTwice + i); }
    __device__ __forceinline__ uint32_t once_full(uint32_t i) const { return bar0 + 8 * (1 + 2 * Cfg::kTwice + i); }
    __device__ __forceinline__ uint32_t once_empty(uint32_t i) const { return bar0 + 8 * (1 + 2 * Cfg::kTwice + Cfg::kOnce + i); }
    __device__ __forceinline__ uint32_t more(uint32_t i) const { return bar0 + 8 * (1 + 2 * Cfg::kTwice + 2 * Cfg::kOnce + i); }
    __device__ __forceinline__ uint32_t s_full(uint32_t i) const { return more(i); }          // 2
    __device__ __forceinline__ uint32_t dp_full() const { return more(2); }
    __device__ __forceinline__ uint32_t p_ready() const { return more(3); }
    __device__ __forceinline__ uint32_t ds_ready() const { return more(4); }
    __device__ __forceinline__ uint32_t done() const { return more(5); }
    __device__ __forceinline__ uint32_t stats_full(uint32_t i) const { return more(6 + i); }  // 2
    __device__ __forceinline__ uint32_t stats_empty(uint32_t i) const { return more(8 + i); } // 2
    __device__ __forceinline__ uint32_t drained() const { return more(10); }
    // Dynamic shared memory starts on 1024 bytes, which the tiles need and the largest block has no room to make up for.
    static __device__ __forceinline__ bool fits(const unsigned char* raw, const FgAttnArgs& a) {
        const uint32_t at = smem_u32(raw);
        if (((at + 1023u) & ~1023u) - at + Cfg::kUsed <= Cfg::kSmem) return true;
        if (threadIdx.x == 0) atomicOr(a.dev_status, FG_DEVERR_TMA_WAIT);
        return false;
    }
    __device__ __forceinline__ BwdBlock(unsigned char* raw, const FgAttnArgs& a) {
        base = (smem_u32(raw) + 1023u) & ~1023u;
        bar0 = stats(2);
        unsigned char* const tail = raw + (bar0 + 8 * Cfg::kBars - smem_u32(raw));
        volatile uint32_t* const slot = reinterpret_cast<volatile uint32_t*>(tail);
        warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
        lane = threadIdx.x & 31;
        if (threadIdx.x == 0) {
            for (int i = 0; i < Cfg::kBars; ++i) {
                const int m = i - (1 + 2 * Cfg::kTwice + 2 * Cfg::kOnce);
                mbar_init(bar0 + 8 * i, m == 3 || m == 4 || m == 8 || m == 9 ? 256 : m == 6 || m == 7 ? 64 : 1);
            }
            fence_mbar_init();
        }
        if (warp == 9) {
            tmem_alloc(bar0 + 8 * Cfg::kBars, kTmemCols);
            tmem_relinquish();
        }
        fg_grid_enter();
        if (threadIdx.x == 0) slot[1] = (uint32_t)*reinterpret_cast<volatile int*>(a.dev_status);
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        tmem = __shfl_sync(0xffffffffu, slot[0], 0);
        go = __all_sync(0xffffffffu, slot[1] == 0);
    }
    __device__ __forceinline__ void end() const {
        __syncwarp();
        tc_fence_before();
        __syncthreads();
        if (warp == 9) {
            tc_fence_after();
            tmem_dealloc(tmem, kTmemCols);
        }
    }
    // Loads are waited for by the warp that asked for them, and products by the one that issued them, whatever became of the other roles.
    __device__ __forceinline__ void await_loads(uint32_t n, const FgAttnArgs& a) const {
        if (!await(stay_full(), 0, a.dev_status, FG_DEVERR_TMA_WAIT)) return;
        for (uint32_t i = n > (uint32_t)Cfg::kTwice ? n - Cfg::kTwice : 0; i < n; ++i)
            if (!await(twice_full(i % Cfg::kTwice), (i / Cfg::kTwice) & 1, a.dev_status, FG_DEVERR_TMA_WAIT)) return;
        for (uint32_t i = n > (uint32_t)Cfg::kOnce ? n - Cfg::kOnce : 0; i < n; ++i)
            if (!await(once_full(i % Cfg::kOnce), (i / Cfg::kOnce) & 1, a.dev_status, FG_DEVERR_TMA_WAIT)) return;
    }
    __device__ __forceinline__ void drain(const FgAttnArgs& a) const {
        if (elect_one()) mma_commit(drained());
        __syncwarp();
        await(drained(), 0, a.dev_status, FG_DEVERR_MMA_WAIT);
    }
    // Zeros for rows `from` on of a tile, as far as a product of 16 rows at a time reads.
    __device__ __forceinline__ void clear(uint32_t tile, uint32_t from) const {
        const uint32_t end = round_up(from, 16);
        for (uint32_t i = from * 8 + lane; i < end * 8; i += 32)
#pragma unroll
            for (int h = 0; h < DP / 64; ++h) fg_store_shared(tile + h * kHalfBytes + i * 16, make_uint4(0, 0, 0, 0));
        fence_proxy_async();
        __syncwarp();
    }
    // 128 x n products of two tiles' rows over head_dim.
    __device__ __forceinline__ void rows_by_rows(uint32_t d, uint32_t x, uint32_t y, uint32_t id, uint32_t steps) const {
        const uint64_t x_d = make_desc_kmajor<128>(x), y_d = make_desc_kmajor<128>(y);
        if (steps == DP / 16) {
#pragma unroll
            for (uint32_t c = 0; c < DP / 16; ++c) {
                const uint64_t at = (uint64_t)((c & 3) * 2 + (c >> 2) * (kHalfBytes >> 4));
                mma_f16(d, x_d + at, y_d + at, id, c != 0);
            }
        } else
            for (uint32_t c = 0; c < steps; ++c) {
                const uint64_t at = (uint64_t)((c & 3) * 2 + (c >> 2) * (kHalfBytes >> 4));
                mma_f16(d, x_d + at, y_d + at, id, c != 0);
            }
    }
    // d += (what the two groups left behind `w`) times the first 16 * steps rows of a tile.
    __device__ __forceinline__ void weights_by_rows(uint32_t d, uint32_t w, uint32_t tile, uint32_t id, uint32_t steps, uint32_t add) const {
        const uint64_t t_d = make_desc_mnmajor(tile, kHalfBytes, 1024, 2);
        if (steps == 8) {
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) mma_f16_ta(d, w + (c & 3) * 8 + (c >> 2) * 64, t_d + (uint64_t)(c * 128), id, add | c);
        } else
            for (uint32_t c = 0; c < steps; ++c) mma_f16_ta(d, w + (c & 3) * 8 + (c >> 2) * 64, t_d + (uint64_t)(c * 128), id, add | c);
    }
};

// 64 sums of a lane, times f, as 16-bit columns from `to` on (`columns` of them are there).
template <typename T, int N>
__device__ __forceinline__ void put_sums(uint32_t from, T* to, bool there, int columns, float f) {
#pragma unroll
    for (int c = 0; c < N; c += 32) {
        uint32_t o[32];
        tmem_ld_32x32(from + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
            if constexpr (sizeof(T) == 4) {
                float4* const p = reinterpret_cast<float4*>(to + c + e);
                if (!there || c + e >= columns) continue;
                p[0] = make_float4(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f, __uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
                p[1] = make_float4(__uint_as_float(o[e + 4]) * f, __uint_as_float(o[e + 5]) * f, __uint_as_float(o[e + 6]) * f, __uint_as_float(o[e + 7]) * f);
            } else {
            const uint4 v = make_uint4(pack2<T>(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f), pack2<T>(__uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f),
                                       pack2<T>(__uint_as_float(o[e + 4]) * f, __uint_as_float(o[e + 5]) * f), pack2<T>(__uint_as_float(o[e + 6]) * f, __uint_as_float(o[e + 7]) * f));
            if (there && c + e < columns) *reinterpret_cast<uint4*>(to + c + e) = v;
            }
        }
    }
}

template <typename T, int DP>
__device__ __forceinline__ void tc_dq_tile(const CUtensorMap& tm_q, const CUtensorMap& tm_do, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const FgAttnArgs& a,
                                           uint32_t tokens, uint32_t number, uint32_t kv, const BwdBlock<DP>& blk) {
    using Cfg = BwdCfg<DP>;
    const int warp = blk.warp;
    const uint32_t tmem = blk.tmem, t_dp = tmem + 256, t_dq = tmem + 384;      // scores at 0 and 128
    uint32_t tile;
    const int b = blk.go ? fg_attn_find(a.q_starts, a.sequences, a.queries, 1, tokens, number, &tile) : -1;
    if (b >= 0) {
        const FgAttnSeq s(a, b);
        const uint64_t tok0_ = (uint64_t)tile * tokens;
        const uint32_t tok0 = tok0_ < s.nq ? (uint32_t)tok0_ : s.nq, n_tok = min(tokens, s.nq - tok0);
        const uint32_t hi = __shfl_sync(0xffffffffu, n_tok ? s.seen(a, tok0 + n_tok - 1) : 0, 0), n = (hi + kRows - 1) / kRows;
        const uint32_t fmt = kFormat<T>, dim16 = round_up(a.dim, 16), steps = dim16 / 16;
        if (warp >= 8) reg_release<72>();
        if (warp == 8) {
            // ---- loads: q and dout, then k (read twice) and v ----
            uint32_t j = 0;
            for (; j < n; ++j) {
                const uint32_t u = j % Cfg::kTwice, w = j % Cfg::kOnce;
                if (!await(blk.twice_empty(u), ((j / Cfg::kTwice) & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
                if (!await(blk.once_empty(w), ((j / Cfg::kOnce) & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
                if (elect_one()) {
                    if (j == 0) {
                        mbar_expect_tx(blk.stay_full(), 2 * (DP / 64) * 128 * tokens * a.group);
#pragma unroll
                        for (int h = 0; h < DP / 64; ++h) {
                            tma_load_3d(blk.stay(0) + h * kHalfBytes, &tm_q, blk.stay_full(), 64 * h, (int)(kv * a.group), (int)(s.q0 + tok0));
                            tma_load_3d(blk.stay(1) + h * kHalfBytes, &tm_do, blk.stay_full(), 64 * h, (int)(kv * a.group), (int)(s.q0 + tok0));
                        }
                    }
                    mbar_expect_tx(blk.twice_full(u), Cfg::kTile);
                    mbar_expect_tx(blk.once_full(w), Cfg::kTile);
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h) {
                        tma_load_3d(blk.twice(u) + h * kHalfBytes, &tm_k, blk.twice_full(u), 64 * h, (int)kv, (int)(s.k0 + j * kRows));
                        tma_load_3d(blk.once(w) + h * kHalfBytes, &tm_v, blk.once_full(w), 64 * h, (int)kv, (int)(s.k0 + j * kRows));
                    }
                }
                __syncwarp();
            }
            if (j) blk.await_loads(j, a);
        } else if (warp == 9) {
            // ---- products ----
            const uint32_t id_dq = make_idesc(fmt, 128, dim16) | kIdescBMnMajor;
            auto cols = [&](uint32_t j) { return round_up(min((uint32_t)kRows, hi - j * kRows), 16); };
            bool ok = n != 0 && await(blk.stay_full(), 0, a.dev_status, FG_DEVERR_MMA_WAIT);
            auto scores = [&](uint32_t j) {
                const uint32_t u = j % Cfg::kTwice;
                if (!(ok = await(blk.twice_full(u), (j / Cfg::kTwice) & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) return;
                const uint32_t left = s.nk - j * kRows;
                if (left < kRows && (left & 15)) blk.clear(blk.twice(u), left);      // dS of these keys is zero, k need not be a number
                tc_fence_after();
                if (elect_one()) {
                    blk.rows_by_rows(tmem + (j & 1) * 128, blk.stay(0), blk.twice(u), make_idesc(fmt, 128, cols(j)), steps);
                    mma_commit(blk.s_full(j & 1));
                }
                __syncwarp();
            };
            auto dp = [&](uint32_t j) {
                const uint32_t w = j % Cfg::kOnce;
                if (!(ok = await(blk.once_full(w), (j / Cfg::kOnce) & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) return;
                tc_fence_after();
                if (elect_one()) {
                    blk.rows_by_rows(t_dp, blk.stay(1), blk.once(w), make_idesc(fmt, 128, cols(j)), steps);
                    mma_commit(blk.dp_full());
                    mma_commit(blk.once_empty(w));
                }
                __syncwarp();
            };
            if (ok) scores(0);
            if (ok) dp(0);
            if (ok && n > 1) scores(1);
            for (uint32_t j = 0; ok && j < n; ++j) {
                if (!(ok = await(blk.ds_ready(), j & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) break;
                tc_fence_after();
                if (j + 1 < n) dp(j + 1);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t u = j % Cfg::kTwice;
                    blk.weights_by_rows(t_dq, tmem + (j & 1) * 128, blk.twice(u), id_dq, cols(j) / 16, j);
                    mma_commit(blk.twice_empty(u));
                    if (j + 1 == n) mma_commit(blk.done());
                }
                __syncwarp();
                if (j + 2 < n) scores(j + 2);
            }
            blk.drain(a);
        } else if (warp < 8) {
            reg_acquire<216>();
            const uint32_t side = warp >> 2, r = threadIdx.x & 127, i = tok0 + r / a.group, head = kv * a.group + r % a.group;
            const bool there = r / a.group < n_tok;
            const uint32_t seen = there ? s.seen(a, i) : 0, lanes = (uint32_t)(warp & 3) << 21;
            float lse = INFINITY, delta = 0.0f;
            if (there) {
                const uint64_t line = (uint64_t)head * a.queries + s.q0 + i;
                lse = a.lse_in[line];
                lse = lse == -INFINITY ? INFINITY : lse * kFgLog2e;
                delta = a.delta[line];
            }
            const float factor = std::is_same_v<T, __half> ? gradient_factor(a, b, kv) : 1.0f, by = a.scale * kFgLog2e;
            const float2 by2 = make_float2(by, by), lse2 = make_float2(-lse, -lse), factor2 = make_float2(factor, factor), delta2 = make_float2(-delta * factor, -delta * factor);
            bool ok = true;
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t t_s = tmem + lanes + (j & 1) * 128 + side * 64;
                if (!(ok = await(blk.s_full(j & 1), (j >> 1) & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                tc_fence_after();
                uint32_t x[2][32], y[2][32];
                tmem_ld_32x32(t_s, x[0]);
                tmem_ld_32x32(t_s + 32, x[1]);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float2 e = fg_fma2(make_float2(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])), by2, lse2);
                    x[c / 32][c % 32] = __float_as_uint(fg_ex2_fast(e.x));
                    x[c / 32][c % 32 + 1] = __float_as_uint(fg_ex2_fast(e.y));
                }
                if (!(ok = await(blk.dp_full(), j & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                tc_fence_after();
                tmem_ld_32x32(t_dp + lanes + side * 64, y[0]);
                tmem_ld_32x32(t_dp + lanes + side * 64 + 32, y[1]);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    float2 e = fg_fma2(make_float2(__uint_as_float(y[c / 32][c % 32]), __uint_as_float(y[c / 32][c % 32 + 1])), factor2, delta2);
                    e = fg_mul2(e, make_float2(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])));
                    y[c / 32][c % 32] = __float_as_uint(e.x);
                    y[c / 32][c % 32 + 1] = __float_as_uint(e.y);
                }
                const uint32_t from = j * kRows + side * 64, end = from < seen ? seen - from : 0;
                if (__any_sync(0xffffffffu, end < 64))
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if ((uint32_t)c >= end) y[c / 32][c % 32] = 0;
                uint32_t p[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) p[c] = pack2<T>(__uint_as_float(y[c / 16][c % 16 * 2]), __uint_as_float(y[c / 16][c % 16 * 2 + 1]));
                tmem_st_32x32(t_s, p);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(blk.ds_ready());
            }
            if (ok && n) ok = await(blk.done(), 0, a.dev_status, FG_DEVERR_EPI_WAIT);
            if (ok && n_tok) {
                tc_fence_after();
                T* const to = static_cast<T*>(a.dq) + (uint64_t)(s.q0 + i) * a.q_stride + (uint64_t)head * a.dim + side * (DP / 2);
                const int columns = (int)a.dim - (int)side * (DP / 2);
                if (n) put_sums<T, DP / 2>(t_dq + lanes + side * (DP / 2), to, there, columns, a.scale / factor);
                else if (there)
                    for (int c = 0; c < DP / 2 && c < columns; c += 8) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
            }
        }
    }
}

template <typename T, int DP>
__device__ __forceinline__ void tc_dkv_tile(const CUtensorMap& tm_q, const CUtensorMap& tm_do, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const FgAttnArgs& a,
                                            uint32_t tokens, uint32_t number, uint32_t share, uint32_t kv, const BwdBlock<DP>& blk) {
    using Cfg = BwdCfg<DP>;
    const int warp = blk.warp, lane = blk.lane;
    const uint32_t tmem = blk.tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;      // scores at 0
    uint32_t tile;
    const int b = blk.go ? fg_attn_find(a.k_starts, a.sequences, a.keys, 1, kRows, number, &tile) : -1;
    if (b >= 0) {
        const FgAttnSeq s(a, b);
        const uint64_t j0_ = (uint64_t)tile * kRows;
        const uint32_t j0 = j0_ < s.nk ? (uint32_t)j0_ : s.nk, n_key = min((uint32_t)kRows, s.nk - j0);
        const uint32_t seen0 = n_key ? s.first_query(a, j0) : s.nq, each = ((s.nq - seen0 + tokens - 1) / tokens + a.row_shares - 1) / a.row_shares;
        const uint32_t tok0 = (uint32_t)min((uint64_t)s.nq, seen0 + (uint64_t)share * each * tokens);      // of this share
        const uint32_t left = __shfl_sync(0xffffffffu, (uint32_t)min((uint64_t)(s.nq - tok0), (uint64_t)each * tokens), 0), n = (left + tokens - 1) / tokens;
        const uint32_t fmt = kFormat<T>, dim16 = round_up(a.dim, 16), steps = dim16 / 16;
        auto n_row = [&](uint32_t i) { return min(tokens, left - i * tokens) * a.group; };
        if (warp >= 8) reg_release<72>();
        if (warp == 8) {
            // ---- loads: k and v, then q (read twice, and last) and dout ----
            const uint32_t bytes = DP / 64 * 128 * tokens * a.group;
            uint32_t i = 0;
            for (; i < n; ++i) {
                const uint32_t u = i % Cfg::kTwice, w = i % Cfg::kOnce;
                const int at = (int)(s.q0 + tok0 + i * tokens);
                if (!await(blk.twice_empty(u), ((i / Cfg::kTwice) & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
                if (!await(blk.once_empty(w), ((i / Cfg::kOnce) & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
                if (elect_one()) {
                    if (i == 0) {
                        mbar_expect_tx(blk.stay_full(), 2 * Cfg::kTile);
#pragma unroll
                        for (int h = 0; h < DP / 64; ++h) {
                            tma_load_3d(blk.stay(0) + h * kHalfBytes, &tm_k, blk.stay_full(), 64 * h, (int)kv, (int)(s.k0 + j0));
                            tma_load_3d(blk.stay(1) + h * kHalfBytes, &tm_v, blk.stay_full(), 64 * h, (int)kv, (int)(s.k0 + j0));
                        }
                    }
                    mbar_expect_tx(blk.twice_full(u), bytes);
                    mbar_expect_tx(blk.once_full(w), bytes);
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h) {
                        tma_load_3d(blk.twice(u) + h * kHalfBytes, &tm_q, blk.twice_full(u), 64 * h, (int)(kv * a.group), at);
                        tma_load_3d(blk.once(w) + h * kHalfBytes, &tm_do, blk.once_full(w), 64 * h, (int)(kv * a.group), at);
                    }
                }
                __syncwarp();
            }
            if (i) blk.await_loads(i, a);
        } else if (warp == 9) {
            // ---- products ----
            const uint32_t id_sum = make_idesc(fmt, 128, dim16) | kIdescBMnMajor;
            bool ok = n != 0 && await(blk.stay_full(), 0, a.dev_status, FG_DEVERR_MMA_WAIT);
            // (rows behind the sequence's end weigh nothing, but may not be numbers: zeros, and no product goes further)
            auto scores = [&](uint32_t i) {
                const uint32_t u = i % Cfg::kTwice, rows = n_row(i);
                if (!(ok = await(blk.twice_full(u), (i / Cfg::kTwice) & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) return;
                if (rows & 15) blk.clear(blk.twice(u), rows);
                tc_fence_after();
                if (elect_one()) {
                    blk.rows_by_rows(tmem, blk.stay(0), blk.twice(u), make_idesc(fmt, 128, round_up(rows, 16)), steps);
                    mma_commit(blk.s_full(0));
                }
                __syncwarp();
            };
            auto dp = [&](uint32_t i) {
                const uint32_t w = i % Cfg::kOnce, rows = n_row(i);
                if (!(ok = await(blk.once_full(w), (i / Cfg::kOnce) & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) return;
                if (rows & 15) blk.clear(blk.once(w), rows);
                tc_fence_after();
                if (elect_one()) {
                    blk.rows_by_rows(t_dp, blk.stay(1), blk.once(w), make_idesc(fmt, 128, round_up(rows, 16)), steps);
                    mma_commit(blk.dp_full());
                }
                __syncwarp();
            };
            if (ok) scores(0);
            if (ok) dp(0);
            for (uint32_t i = 0; ok && i < n; ++i) {
                const uint32_t row_steps = (n_row(i) + 15) / 16;
                if (!(ok = await(blk.p_ready(), i & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) break;
                tc_fence_after();
                if (elect_one()) {
                    blk.weights_by_rows(t_dv, tmem, blk.once(i % Cfg::kOnce), id_sum, row_steps, i);
                    mma_commit(blk.once_empty(i % Cfg::kOnce));
                }
                __syncwarp();
                if (i + 1 < n) scores(i + 1);
                if (!ok || !(ok = await(blk.ds_ready(), i & 1, a.dev_status, FG_DEVERR_MMA_WAIT))) break;
                tc_fence_after();
                if (elect_one()) {
                    blk.weights_by_rows(t_dk, t_dp, blk.twice(i % Cfg::kTwice), id_sum, row_steps, i);
                    mma_commit(blk.twice_empty(i % Cfg::kTwice));
                    if (i + 1 == n) mma_commit(blk.done());
                }
                __syncwarp();
                if (i + 1 < n) dp(i + 1);
            }
            blk.drain(a);
        } else if (warp >= 10) {
            // ---- lse (in powers of two; infinite where a row weighs nothing) and delta of the tiles' rows ----
            const float factor = std::is_same_v<T, __half> ? gradient_factor(a, b, kv) : 1.0f;
            const uint32_t first = (warp - 10) * 32 + lane;
            for (uint32_t i = 0; i < n; ++i) {
                if (!await(blk.stats_empty(i & 1), ((i >> 1) & 1) ^ 1, a.dev_status, FG_DEVERR_TMA_WAIT)) break;
                const uint32_t rows = n_row(i);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t r = first + 64 * h;
                    float lse = INFINITY, delta = 0.0f;
                    if (r < rows) {
                        const uint64_t line = (uint64_t)(kv * a.group + r % a.group) * a.queries + s.q0 + tok0 + i * tokens + r / a.group;
                        lse = a.lse_in[line];
                        lse = lse == -INFINITY ? INFINITY : lse * kFgLog2e;
                        delta = a.delta[line] * factor;
                    }
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(blk.stats(i & 1) + 4 * r), "f"(-lse) : "memory");
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(blk.stats(i & 1) + 4 * (kRows + r)), "f"(-delta) : "memory");
                }
                mbar_arrive(blk.stats_full(i & 1));
            }
        } else {
            reg_acquire<216>();
            const uint32_t side = warp >> 2, key = j0 + (threadIdx.x & 127), lanes = (uint32_t)(warp & 3) << 21;
            const bool there = (threadIdx.x & 127) < n_key;
            const uint32_t first = there ? s.first_query(a, key) : s.nq;      // the first query that sees the key
            const float factor = std::is_same_v<T, __half> ? gradient_factor(a, b, kv) : 1.0f, by = a.scale * kFgLog2e;
            const float2 by2 = make_float2(by, by), factor2 = make_float2(factor, factor);
            bool ok = true;
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t t_s = tmem + lanes + side * 64, stat = blk.stats(i & 1) + side * 256;
                if (!(ok = await(blk.stats_full(i & 1), (i >> 1) & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                if (!(ok = await(blk.s_full(0), i & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                tc_fence_after();
                uint32_t x[2][32], y[2][32], p[32];
                tmem_ld_32x32(t_s, x[0]);
                tmem_ld_32x32(t_s + 32, x[1]);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    const uint4 l = fg_load_shared(stat + 4 * c);
                    float2 e = fg_fma2(make_float2(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])), by2, make_float2(__uint_as_float(l.x), __uint_as_float(l.y)));
                    x[c / 32][c % 32] = __float_as_uint(fg_ex2_fast(e.x));
                    x[c / 32][c % 32 + 1] = __float_as_uint(fg_ex2_fast(e.y));
                    e = fg_fma2(make_float2(__uint_as_float(x[c / 32][c % 32 + 2]), __uint_as_float(x[c / 32][c % 32 + 3])), by2, make_float2(__uint_as_float(l.z), __uint_as_float(l.w)));
                    x[c / 32][c % 32 + 2] = __float_as_uint(fg_ex2_fast(e.x));
                    x[c / 32][c % 32 + 3] = __float_as_uint(fg_ex2_fast(e.y));
                }
                // Columns before `start` do not see the key.
                const uint32_t at = tok0 + i * tokens, skip = (first > at ? min(first - at, tokens) : 0) * a.group, start = skip > side * 64 ? skip - side * 64 : 0;
                const bool some = __any_sync(0xffffffffu, start != 0);
                if (some)
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if ((uint32_t)c < start) x[c / 32][c % 32] = 0;
#pragma unroll
                for (int c = 0; c < 32; ++c) p[c] = pack2<T>(__uint_as_float(x[c / 16][c % 16 * 2]), __uint_as_float(x[c / 16][c % 16 * 2 + 1]));
                tmem_st_32x32(t_s, p);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(blk.p_ready());
                if (!(ok = await(blk.dp_full(), i & 1, a.dev_status, FG_DEVERR_EPI_WAIT))) break;
                tc_fence_after();
                tmem_ld_32x32(t_s + 128, y[0]);
                tmem_ld_32x32(t_s + 160, y[1]);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    const uint4 l = fg_load_shared(stat + 4 * (kRows + c));
                    float2 e = fg_fma2(make_float2(__uint_as_float(y[c / 32][c % 32]), __uint_as_float(y[c / 32][c % 32 + 1])), factor2, make_float2(__uint_as_float(l.x), __uint_as_float(l.y)));
                    e = fg_mul2(e, make_float2(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])));
                    y[c / 32][c % 32] = __float_as_uint(e.x);
                    y[c / 32][c % 32 + 1] = __float_as_uint(e.y);
                    e = fg_fma2(make_float2(__uint_as_float(y[c / 32][c % 32 + 2]), __uint_as_float(y[c / 32][c % 32 + 3])), factor2, make_float2(__uint_as_float(l.z), __uint_as_float(l.w)));
                    e = fg_mul2(e, make_float2(__uint_as_float(x[c / 32][c % 32 + 2]), __uint_as_float(x[c / 32][c % 32 + 3])));
                    y[c / 32][c % 32 + 2] = __float_as_uint(e.x);
                    y[c / 32][c % 32 + 3] = __float_as_uint(e.y);
                }
                mbar_arrive(blk.stats_empty(i & 1));
                if (some)
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if ((uint32_t)c < start) y[c / 32][c % 32] = 0;
#pragma unroll
                for (int c = 0; c < 32; ++c) p[c] = pack2<T>(__uint_as_float(y[c / 16][c % 16 * 2]), __uint_as_float(y[c / 16][c % 16 * 2 + 1]));
                tmem_st_32x32(t_s + 128, p);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(blk.ds_ready());
            }
            if (ok && n) ok = await(blk.done(), 0, a.dev_status, FG_DEVERR_EPI_WAIT);
            if (ok && n_key) {
                tc_fence_after();
                T* const to = side ? static_cast<T*>(a.dk) + (uint64_t)(s.k0 + key) * a.k_stride + (uint64_t)kv * a.dim
                                   : static_cast<T*>(a.dv) + (uint64_t)(s.k0 + key) * a.v_stride + (uint64_t)kv * a.dim;
                if (a.row_shares > 1) {
                    float* const part = fg_attn_part(a, share, side ? 0 : 1, s.k0 + key, kv);
                    if (n) put_sums<float, DP>((side ? t_dk : t_dv) + lanes, part, there, (int)a.dim, side ? a.scale / factor : 1.0f);
                    else if (there)
                        for (uint32_t c = 0; c < a.dim; c += 4) *reinterpret_cast<uint4*>(part + c) = make_uint4(0, 0, 0, 0);
                } else if (n) put_sums<T, DP>((side ? t_dk : t_dv) + lanes, to, there, (int)a.dim, side ? a.scale / factor : 1.0f);
                else if (there)
                    for (uint32_t c = 0; c < a.dim; c += 8) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
            }
        }
    }
}

// Tiles of keys first (they have more to do), then tiles of rows, which fill the SMs that the last of those leave; the longest of either first.
template <typename T, int DP>
__global__ void __launch_bounds__(BwdCfg<DP>::kThreads, 1)
attn_tc_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FgAttnArgs a, uint32_t tokens, uint32_t key_tiles, uint32_t row_tiles) {
    extern __shared__ __align__(1024) unsigned char raw[];
    if (!BwdBlock<DP>::fits(raw, a)) return;
    const BwdBlock<DP> blk(raw, a);
    const uint32_t number = blockIdx.x / a.kv_heads, kv = blockIdx.x % a.kv_heads, key_blocks = key_tiles * a.row_shares;
    if (number < key_blocks) tc_dkv_tile<T, DP>(tm_q, tm_do, tm_k, tm_v, a, tokens, number / a.row_shares, number % a.row_shares, kv, blk);
    else tc_dq_tile<T, DP>(tm_q, tm_do, tm_k, tm_v, a, tokens, row_tiles - 1 - (number - key_blocks), kv, blk);
    blk.end();
}

// delta_i = dout_i . out_i: L lanes of 16 bytes per row of a head, [heads][queries].
template <typename T, int L>
__global__ void __launch_bounds__(256) attn_tc_delta_kernel(const FgAttnArgs a, float* delta) {
    constexpr int kLines = 256 / L * 4;      // of (query, head): four per thread
    fg_grid_enter();
    const uint32_t sub = threadIdx.x % L;
    const uint64_t lines = (uint64_t)a.queries * a.heads, first = (uint64_t)blockIdx.x * kLines + threadIdx.x / L;
    uint4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t line = first + i * (256 / L), at = line * a.dim + sub * 8;
        const bool there = line < lines && sub * 8 < a.dim;
        x[i] = there ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.out) + at) : make_uint4(0, 0, 0, 0);
        y[i] = there ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.dout) + at) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t line = first + i * (256 / L);
        float u[8], v[8], d = 0.0f;
        FgPack<T>::widen(x[i], u);
        FgPack<T>::widen(y[i], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) d = __fmaf_rn(u[e], v[e], d);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if (sub == 0 && line < lines) delta[line % a.heads * a.queries + line / a.heads] = d;
    }
}
// The largest |dout| and |v| of the sequences' rows, by heads of k and v (as bits, so NaN is larger than infinity): 64 rows of a head, or of its queries' heads, a block, first those of dout.
template <typename T>
__global__ void __launch_bounds__(256) attn_most_kernel(const FgAttnArgs a, uint32_t row_tiles, uint32_t* most) {
    fg_grid_enter();
    const bool keys = blockIdx.x >= row_tiles;
    uint32_t tile;
    const int b = fg_attn_find(keys ? a.k_starts : a.q_starts, a.sequences, keys ? a.keys : a.queries, 1, 64, blockIdx.x - (keys ? row_tiles : 0), &tile);
    if (b < 0) return;
    const FgAttnSeq s(a, b);
    const uint64_t rows = keys ? s.nk : s.nq, r0 = (uint64_t)tile * 64, stride = keys ? a.v_stride : (uint64_t)a.heads * a.dim;
    if (r0 >= rows) return;
    const uint32_t kv = blockIdx.y, width = (keys ? 1 : a.group) * a.dim, line = width / 8;      // (in 16-byte words)
    const uint32_t n = (uint32_t)min((uint64_t)64, rows - r0) * line;
    const T* const x = static_cast<const T*>(keys ? a.v : a.dout) + ((keys ? s.k0 : s.q0) + r0) * stride + (uint64_t)kv * width;
    uint32_t m = 0;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        const uint32_t r = i / line, c = i - r * line;
        float v[8];
        FgPack<T>::widen(*reinterpret_cast<const uint4*>(x + r * stride + c * 8), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(fabsf(v[e])));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0 && m) atomicMax(most + 2 * ((uint64_t)b * a.kv_heads + kv) + keys, m);      // (the largest of numbers: whoever comes first)
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
    if (tiles * a.kv_heads >= (1ull << 31) - 65536) return fg_fail(ctx, FG_ERR_INVALID_ARGUMENT, "attention: tensor too large");
    const uint64_t all = tiles * a.kv_heads, sms = fg_free_sms(ctx);
    fg_launch(ctx, attn_tc_fwd_kernel<T, DP>, (unsigned)(all < sms ? all : sms), Cfg::kThreads, Cfg::kSmem, q, k, v, a, tokens, (uint32_t)tiles, fg_arrivals(ctx));
    FG_LAUNCHED(ctx);
    return FG_OK;
}

template <typename T, int DP>
int32_t bwd_launch(fg_ctx* ctx, FgAttnArgs a) {
    using Cfg = BwdCfg<DP>;
    constexpr bool half = std::is_same_v<T, __half>;
    const uint64_t lines = (uint64_t)a.queries * a.heads;
    int32_t s = fg_attn_bwd_room(ctx, a, kRows, half);
    if (s != FG_OK) return s;
    uint32_t* const most = const_cast<uint32_t*>(a.most);
    float* const delta = const_cast<float*>(a.delta);
    const uint32_t lanes = a.dim > 64 ? 16 : a.dim > 32 ? 8 : a.dim > 16 ? 4 : a.dim > 8 ? 2 : 1, per = 1024 / lanes;
    const auto kernel = lanes == 16 ? attn_tc_delta_kernel<T, 16> : lanes == 8 ? attn_tc_delta_kernel<T, 8> : lanes == 4 ? attn_tc_delta_kernel<T, 4>
                        : lanes == 2 ? attn_tc_delta_kernel<T, 2> : attn_tc_delta_kernel<T, 1>;
    if (lines) {
        fg_launch(ctx, kernel, (unsigned)((lines + per - 1) / per), 256, 0, a, delta);
        FG_LAUNCHED(ctx);
    }
    if (half) {
        FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(most, 0, 8ull * a.sequences * a.kv_heads, ctx->stream));
        const uint64_t row_tiles = fg_attn_tiles(a.sequences, a.queries, 1, 64), both = row_tiles + fg_attn_tiles(a.sequences, a.keys, 1, 64);
        fg_launch(ctx, attn_most_kernel<T>, dim3((unsigned)both, a.kv_heads), 256, 0, a, (uint32_t)row_tiles, most);
        FG_LAUNCHED(ctx);
    }
    const uint32_t tokens = kRows / a.group;
    CUtensorMap q, d, k, v;
    if ((s = make_map(ctx, &q, a.q, half, a.dim, a.heads, a.queries, a.q_stride, a.group, tokens)) != FG_OK) return s;
    if ((s = make_map(ctx, &d, a.dout, half, a.dim, a.heads, a.queries, (uint64_t)a.heads * a.dim, a.group, tokens)) != FG_OK) return s;
    if ((s = make_map(ctx, &k, a.k, half, a.dim, a.kv_heads, a.keys, a.k_stride, 1, kRows)) != FG_OK) return s;
    if ((s = make_map(ctx, &v, a.v, half, a.dim, a.kv_heads, a.keys, a.v_stride, 1, kRows)) != FG_OK) return s;
    const uint64_t row_tiles = a.dq ? fg_attn_tiles(a.sequences, a.queries, 1, tokens) : 0, key_tiles = a.dk ? fg_attn_tiles(a.sequences, a.keys, 1, kRows) : 0;
    const uint64_t blocks = (row_tiles + key_tiles * a.row_shares) * a.kv_heads;
    if (blocks >= 1ull << 31) return fg_fail(ctx, FG_ERR_INVALID_ARGUMENT, "attention: tensor too large");
    static std::atomic<uint64_t> done{0};
    if ((s = allow_shared(ctx, done, attn_tc_bwd_kernel<T, DP>, Cfg::kSmem)) != FG_OK) return s;
    fg_launch(ctx, attn_tc_bwd_kernel<T, DP>, (unsigned)blocks, Cfg::kThreads, Cfg::kSmem, q, d, k, v, a, tokens, (uint32_t)key_tiles, (uint32_t)row_tiles);
    FG_LAUNCHED(ctx);
    return a.row_shares > 1 ? fg_attn_fold(ctx, half ? FG_DTYPE_F16 : FG_DTYPE_BF16, a) : FG_OK;
}

template <typename T, int DP, int kW>
int32_t few_launch(fg_ctx* ctx, const FgAttnArgs& a) {
    using Cfg = FewCfg<DP>;
    constexpr bool half = std::is_same_v<T, __half>;
    static std::atomic<uint64_t> done{0};
    int32_t s = allow_shared(ctx, done, attn_few_kernel<T, DP, kW>, Cfg::kSmem);
    if (s != FG_OK) return s;
    CUtensorMap k, v;
    if ((s = make_map(ctx, &k, a.k, half, a.dim, a.kv_heads, a.keys, a.k_stride, 1, Cfg::kKeys)) != FG_OK) return s;
    if ((s = make_map(ctx, &v, a.v, half, a.dim, a.kv_heads, a.keys, a.v_stride, 1, Cfg::kKeys)) != FG_OK) return s;
    const uint64_t blocks = (uint64_t)a.sequences * a.splits * a.kv_heads;
    if (blocks >= 1ull << 31) return fg_fail(ctx, FG_ERR_INVALID_ARGUMENT, "attention: tensor too large");
    fg_launch(ctx, attn_few_kernel<T, DP, kW>, (unsigned)blocks, Cfg::kThreads, Cfg::kSmem, k, v, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T>
int32_t few(fg_ctx* ctx, const FgAttnArgs& a, uint32_t rows) {
    if (a.dim <= 64) return rows <= 16 ? few_launch<T, 64, 1>(ctx, a) : rows <= 32 ? few_launch<T, 64, 2>(ctx, a) : few_launch<T, 64, 4>(ctx, a);
    return rows <= 16 ? few_launch<T, 128, 1>(ctx, a) : rows <= 32 ? few_launch<T, 128, 2>(ctx, a) : few_launch<T, 128, 4>(ctx, a);
}

}  // namespace

bool fg_attn_tc_suits(const fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a) {
    if (dtype == FG_DTYPE_F32 || !ctx->tmap_encode || a.dim % 8 || a.dim > 128 || a.group > (uint32_t)kRows || !(a.scale > 0.0f) || !a.keys || !a.queries) return false;
    const uint64_t strides = a.q_stride | a.k_stride | a.v_stride;
    return strides % 8 == 0 && fg_aligned16(a.q) && fg_aligned16(a.k) && fg_aligned16(a.v) && fg_aligned16(a.out) && fg_aligned16(a.dout) && fg_aligned16(a.dq) &&
           fg_aligned16(a.dk) && fg_aligned16(a.dv);
}
int32_t fg_attn_tc_fwd(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a) {
    if (dtype == FG_DTYPE_F16) return a.dim <= 64 ? fwd_launch<__half, 64>(ctx, a) : fwd_launch<__half, 128>(ctx, a);
    return a.dim <= 64 ? fwd_launch<__nv_bfloat16, 64>(ctx, a) : fwd_launch<__nv_bfloat16, 128>(ctx, a);
}
int32_t fg_attn_tc_bwd(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a) {
    if (dtype == FG_DTYPE_F16) return a.dim <= 64 ? bwd_launch<__half, 64>(ctx, a) : bwd_launch<__half, 128>(ctx, a);
    return a.dim <= 64 ? bwd_launch<__nv_bfloat16, 64>(ctx, a) : bwd_launch<__nv_bfloat16, 128>(ctx, a);
}
int32_t fg_attn_few(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a, uint32_t rows) {
    return dtype == FG_DTYPE_F16 ? few<__half>(ctx, a, rows) : few<__nv_bfloat16>(ctx, a, rows);
}
