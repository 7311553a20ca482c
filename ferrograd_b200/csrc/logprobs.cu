// Log probabilities of given tokens, with the rows' entropies and largest entries, and the gradient of the logits.
//
// With z = scale * x, m the largest z of the row and l = sum(exp(z - m)): lse = m + log l, logprob = z[target] - lse and
// entropy = log l - sum(exp(z - m) * (z - m)) / l.  The gradient, of dlogprob and dentropy: dx_c = scale * (dlogprob * ([c == target] - p_c) -
// dentropy * p_c * (log p_c + entropy)) with p_c = exp(z_c - lse).
#include "ptx_sm100.cuh"
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
    uint32_t blocks;      // of a row's cluster
};
struct LogprobBwdArgs {
    const void* x;
    const uint32_t* targets;
    const float *lse, *entropy, *dlogprob, *dentropy;
    void* dx;
    uint32_t rows, cols;
    float scale;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A row as 16-byte words of memory, with the elements before the first whole word and behind the last.
template <typename T>
struct RowWords {
    static constexpr int E = FgPack<T>::E;
    uint32_t head, words, tail;
    __device__ __forceinline__ RowWords(const T* row, uint32_t cols) {
        const uint32_t off = reinterpret_cast<uintptr_t>(row) & 15u;
        head = min(off ? (16 - off) / (uint32_t)sizeof(T) : 0u, cols);
        words = (cols - head) / E;
        tail = cols - head - words * E;
    }
};

// A part of a row in powers of two: the largest entry, with y = (x - m) * scale * log2(e) the sum of 2^y, and of 2^y * y.
struct alignas(16) Part {
    float m, l, e;
    uint32_t count;      // of alternatives (between blocks)
    // Another part.  sum w (y + d) = sum w y + d sum w; a part whose weights vanish beside the other's adds nothing, whatever its distance.
    __device__ __forceinline__ void join(const Part& o, float by) {
        const float top = fmaxf(m, o.m);
        if (top == -INFINITY) {      // no weight, unless it is NaN
            l += o.l;
            return;
        }
        const float d = (m - top) * by, od = (o.m - top) * by, w = fg_ex2_fast(d), ow = fg_ex2_fast(od);
        e = (w == 0.0f ? 0.0f : w * __fmaf_rn(l, d, e)) + (ow == 0.0f ? 0.0f : ow * __fmaf_rn(o.l, od, o.e));
        l = __fmaf_rn(l, w, o.l * ow);
        m = top;
    }
    __device__ __forceinline__ void join_lanes(float by) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) join(Part{__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, l, o), __shfl_xor_sync(0xffffffffu, e, o)}, by);
    }
};

// Entries in the order of the alternatives: larger values first, of equal ones the lower index; 0 for what is never among them.
__device__ __forceinline__ uint64_t order_key(float v, uint32_t c) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);      // (zeros of both signs are equal)
    return (uint64_t)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - c);
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// One thread's way through its words of a row, kWords on their way at a time.
// What bounds it beside the memory is issue: per entry a fused multiply-add, a maximum, an exponential and one or two sums.  The largest entry so far moves
// only when a batch of words has a larger one, which is rare behind the first; the alternatives' search costs nothing else than its place.
constexpr int kWords = 4, kThreads = 256, kList = 2048, kMaxCluster = 8;
template <typename T, bool kEntropy, bool kTop>
struct Scan {
    static constexpr int E = FgPack<T>::E;
    Part p{-INFINITY, 0.0f, 0.0f};      // (its largest; the sums by pairs)
    float2 l2 = make_float2(0.0f, 0.0f), e2 = l2;
    uint64_t best = 0;      // order_key of the largest entry, or of its value and a later index
    float by;
    __device__ __forceinline__ explicit Scan(float by_) : by(by_) {}
    __device__ __forceinline__ void rise(float top, uint64_t key) {
        const float d = (p.m - top) * by, f = fg_ex2_fast(d);
        if (kEntropy) e2 = f == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(f * __fmaf_rn(l2.x, d, e2.x), f * __fmaf_rn(l2.y, d, e2.y));
        l2 = make_float2(l2.x * f, l2.y * f);
        p.m = top;
        if (kTop) best = key;
    }
    // Two entries.  The difference comes first: an entry times `by` may be beyond the largest number.
    __device__ __forceinline__ void add(float2 x, float2 less) {
        const float2 y = fg_mul2(fg_add2(x, less), make_float2(by, by)), w = make_float2(fg_ex2_fast(y.x), fg_ex2_fast(y.y));
        l2 = fg_add2(l2, w);
        if (kEntropy) e2 = fg_fma2(w, make_float2(fmaxf(y.x, -1024.0f), fmaxf(y.y, -1024.0f)), e2);      // (a weight of zero times -inf)
    }
    __device__ __forceinline__ float less() const { return p.m == -INFINITY ? 0.0f : -p.m; }
    __device__ __forceinline__ void one(float x, uint32_t c) {
        if (x > p.m) rise(x, kTop ? order_key(x, c) : 0);
        add(make_float2(x, -INFINITY), make_float2(less(), 0.0f));
    }
    __device__ __forceinline__ Part part() const { return Part{p.m, l2.x + l2.y, e2.x + e2.y}; }
    // Words w, w + step, .. below `end`, the first at p.
    __device__ __forceinline__ void words(const T* row, uint32_t head, uint32_t w, uint32_t end, uint32_t step) {
        const uint4* const at = reinterpret_cast<const uint4*>(row + head);
        for (; w < end; w += kWords * step) {
            uint4 v[kWords];
            float2 x[kWords][E / 2];
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                if (w + i * step < end) v[i] = __ldg(at + w + i * step);
            float most[kWords], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                if (w + i * step < end) FgPack<T>::widen(v[i], x[i]);
                else
#pragma unroll
                    for (int e = 0; e < E / 2; ++e) x[i][e] = make_float2(-INFINITY, -INFINITY);
                most[i] = -INFINITY;
#pragma unroll
                for (int e = 0; e < E / 2; ++e) most[i] = max3(most[i], x[i][e].x, x[i][e].y);
                top = fmaxf(top, most[i]);
            }
            if (top > p.m) {
                uint32_t at_word = w;      // the first word that has it; its last index stands for the entry's, so that the key is no larger
                if (kTop)
#pragma unroll
                    for (int i = kWords - 1; i >= 0; --i)
                        if (most[i] == top) at_word = w + i * step;
                rise(top, kTop ? order_key(top, head + at_word * E + E - 1) : 0);
            }
            const float2 from = make_float2(less(), less());
#pragma unroll
            for (int i = 0; i < kWords; ++i)
#pragma unroll
                for (int e = 0; e < E / 2; ++e) add(x[i][e], from);
        }
    }
};

__device__ __forceinline__ void write_statistics(const LogprobArgs& a, uint32_t r, const Part& p, float at_target) {
    const float log_l = __log2f(p.l) * kLn2;
    const bool none = p.l == 0.0f;
    if (a.logprob) a.logprob[r] = none ? -INFINITY : __fmaf_rn(at_target - p.m, a.scale, -log_l);
    if (a.entropy) a.entropy[r] = none ? 0.0f : log_l - p.e / p.l * kLn2;
    if (a.lse) a.lse[r] = none ? -INFINITY : __fmaf_rn(p.m, a.scale, log_l);
}
__device__ __forceinline__ void write_padding(const LogprobArgs& a, uint32_t r, uint32_t thread, uint32_t threads) {
    if (thread == 0) {
        if (a.logprob) a.logprob[r] = 0.0f;
        if (a.entropy) a.entropy[r] = 0.0f;
        if (a.lse) a.lse[r] = 0.0f;
    }
    for (uint32_t i = thread; i < a.top; i += threads) {
        a.top_ids[(uint64_t)r * a.top + i] = FG_NO_TOKEN;
        a.top_logprobs[(uint64_t)r * a.top + i] = -INFINITY;
    }
}

// Short rows without alternatives: a warp each.
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(kThreads) logprob_warp_kernel(const LogprobArgs a) {
    fg_grid_enter();
    const uint64_t r = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (r >= a.rows) return;
    const uint32_t lane = threadIdx.x & 31, target = a.targets ? a.targets[r] : 0;
    if (target >= a.cols) return write_padding(a, (uint32_t)r, lane, 32);
    const T* const row = static_cast<const T*>(a.x) + r * a.cols;
    const RowWords<T> w(row, a.cols);
    const float by = a.scale * kLog2e, at_target = fg_widen(row[target]);
    Scan<T, kEntropy, false> scan(by);
    if (lane < w.head) scan.one(fg_widen(row[lane]), lane);
    scan.words(row, w.head, lane, w.words, 32);
    if (lane < w.tail) scan.one(fg_widen(row[a.cols - w.tail + lane]), 0);
    Part p = scan.part();
    p.join_lanes(by);
    if (lane == 0) write_statistics(a, (uint32_t)r, p, at_target);
}

// Places of a list's entries in the order of the alternatives: how many are larger.  `put` gets those below `top`.
template <typename F>
__device__ __forceinline__ void place_entries(const uint64_t* list, uint32_t n, uint32_t top, F put) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t k = list[i];
        uint32_t larger = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < n; ++j) larger += list[j] > k;
        if (larger < top) put(larger, k);
    }
}

// A row per cluster of blocks, each with a stretch of it.
// The alternatives: the warps that have words each name the same number of their lanes' largest entries, `top` or more together, so the least of them is a bound
// that the top entries reach, and few others do: a second reading (from the L2) lists those, and the list is put in order by counting how many are larger.  Where
// more than the list holds reach the bound (a few threads have them), the largest below the one before is sought top times over.  The blocks' lists go to
// the first, which puts them in order the same way.
template <typename T, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kThreads, 4) logprob_row_kernel(const LogprobArgs a) {
    constexpr int E = FgPack<T>::E, kWarps = kThreads / 32;
    __shared__ Part parts[kWarps], others[kMaxCluster];
    __shared__ uint64_t keys[kWarps], list[kTop ? kList : 1], sorted[kTop ? kMaxTop : 1], all[kTop ? kMaxTop * kMaxCluster : 1];
    __shared__ uint32_t count, names[kWarps];
    fg_grid_enter();
    const uint32_t blocks = a.blocks, rank = blockIdx.x % blocks, r = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31;
    const uint32_t target = a.targets ? a.targets[r] : 0;
    if (target >= a.cols) {      // (the whole cluster)
        if (rank == 0) write_padding(a, r, tid, kThreads);
        return;
    }
    const T* const row = static_cast<const T*>(a.x) + (uint64_t)r * a.cols;
    const RowWords<T> w(row, a.cols);
    if (blocks > 1) fgptx::cluster_arrive();
    const uint32_t from = (uint32_t)((uint64_t)w.words * rank / blocks), to = (uint32_t)((uint64_t)w.words * (rank + 1) / blocks);
    const float by = a.scale * kLog2e, at_target = rank == 0 ? fg_widen(row[target]) : 0.0f;
    Scan<T, kEntropy, kTop> scan(by);
    const bool has_head = rank == 0 && tid < w.head, has_tail = rank + 1 == blocks && tid < w.tail;
    if (has_head) scan.one(fg_widen(row[tid]), tid);
    scan.words(row, w.head, from + tid, to, kThreads);
    if (has_tail) scan.one(fg_widen(row[a.cols - w.tail + tid]), a.cols - w.tail + tid);
    Part p = scan.part();
    p.join_lanes(by);
    if (lane == 0) parts[tid >> 5] = p;
    if (kTop) {
        const uint32_t busy = min((uint32_t)kWarps, (to - from + 31) / 32), each = (a.top + (busy ? busy : 1) - 1) / (busy ? busy : 1);
        uint32_t v = (uint32_t)(scan.best >> 32), named = 0;
        uint64_t least = ~0ull;
        for (; named < each; ++named) {
            const uint32_t most = __reduce_max_sync(0xffffffffu, v), from_lane = __ffs(__ballot_sync(0xffffffffu, v == most)) - 1;
            if (most == 0) break;      // no more
            const uint64_t k = __shfl_sync(0xffffffffu, scan.best, from_lane);
            if (k < least) least = k;
            if (lane == from_lane) v = 0;
        }
        if (lane == 0) { keys[tid >> 5] = least; names[tid >> 5] = named; }
        if (tid == 0) count = 0;
        if (tid < kMaxTop) sorted[tid] = 0;
    }
    __syncthreads();
    p = lane < kWarps ? parts[lane] : Part{-INFINITY, 0.0f, 0.0f};
    p.join_lanes(by);      // (every warp)
    uint32_t n = 0;        // of this block's alternatives
    if (kTop) {
        uint64_t least = ~0ull;
        uint32_t named = 0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            least = least < keys[i] ? least : keys[i];
            named += names[i];
        }
        if (named < a.top) least = 1;      // every entry that may be an alternative
        // The entries of this block that reach `floor`: found by words, their indices from a short loop (unrolled into every entry's place it took longer to
        // fetch than to run).
        auto each = [&](float floor, auto take) {
            if (has_head) take(fg_widen(row[tid]), tid);
            if (has_tail) take(fg_widen(row[a.cols - w.tail + tid]), a.cols - w.tail + tid);
            const uint4* const at = reinterpret_cast<const uint4*>(row + w.head);
            for (uint32_t i = from + tid; i < to; i += kWords * kThreads) {
                uint4 v[kWords];
#pragma unroll
                for (int j = 0; j < kWords; ++j)
                    if (i + j * kThreads < to) v[j] = __ldg(at + i + j * kThreads);
                uint32_t reach = 0;
#pragma unroll
                for (int j = 0; j < kWords; ++j)
                    if (i + j * kThreads < to) {
                        float x[E];
                        FgPack<T>::widen(v[j], x);
#pragma unroll
                        for (int e = 0; e < E; ++e) reach |= (x[e] >= floor ? 1u : 0u) << (j * E + e);
                    }
                while (reach) {
                    const uint32_t bit = __ffs(reach) - 1, c = w.head + (i + bit / E * kThreads) * E + bit % E;
                    reach &= reach - 1;
                    take(fg_widen(row[c]), c);
                }
            }
        };
        // The value of the bound: no key is made for what lies below.
        const uint32_t hi = (uint32_t)(least >> 32);
        const float floor = least == 1 ? -INFINITY : __uint_as_float(hi & 0x80000000u ? hi & 0x7fffffffu : ~hi);
        if (scan.p.m >= floor)      // (no entry of other threads reaches it)
            each(floor, [&](float x, uint32_t c) {
                const uint64_t k = order_key(x, c);
                if (k < least) return;
                const uint32_t i = atomicAdd(&count, 1);      // (the order in the list does not matter)
                if (i < kList) list[i] = k;
            });
        __syncthreads();
        n = count;
        if (n <= kList) {
            place_entries(list, n, a.top, [&](uint32_t i, uint64_t k) { sorted[i] = k; });
        } else {
            uint64_t last = ~0ull;
            for (uint32_t i = 0; i < a.top; ++i) {
                uint64_t k = 0;
                each(-INFINITY, [&](float x, uint32_t c) {
                    const uint64_t o = order_key(x, c);
                    if (o < last) k = max64(k, o);
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) k = max64(k, __shfl_xor_sync(0xffffffffu, k, o));
                __syncthreads();
                if (lane == 0) keys[tid >> 5] = k;
                __syncthreads();
                for (int i2 = 0; i2 < kWarps; ++i2) k = max64(k, keys[i2]);
                if (tid == 0) sorted[i] = k;
                last = k;
            }
        }
        n = min(n, a.top);
        __syncthreads();
    }
    if (blocks > 1) {
        fgptx::cluster_wait();      // (the first block has been there since the arrival above)
        if (rank != 0) {
            if (kTop && tid < n) {
                const uint32_t at = fgptx::map_to_cta((uint32_t)__cvta_generic_to_shared(all + rank * kMaxTop + tid), 0);
                fgptx::st_cluster(at, (uint32_t)sorted[tid], (uint32_t)(sorted[tid] >> 32));
            }
            if (tid == 0) {
                const uint32_t at = fgptx::map_to_cta((uint32_t)__cvta_generic_to_shared(others + rank), 0);
                fgptx::st_cluster(at, __float_as_uint(p.m), __float_as_uint(p.l));
                fgptx::st_cluster(at + 8, __float_as_uint(p.e), n);
            }
        }
        fgptx::cluster_sync_all();
        if (rank != 0) return;
        if (kTop) {
            // The lists behind one another, then in order.
            uint32_t total = n;
            if (tid < n) list[tid] = sorted[tid];
            for (uint32_t o = 1; o < blocks; ++o) {
                const uint32_t m = others[o].count;
                if (tid < m) list[total + tid] = all[o * kMaxTop + tid];
                total += m;
            }
            __syncthreads();
            place_entries(list, total, a.top, [&](uint32_t i, uint64_t k) { sorted[i] = k; });      // (there are as many as before, or more)
            __syncthreads();
        }
        for (uint32_t o = 1; o < blocks; ++o) p.join(others[o], by);
    }
    if (tid == 0) write_statistics(a, r, p, at_target);
    if (kTop && tid < a.top) {
        const uint64_t k = sorted[tid];
        const uint32_t hi = (uint32_t)(k >> 32);
        const float x = __uint_as_float(hi & 0x80000000u ? hi & 0x7fffffffu : ~hi);
        a.top_ids[(uint64_t)r * a.top + tid] = k ? 0xffffffffu - (uint32_t)k : FG_NO_TOKEN;
        a.top_logprobs[(uint64_t)r * a.top + tid] = k ? __fmaf_rn(x - p.m, a.scale, -(__log2f(p.l) * kLn2)) : -INFINITY;
    }
}

// The gradient: a warp per stretch of 32 * kWords words of a row.
// With y = log p = x * scale - lse: dx = p * (A + B y), A = -scale * (dlogprob + dentropy * entropy), B = -scale * dentropy.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_bwd_kernel(const LogprobBwdArgs a, uint32_t stretches) {
    constexpr int E = FgPack<T>::E;
    fg_grid_enter();
    const uint64_t unit = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), r = unit / stretches;
    if (r >= a.rows) return;
    const uint32_t part = (uint32_t)(unit - r * stretches), lane = threadIdx.x & 31;
    const T* const row = static_cast<const T*>(a.x) + r * a.cols;
    T* const to = static_cast<T*>(a.dx) + r * a.cols;
    // Words of the gradient's row: those of the logits' where both lie alike on 16-byte boundaries, elements otherwise.
    const bool alike = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(to)) & 15u) == 0;
    RowWords<T> w(row, a.cols);
    if (!alike) { w.head = a.cols; w.words = w.tail = 0; }
    const uint32_t first = part * 32 * kWords + lane;
    uint4 v[kWords];
    const uint4* const at = reinterpret_cast<const uint4*>(row + w.head);
#pragma unroll
    for (int i = 0; i < kWords; ++i)
        if (first + 32 * i < w.words) v[i] = at[first + 32 * i];
    const uint32_t target = a.targets ? a.targets[r] : 0xfffffffeu;
    const float lse = a.lse[r], gl = a.dlogprob ? a.scale * a.dlogprob[r] : 0.0f, ge = a.dentropy ? a.scale * a.dentropy[r] : 0.0f, h = a.dentropy ? a.entropy[r] : 0.0f;
    const bool zero = (a.targets && target >= a.cols) || lse == -INFINITY;
    const float A = -__fmaf_rn(ge, h, gl), B = -ge;
    auto gradient = [&](float x, uint32_t c) {
        const float y = __fmaf_rn(x, a.scale, -lse);
        const float g = fg_ex2_fast(y * kLog2e) * __fmaf_rn(B, fmaxf(y, -1024.0f), A);      // (a weight of zero times -inf)
        return zero ? 0.0f : c == target ? g + gl : g;
    };
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        const uint32_t word = first + 32 * i;
        if (word >= w.words) continue;
        float x[E];
        FgPack<T>::widen(v[i], x);
        const uint32_t c = w.head + word * E;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = gradient(x[e], c + e);
        reinterpret_cast<uint4*>(to + w.head)[word] = FgPack<T>::narrow(x);
    }
    if (!alike) {
        const uint32_t begin = part * 32 * kWords * E, end = min(a.cols, begin + 32 * kWords * E);
        for (uint32_t c = begin + lane; c < end; c += 32) to[c] = fg_narrow<T>(gradient(fg_widen(row[c]), c));
    } else if (part == 0) {
        if (lane < w.head) to[lane] = fg_narrow<T>(gradient(fg_widen(row[lane]), lane));
        const uint32_t c = a.cols - w.tail + lane;
        if (lane < w.tail) to[c] = fg_narrow<T>(gradient(fg_widen(row[c]), c));
    }
}

template <typename T, bool kEntropy, bool kTop>
int32_t row_launch(fg_ctx* ctx, LogprobArgs a) {
    // Few rows are shared out: blocks for about four on an SM, each with 2 KB at least.
    a.blocks = 1;
    while (a.blocks < kMaxCluster && (uint64_t)a.rows * a.blocks * 2 <= 4ull * ctx->sm_count && (uint64_t)a.cols * sizeof(T) >= 4096ull * a.blocks) a.blocks *= 2;
    if ((uint64_t)a.rows * a.blocks >= 1ull << 31) return fg_fail(ctx, FG_ERR_INVALID_ARGUMENT, "fg_logprobs_fwd: tensor too large");
    fg_launch_cluster(ctx, logprob_row_kernel<T, kEntropy, kTop>, a.rows * a.blocks, kThreads, 0, a.blocks, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T>
int32_t logprobs_fwd(fg_ctx* ctx, const LogprobArgs& a) {
    const bool entropy = a.entropy;
    if (a.top) return entropy ? row_launch<T, true, true>(ctx, a) : row_launch<T, false, true>(ctx, a);
    if ((uint64_t)a.cols * sizeof(T) <= 8192 && a.rows > 4u * ctx->sm_count) {
        fg_launch(ctx, entropy ? logprob_warp_kernel<T, true> : logprob_warp_kernel<T, false>, (unsigned)(((uint64_t)a.rows + 7) / 8), kThreads, 0, a);
        FG_LAUNCHED(ctx);
        return FG_OK;
    }
    return entropy ? row_launch<T, true, false>(ctx, a) : row_launch<T, false, false>(ctx, a);
}
template <typename T>
int32_t logprobs_bwd(fg_ctx* ctx, const LogprobBwdArgs& a) {
    constexpr uint32_t each = 32 * kWords * FgPack<T>::E;
    const uint32_t stretches = (uint32_t)(((uint64_t)a.cols + each - 1) / each);
    const uint64_t blocks = ((uint64_t)a.rows * stretches + 7) / 8;
    if (blocks >= 1ull << 31) return fg_fail(ctx, FG_ERR_INVALID_ARGUMENT, "fg_logprobs_bwd: tensor too large");
    fg_launch(ctx, logprob_bwd_kernel<T>, (unsigned)blocks, kThreads, 0, a, stretches);
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
    FG_REQUIRE(ctx, cols >= 1 && cols <= 1u << 31, "fg_logprobs_fwd: cols must be 1 to 2^31");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_logprobs_fwd: tensor too large");
    FG_REQUIRE(ctx, scale > 0.0f && scale <= 0x1p127f, "fg_logprobs_fwd: scale must be > 0, and 2^127 at most");      // (times log2 e it stays a number)
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
    return FG_BY_DTYPE(dtype, logprobs_fwd, ctx, LogprobArgs{logits, targets, rows, cols, top, scale, logprob_out, entropy_out, lse_out, top_ids_out, top_logprobs_out, 1});
}

int32_t fg_logprobs_bwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* logits, const uint32_t* targets, float scale,
                        const float* lse, const float* entropy, const float* dlogprob, const float* dentropy, void* dlogits) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_logprobs_bwd: unknown dtype");
    FG_REQUIRE(ctx, logits && lse && dlogits, "fg_logprobs_bwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1 && cols <= 1u << 31, "fg_logprobs_bwd: cols must be 1 to 2^31");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_logprobs_bwd: tensor too large");
    FG_REQUIRE(ctx, scale > 0.0f && scale <= 0x1p127f, "fg_logprobs_bwd: scale must be > 0, and 2^127 at most");
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
