// One token per row of logits: temperature, top-k, top-p, min-p, and a draw with the caller's random numbers.
//
// With m the largest logit of a row and w = exp((x - m) / T), whole numbers carry the weights: q = round(2^42 w).  Their sums are
// exact in 64 bits (2^21 columns at most), so neither the order of a sum nor who adds it shows in the result, and a running sum
// can be cut anywhere.  The exponent is taken in 64-bit floating point: what an f32 exponential is off by (2^-22) would put the draw
// on the other side of a border between two tokens once in some hundred rows of 32000.
//
// Logits are compared as ordered 32-bit keys.  A border (the k-th largest, the last of the nucleus) is found by parting the range
// of keys that still holds it into 256 pieces and adding up what lies in each: counts for top-k, weights for top-p; four or five
// rounds leave one key.  Of equal logits at the border the first ones are kept.
#include "rows.cuh"

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr unsigned kFull = 0xffffffffu;
constexpr double kOne = 4398046511104.0;      // 2^42

struct SampleArgs {
    const void* logits;
    const float *u, *temperature;
    const uint32_t* top_k;
    const float *top_p, *min_p;
    uint32_t* token;
    float* prob;
    uint32_t rows, cols;
};

// Order of keys = order of logits; 0 for what is never drawn (-inf, NaN).  -0 and +0 have one key.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

struct Weights {
    double m, c;          // the largest logit; log2(e) / T
    bool all_or_none;     // the largest is +inf: it alone has weight
    __device__ __forceinline__ double of(uint32_t key, uint32_t kmax) const {
        if (key == kmax) return 1.0;
        return all_or_none ? 0.0 : exp2(((double)logit_of(key) - m) * c);
    }
    __device__ __forceinline__ uint64_t whole(uint32_t key, uint32_t kmax) const { return (uint64_t)__double2ll_rn(of(key, kmax) * kOne); }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
__device__ __forceinline__ uint64_t block_sum64(uint64_t v, uint64_t* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_sum64(v);
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = warp_sum64(red[lane]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ uint32_t block_max32(uint32_t v, uint64_t* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = __reduce_max_sync(kFull, v);
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = __reduce_max_sync(kFull, (uint32_t)red[lane]);
    __syncthreads();
    return v;
}

struct Border { uint32_t key; uint64_t above, at; };      // the sum over larger keys, and over this one

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    __shared__ uint64_t red[kWarps], hist[256], mass[kWarps], ties[kWarps];
    __shared__ Border border;
    __shared__ uint32_t next_lo, next_hi, chosen;
    fg_grid_enter();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t n = a.cols;
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* row = static_cast<const T*>(a.logits) + (uint64_t)r * n;
        auto key_at = [&](uint32_t i) { return key_of(fg_widen(row[i])); };
        uint32_t kmax = 0, imin = 0;      // imin: ~(smallest key)
        uint64_t count = 0;
        for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t k = key_at(i);
            kmax = max(kmax, k);
            if (k) { imin = max(imin, ~k); ++count; }
        }
        kmax = block_max32(kmax, red);
        const uint32_t kmin = ~block_max32(imin, red);
        count = block_sum64(count, red);
        if (kmax == 0) {
            if (tid == 0) { a.token[r] = FG_NO_TOKEN; if (a.prob) a.prob[r] = 0.0f; }
            continue;
        }
        const float temperature = a.temperature ? a.temperature[r] : 1.0f;
        if (!(temperature > 0.0f)) {      // the first maximum
            uint32_t first = 0;
            for (uint32_t i = tid; i < n; i += kThreads)
                if (key_at(i) == kmax) { first = ~i; break; }
            first = ~block_max32(first, red);
            if (tid == 0) { a.token[r] = first; if (a.prob) a.prob[r] = 1.0f; }
            continue;
        }
        const Weights w{(double)logit_of(kmax), 1.4426950408889634 / (double)temperature, logit_of(kmax) == INFINITY};

        // The border at which the sum over the keys from the top down reaches `target`; all that have a key reach it.
        auto find = [&](uint32_t lo, uint64_t target, bool by_mass) {
            uint32_t hi = kmax;
            uint64_t above = 0;
            Border at{};
            for (int round = 0; round < 5; ++round) {      // 32 bits of range, eight less after each
                const int bits = 32 - __clz(hi - lo), shift = bits > 8 ? bits - 8 : 0;
                for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
                __syncthreads();
                for (uint32_t i = tid; i < n; i += kThreads) {
                    const uint32_t k = key_at(i);
                    if (k >= lo && k <= hi) {
                        const uint64_t v = by_mass ? w.whole(k, kmax) : 1;
                        if (v) atomicAdd((unsigned long long*)&hist[(k - lo) >> shift], (unsigned long long)v);
                    }
                }
                __syncthreads();
                if (tid == 0) {
                    int b = 255;
                    uint64_t s = above;
                    while (b > 0 && s + hist[b] < target) s += hist[b--];
                    border = Border{lo + ((uint32_t)b << shift), s, hist[b]};
                    next_lo = lo + ((uint32_t)b << shift);
                    next_hi = next_lo + min(hi - next_lo, (1u << shift) - 1);
                }
                __syncthreads();
                at = border;
                lo = next_lo; hi = next_hi; above = at.above;
                __syncthreads();
                if (shift == 0) break;
            }
            return at;
        };

        // Kept: keys above `cut`, and the first `ties_kept` of those at it.
        uint32_t cut = kmin;
        uint64_t ties_kept = ~0ull;
        const uint32_t k = a.top_k ? a.top_k[r] : 0;
        if (k != 0 && k < count) {
            const Border at = find(kmin, k, false);
            cut = at.key;
            ties_kept = k - at.above;
        }
        const float p = a.top_p ? a.top_p[r] : 1.0f;
        if (p < 1.0f) {
            uint64_t s = 0, t = 0;
            for (uint32_t i = tid; i < n; i += kThreads) {
                const uint32_t key = key_at(i);
                if (key > cut) s += w.whole(key, kmax);
                else if (key == cut) ++t;
            }
            s = block_sum64(s, red);
            t = block_sum64(t, red);
            const uint64_t at_cut = w.whole(cut, kmax);
            s += min(t, ties_kept) * at_cut;
            const uint64_t target = max((uint64_t)1, (uint64_t)__double2ull_ru((double)max(p, 0.0f) * (double)s));
            const Border at = find(cut, target, true);
            const uint64_t each = w.whole(at.key, kmax), need = (target - at.above + each - 1) / each;
            ties_kept = at.key == cut ? min(ties_kept, need) : need;
            cut = at.key;
        }
        const float mp = a.min_p ? a.min_p[r] : 0.0f;
        const double least = mp > 0.0f ? (double)min(mp, 1.0f) : 0.0;
        // (the smallest key that min_p keeps is not looked for: a weight is compared where it is needed)
        const uint64_t at_cut = w.of(cut, kmax) >= least ? w.whole(cut, kmax) : 0;

        // The draw.  A warp holds a stretch of the row; sums over the stretches before it say how many ties at the cut it keeps.
        const uint32_t len = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
        const uint32_t i0 = min((uint64_t)n, (uint64_t)warp * len), i1 = min((uint64_t)n, (uint64_t)i0 + len);
        auto weigh = [&](uint32_t key) {
            if (key <= cut) return (uint64_t)0;
            const double v = w.of(key, kmax);
            return v >= least ? (uint64_t)__double2ll_rn(v * kOne) : (uint64_t)0;
        };
        uint64_t s = 0, t = 0;
        for (uint32_t i = i0 + lane; i < i1; i += 32) {
            const uint32_t key = key_at(i);
            s += weigh(key);
            t += key == cut;
        }
        s = warp_sum64(s);
        t = warp_sum64(t);
        if (lane == 0) { mass[warp] = s; ties[warp] = t; }
        if (tid == 0) chosen = FG_NO_TOKEN;
        __syncthreads();
        uint64_t before = 0, total = 0, ties_before = 0, left = ties_kept;      // of this warp's stretch
        for (int j = 0; j < kWarps; ++j) {
            if (j == warp) { before = total; ties_before = ties_kept - left; }
            const uint64_t kept = min(left, ties[j]);
            total += mass[j] + kept * at_cut;
            left -= kept;
        }
        const float uu = a.u[r];
        const uint64_t goal = (uint64_t)((double)(uu > 0.0f ? min(uu, 0.99999994f) : 0.0f) * (double)total);
        const uint64_t end = before + mass[warp] + min(ties[warp], ties_kept - ties_before) * at_cut;
        if (before <= goal && goal < end) {
            uint64_t sum = before, room = ties_kept - ties_before;
            for (uint32_t i = i0; i < i1; i += 32) {
                const uint32_t key = i + lane < i1 ? key_at(i + lane) : 0;
                const unsigned same = __ballot_sync(kFull, key == cut && key != 0);
                uint64_t v = weigh(key);
                if (key == cut && key != 0 && (uint64_t)__popc(same & ((1u << lane) - 1)) < room) v = at_cut;
                uint64_t run = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t up = __shfl_up_sync(kFull, run, o);
                    if (lane >= o) run += up;
                }
                const unsigned over = __ballot_sync(kFull, sum + run > goal);
                if (over) {
                    if (lane == __ffs(over) - 1) {
                        a.token[r] = i + lane;
                        if (a.prob) a.prob[r] = (float)((double)v / (double)total);
                    }
                    break;
                }
                sum += __shfl_sync(kFull, run, 31);
                room -= min(room, (uint64_t)__popc(same));
            }
        }
        __syncthreads();
    }
}

template <typename T>
int32_t sample(fg_ctx* ctx, const SampleArgs& a) {
    const uint32_t cap = 2u * ctx->sm_count;
    fg_launch(ctx, sample_kernel<T>, a.rows < cap ? a.rows : cap, kThreads, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

}  // namespace

extern "C" int32_t fg_sample(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* logits, const float* u,
                             const float* temperature, const uint32_t* top_k, const float* top_p, const float* min_p, uint32_t* token_out,
                             float* prob_out) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_sample: unknown dtype");
    FG_REQUIRE(ctx, logits && u && token_out, "fg_sample: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1 && cols <= FG_SAMPLE_MAX_COLS, "fg_sample: cols must be 1 to FG_SAMPLE_MAX_COLS");
    FG_REQUIRE(ctx, fg_at_element(logits, fg_dtype_size(dtype)) && fg_at_element(u, 4) && fg_at_element(temperature, 4) && fg_at_element(top_k, 4) &&
                        fg_at_element(top_p, 4) && fg_at_element(min_p, 4) && fg_at_element(token_out, 4) && fg_at_element(prob_out, 4),
               "fg_sample: a tensor does not start at an element");
    if (rows == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, sample, ctx, SampleArgs{logits, u, temperature, top_k, top_p, min_p, token_out, prob_out, rows, cols});
}
