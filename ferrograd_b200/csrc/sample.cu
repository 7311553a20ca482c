// One token per row of logits: temperature, top-k, top-p, min-p, and a draw with the caller's random numbers.
//
// With m the largest logit of a row and w = exp((x - m) / T), whole numbers carry the weights: q = round(2^42 w).  Their sums are
// exact in 64 bits (2^21 columns at most), so neither the order of a sum nor who adds it shows in the result, and a running sum
// can be cut anywhere.  The exponent is taken in 64-bit floating point: what an f32 exponential is off by (2^-22) would put the draw
// on the other side of a border between two tokens once in some hundred rows of 32000.
//
// A row is read once, by a cluster of CTAs that keep their slices in shared memory.  Few of its tokens can be drawn when it is
// filtered, so the first thing is to find a bound below the border (by the threads' own maxima for top-k, by a histogram for top-p) and to
// send what lies above it, in order, to the cluster's first CTA, which then works on a short list while the others are done.  A row
// whose list would not fit (equal logits, wide filters) is worked on where it lies, by all CTAs, with the same functions.
//
// Logits are compared as ordered keys.  A border (the k-th largest, the last of the nucleus) is found by parting the range of keys that still
// holds it into 256 pieces and adding up what lies in each: counts for top-k, weights for top-p; up to four rounds leave one key.  Of
// equal logits at the border the first ones are kept.
#include <cooperative_groups.h>

#include "rows.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxCtas = 8;
constexpr int kBins = 2048;                   // of a 32nd of an octave of weight
constexpr uint32_t kLocal = 1024, kGathered = 4096;      // candidates of a CTA, of a row
constexpr unsigned kFull = 0xffffffffu;
constexpr double kOne = 4398046511104.0;      // 2^42

struct SampleArgs {
    const void* logits;
    const float *u, *temperature;
    const uint32_t* top_k;
    const float *top_p, *min_p;
    uint32_t* token;
    float* prob;
    uint32_t rows, cols, slice;               // columns of a CTA
};

// Order of keys = order of logits; 0 for what is never drawn (-inf, NaN).  -0 and +0 have one key.  The low bits that a 16-bit type does not
// have are left out.
template <typename T> constexpr int kDrop = sizeof(T) == 4 ? 0 : std::is_same_v<T, __half> ? 13 : 16;
template <typename T>
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f), key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x > -INFINITY ? key >> kDrop<T> : 0;
}
template <typename T>
__device__ __forceinline__ float logit_of(uint32_t key) {
    const uint32_t k = key << kDrop<T>;
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~(k | ((1u << kDrop<T>) - 1)));
}

// 2^(i / 64)
__device__ const double kRoots[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284, 1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418, 1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687, 1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303, 1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647, 1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267, 1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062, 1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656, 1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};

// round(2^42 exp((x - m) / T)), by 2^t = 2^(n / 64) 2^r with |r| <= 1 / 128 and five terms of the series of 2^r (2^-54 of it).
template <typename T>
struct Weights {
    const double* roots;
    double m, c;              // the largest logit; log2(e) / T
    uint32_t kmax;
    __device__ __forceinline__ double scaled(uint32_t key) const {      // 2^42 w, not rounded; 0 below 2^-44
        if (key == kmax) return kOne;
        const double t = ((double)logit_of<T>(key) - m) * c;
        if (!(t > -44.0)) return 0.0;
        constexpr double kMagic = 6755399441055744.0;      // 1.5 * 2^52: a sum with it has its whole part in the low word
        const double y = __fma_rn(t, 64.0, kMagic);
        const int j = __double2loint(y);
        const double r = __fma_rn(y - kMagic, -0.015625, t);
        constexpr double l = 0.69314718055994530942, c2 = l * l / 2, c3 = l * l * l / 6, c4 = l * l * l * l / 24, c5 = l * l * l * l * l / 120;
        double p = __fma_rn(r, c5, c4);
        p = __fma_rn(r, p, c3);
        p = __fma_rn(r, p, c2);
        p = __fma_rn(r, p, l);
        p = __fma_rn(r, p, 1.0);
        const double v = roots[j & 63] * p;
        return __hiloint2double(__double2hiint(v) + ((j >> 6) + 42 << 20), __double2loint(v));
    }
    static __device__ __forceinline__ uint64_t whole(double v) { return (uint64_t)__double_as_longlong(v + 4503599627370496.0) & 0xfffffffffffffull; }
    __device__ __forceinline__ uint64_t operator()(uint32_t key) const { return whole(scaled(key)); }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

struct Border { uint32_t key; uint64_t above, at; };      // the sum over larger keys, and over this one

struct Shared {
    double roots[64];
    uint64_t hist[2][256];
    uint64_t slots[2][2];                 // what a CTA tells the others
    uint64_t red[kWarps], mass[kWarps], ties[kWarps];
    uint32_t bins[kBins];
    uint2 local[kLocal];                  // (key, column)
    Border border;
    uint32_t next_lo, next_hi, found;
};

// What the functions below go over: units of kPer keys, in the order of the columns.
template <typename T>
struct HeldSlice {      // a slice in shared memory, by 16-byte words; masked where a word reaches over the slice's ends
    static constexpr int kPer = FgPack<T>::E;
    const uint4* words;
    uint32_t units, column;               // of the first word's first element (it may lie before the slice)
    __device__ __forceinline__ void values(uint32_t u, float (&x)[kPer]) const { FgPack<T>::widen(words[u], x); }
    __device__ __forceinline__ void keys(uint32_t u, uint32_t (&k)[kPer]) const {
        float x[kPer];
        values(u, x);
#pragma unroll
        for (int e = 0; e < kPer; ++e) k[e] = key_of<T>(x[e]);
    }
    __device__ __forceinline__ uint32_t column_of(uint32_t u, int e) const { return column + u * kPer + e; }
};
template <typename T>
struct FarSlice {       // a slice that shared memory does not hold
    static constexpr int kPer = 1;
    const T* data;
    uint32_t units, column;
    __device__ __forceinline__ void values(uint32_t u, float (&x)[1]) const { x[0] = fg_widen(data[u]); }
    __device__ __forceinline__ void keys(uint32_t u, uint32_t (&k)[1]) const { k[0] = key_of<T>(fg_widen(data[u])); }
    __device__ __forceinline__ uint32_t column_of(uint32_t u, int) const { return column + u; }
};
struct List {
    static constexpr int kPer = 1;
    const uint2* entries;
    uint32_t units;
    __device__ __forceinline__ void keys(uint32_t u, uint32_t (&k)[1]) const { k[0] = entries[u].x; }
    __device__ __forceinline__ uint32_t column_of(uint32_t u, int) const { return entries[u].y; }
};

// A block and, where kAll, the other CTAs of its cluster.
struct Team {
    Shared& sh;
    uint32_t ctas, cta;
    int turn = 0, round = 0;              // buffers: what is read by others in one step is written again two steps later
    __device__ __forceinline__ uint64_t block_sum(uint64_t v) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        v = warp_sum64(v);
        __syncthreads();
        if (lane == 0) sh.red[warp] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += sh.red[w];
        return v;
    }
    __device__ __forceinline__ uint32_t block_max(uint32_t v) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        v = __reduce_max_sync(kFull, v);
        __syncthreads();
        if (lane == 0) sh.red[warp] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v = max(v, (uint32_t)sh.red[w]);
        return v;
    }
    // Every CTA's pair, to every thread: f(cta, a, b) in the order of the CTAs.
    template <typename F>
    __device__ __forceinline__ void exchange(uint64_t a, uint64_t b, F f) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) { sh.slots[turn][0] = a; sh.slots[turn][1] = b; }
        cluster.sync();
        for (uint32_t c = 0; c < ctas; ++c) {
            const uint64_t* const p = cluster.map_shared_rank(&sh.slots[turn][0], c);
            f(c, p[0], p[1]);
        }
        turn ^= 1;
    }
};

// The border at which the sum over the keys from kmax down to lo (counts, or weights) reaches `target`; all of them together do.
template <bool kAll, typename S, typename T>
__device__ Border find_border(Team& team, const S& source, const Weights<T>& w, uint32_t lo, uint64_t target, bool by_weight) {
    Shared& sh = team.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t hi = w.kmax;
    Border at{};
    uint64_t above = 0;
    for (int round = 0; round < 5; ++round) {      // 32 bits of range, eight less after each
        const int bits = 32 - __clz(hi - lo), shift = bits > 8 ? bits - 8 : 0;
        uint64_t* const hist = sh.hist[team.round ^= 1];
        hist[tid] = 0;
        __syncthreads();
        for (uint32_t u = tid; u < source.units; u += kThreads) {
            uint32_t k[S::kPer];
            source.keys(u, k);
#pragma unroll
            for (int e = 0; e < S::kPer; ++e)
                if (k[e] >= lo && k[e] <= hi) {
                    const uint64_t v = by_weight ? w(k[e]) : 1;
                    if (v) atomicAdd((unsigned long long*)&hist[(k[e] - lo) >> shift], (unsigned long long)v);
                }
        }
        uint64_t v = 0;
        if (kAll) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
            for (uint32_t c = 0; c < team.ctas; ++c) v += cluster.map_shared_rank(hist, c)[tid];
        } else {
            __syncthreads();
            v = hist[tid];
        }
        uint64_t from = v;      // the sum over this piece and those above it
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t down = __shfl_down_sync(kFull, from, o);
            if (lane + o < 32) from += down;
        }
        if (lane == 0) sh.red[warp] = from;
        __syncthreads();
        for (int j = warp + 1; j < kWarps; ++j) from += sh.red[j];
        from += above;
        if (from >= target ? from - v < target : tid == 0) {
            sh.border = Border{lo + ((uint32_t)tid << shift), from - v, v};
            sh.next_lo = lo + ((uint32_t)tid << shift);
            sh.next_hi = sh.next_lo + min(hi - sh.next_lo, (1u << shift) - 1);
        }
        __syncthreads();
        at = sh.border;
        lo = sh.next_lo; hi = sh.next_hi; above = at.above;
        if (shift == 0) break;
    }
    __syncthreads();
    return at;
}

// Keys above `cut` and the first `ties` of those at it, of weight `least` (in parts of 2^42) or more: the first at which their running sum
// exceeds u times the total.
template <bool kAll, typename S, typename T>
__device__ void draw(Team& team, const S& source, const Weights<T>& w, uint32_t cut, uint64_t ties, double least, float u, uint32_t* token, float* prob) {
    Shared& sh = team.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const double cut_scaled = cut ? w.scaled(cut) : 0.0;
    const uint64_t at_cut = cut_scaled >= least ? w.whole(cut_scaled) : 0;
    auto weigh = [&](uint32_t key) -> uint64_t {
        if (key <= cut) return 0;
        const double v = w.scaled(key);
        return v >= least ? w.whole(v) : 0;
    };
    const uint32_t len = ((source.units + kWarps - 1) / kWarps + 31) / 32 * 32;      // a warp's stretch
    const uint32_t u0 = min(source.units, warp * len), u1 = min(source.units, u0 + len);
    uint64_t s = 0, t = 0;
    for (uint32_t i = u0 + lane; i < u1; i += 32) {
        uint32_t k[S::kPer];
        source.keys(i, k);
#pragma unroll
        for (int e = 0; e < S::kPer; ++e) {
            s += weigh(k[e]);
            t += k[e] == cut && cut;
        }
    }
    s = warp_sum64(s);
    t = warp_sum64(t);
    __syncthreads();
    if (lane == 0) { sh.mass[warp] = s; sh.ties[warp] = t; }
    __syncthreads();
    uint64_t before = 0, total = 0, room = ties;      // before this CTA; room for ties at the cut
    auto add = [&](uint64_t mass, uint64_t same) {
        const uint64_t kept = min(room, same);
        room -= kept;
        return mass + kept * at_cut;
    };
    uint64_t own_mass = 0, own_ties = 0;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) { own_mass += sh.mass[j]; own_ties += sh.ties[j]; }
    uint64_t own_room = ties;
    if (kAll)
        team.exchange(own_mass, own_ties, [&](uint32_t c, uint64_t mass, uint64_t same) {
            if (c == team.cta) { before = total; own_room = room; }
            total += add(mass, same);
        });
    else total = add(own_mass, own_ties);
    const uint64_t goal = (uint64_t)((double)(u > 0.0f ? min(u, 0.99999994f) : 0.0f) * (double)total);
    room = own_room;
    for (int j = 0; j < warp; ++j) before += add(sh.mass[j], sh.ties[j]);
    uint64_t left = room;
    if (before <= goal && goal < before + add(sh.mass[warp], sh.ties[warp])) {
        uint64_t sum = before;
        for (uint32_t i = u0; i < u1; i += 32) {
            uint32_t k[S::kPer];
            uint64_t v[S::kPer], run = 0, same = 0;
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) k[e] = 0;
            if (i + lane < u1) source.keys(i + lane, k);
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) same += k[e] == cut && cut;
            uint64_t upto = same;      // ties in this lane and those before it
            if (__any_sync(kFull, same != 0))
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t up = __shfl_up_sync(kFull, upto, o);
                    if (lane >= o) upto += up;
                }
            uint64_t rank = upto - same;
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) {
                v[e] = weigh(k[e]);
                if (k[e] == cut && cut) v[e] = rank++ < left ? at_cut : 0;
                run += v[e];
            }
            uint64_t through = run;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t up = __shfl_up_sync(kFull, through, o);
                if (lane >= o) through += up;
            }
            const unsigned over = __ballot_sync(kFull, sum + through > goal);
            if (over) {
                if (lane == __ffs(over) - 1) {
                    uint64_t at = sum + through - run;
                    bool done = false;
#pragma unroll
                    for (int e = 0; e < S::kPer; ++e) {
                        at += v[e];
                        if (!done && at > goal) {
                            done = true;
                            *token = source.column_of(i + lane, e);
                            if (prob) *prob = (float)((double)v[e] / (double)total);
                        }
                    }
                }
                break;
            }
            sum += __shfl_sync(kFull, through, 31);
            left -= min(left, __shfl_sync(kFull, upto, 31));
        }
    }
}

// The filters on what `source` holds: all that can be drawn, and with kAll all of the row.  `count`: of keys; `all_weight`: of the row, when it
// is known (0: it is that of the source).
template <bool kAll, typename S, typename T>
__device__ void filter_and_draw(Team& team, const S& source, const Weights<T>& w, uint32_t kmin, uint64_t count, uint64_t all_weight, uint32_t k, float p, double least,
                                float u, uint32_t* token, float* prob) {
    uint32_t cut = 0;
    uint64_t ties = 0;
    if (k != 0 && k < count) {
        const Border at = find_border<kAll>(team, source, w, kmin, k, false);
        cut = at.key;
        ties = k - at.above;
    }
    if (p < 1.0f) {
        if (cut || all_weight == 0) {
            uint64_t s = 0, t = 0;
            for (uint32_t i = threadIdx.x; i < source.units; i += kThreads) {
                uint32_t key[S::kPer];
                source.keys(i, key);
#pragma unroll
                for (int e = 0; e < S::kPer; ++e) {
                    if (key[e] > cut) s += w(key[e]);
                    t += key[e] == cut && cut;
                }
            }
            s = team.block_sum(s);
            t = team.block_sum(t);
            if (kAll) {
                uint64_t s_all = 0, t_all = 0;
                team.exchange(s, t, [&](uint32_t, uint64_t a, uint64_t b) { s_all += a; t_all += b; });
                s = s_all;
                t = t_all;
            }
            all_weight = s + (cut ? min(t, ties) * w(cut) : 0);
        }
        const uint64_t target = max((uint64_t)1, (uint64_t)__double2ull_ru((double)max(p, 0.0f) * (double)all_weight));
        const Border at = find_border<kAll>(team, source, w, cut ? cut : kmin, target, true);
        const uint64_t each = w(at.key), need = each ? (target - at.above + each - 1) / each : 0;
        ties = at.key == cut ? min(ties, need) : need;
        cut = at.key;
    }
    draw<kAll>(team, source, w, cut, ties, least, u, token, prob);
}

template <typename T, bool kHeld>
__global__ void __launch_bounds__(kThreads, kHeld ? 4 : 2) sample_kernel(const SampleArgs a) {
    extern __shared__ uint4 dynamic[];      // the slice; later the first CTA's candidates
    __shared__ Shared sh;
    fg_grid_enter();
    cg::cluster_group cluster = cg::this_cluster();
    Team team{sh, cluster.num_blocks(), cluster.block_rank()};
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t r = blockIdx.x / team.ctas;
    using Slice = std::conditional_t<kHeld, HeldSlice<T>, FarSlice<T>>;
    constexpr int E = FgPack<T>::E;
    const uint32_t c0 = min(a.cols, team.cta * a.slice), n = min(a.cols - c0, a.slice);
    const T* const data = static_cast<const T*>(a.logits) + (uint64_t)r * a.cols + c0;
    Slice slice;
    if (tid < 64) sh.roots[tid] = kRoots[tid];
    if constexpr (kHeld) {
        const uint32_t o = (uint32_t)(reinterpret_cast<uintptr_t>(data) & 15u) / sizeof(T), words = n ? (o + n + E - 1) / E : 0;
        const uint32_t base = (uint32_t)__cvta_generic_to_shared(dynamic);
        const char* const first = reinterpret_cast<const char*>(data - o);
        for (uint32_t i = tid; i < words; i += kThreads)
            if (i * E >= o && (i + 1) * E <= o + n) fg_copy_async(base + 16 * i, first + 16ull * i);
        fg_copies_end();
        T* const held = reinterpret_cast<T*>(dynamic);
        if (words && tid < 2 * E) {      // words that reach over the ends
            const uint32_t i = tid < E ? 0 : words - 1, at = i * E + (tid & (E - 1));
            if (!(i * E >= o && (i + 1) * E <= o + n)) held[at] = at >= o && at < o + n ? data[at - o] : fg_narrow<T>(-INFINITY);
        }
        fg_copies_wait<0>();
        __syncthreads();
        slice = Slice{dynamic, words, c0 - o};
    } else {
        __syncthreads();
        slice = Slice{data, n, c0};
    }
    uint32_t* const token = a.token + r;
    float* const prob = a.prob ? a.prob + r : nullptr;

    // The largest logit; each thread keeps its own.
    float mine = -INFINITY;
    for (uint32_t u = tid; u < slice.units; u += kThreads) {
        float x[Slice::kPer];
        slice.values(u, x);
#pragma unroll
        for (int e = 0; e < Slice::kPer; ++e) mine = fmaxf(mine, x[e]);
    }
    const uint32_t largest = team.block_max(key_of<T>(mine));
    uint32_t kmax = 0;
    team.exchange(largest, 0, [&](uint32_t, uint64_t key, uint64_t) { kmax = max(kmax, (uint32_t)key); });
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    if (kmax == 0) {
        if (team.cta == 0 && tid == 0) { *token = FG_NO_TOKEN; if (prob) *prob = 0.0f; }
        cluster.sync();      // (the others' slots are being read)
        return;
    }
    if (!(temperature > 0.0f)) {      // the first maximum
        uint32_t first = 0;
        if (largest == kmax && key_of<T>(mine) == kmax)
            for (uint32_t u = tid; u < slice.units; u += kThreads) {
                uint32_t k[Slice::kPer];
                slice.keys(u, k);
#pragma unroll
                for (int e = Slice::kPer - 1; e >= 0; --e)
                    if (k[e] == kmax) first = max(first, ~slice.column_of(u, e));
            }
        first = team.block_max(first);
        team.exchange(first, 0, [&](uint32_t, uint64_t inverse, uint64_t) { first = max(first, (uint32_t)inverse); });
        if (team.cta == 0 && tid == 0) { *token = ~first; if (prob) *prob = 1.0f; }
        cluster.sync();
        return;
    }
    const float top = logit_of<T>(kmax);
    const Weights<T> w{sh.roots, (double)top, 1.4426950408889634 / (double)temperature, kmax};
    const float rate = (float)w.c, u = a.u[r], p = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
    const uint32_t k = a.top_k ? a.top_k[r] : 0;
    const double least = mp > 0.0f ? (double)min(mp, 1.0f) * kOne : 0.0;
    const bool by_k = k != 0 && k < a.cols, by_p = p < 1.0f;
    if (!by_k && !by_p) {
        draw<true>(team, slice, w, 0, 0, least, u, token, prob);
        cluster.sync();
        return;
    }

    // A bound below the border: `bound` bins of a 32nd of an octave below the largest.
    auto bin_of = [&](float x) {      // grows as x falls
        const float d = (top - x) * rate;
        return d < (float)(kBins / 32) ? (uint32_t)(d * 32.0f) : (uint32_t)kBins - 1;
    };
    uint32_t bound = kBins - 1;
    uint64_t all_weight = 0;
    const bool ordinary = top < INFINITY && rate < 1e30f;      // else bins say nothing
    if (ordinary && by_k) {
        // k threads with a value of a bin or above it say that the k-th largest is not below it; so do k / ctas threads in each CTA.
        const uint32_t bin = key_of<T>(mine) ? bin_of(mine) : kBins;
        auto reached = [&](uint32_t want) {
            uint32_t b = kBins - 1;
            if (want <= kThreads)
                for (uint32_t lo = 0, hi = kBins - 1; lo <= hi;) {      // 11 steps
                    const uint32_t mid = (lo + hi) / 2;
                    if ((uint32_t)__syncthreads_count(bin <= mid) >= want) {
                        b = mid;
                        if (mid == 0) break;
                        hi = mid - 1;
                    } else lo = mid + 1;
                }
            return b;
        };
        const uint32_t share = reached((k + team.ctas - 1) / team.ctas), whole = team.ctas > 1 ? reached(k) : share;
        uint32_t worst = 0, best = kBins - 1;
        team.exchange(share, whole, [&](uint32_t, uint64_t x, uint64_t y) { worst = max(worst, (uint32_t)x); best = min(best, (uint32_t)y); });
        bound = min(worst, best);
    } else if (ordinary) {
        // The weight of the row, exactly, and how many of its tokens lie in each bin: their weight is at least that of the bin's end.
        for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
        __syncthreads();
        uint64_t s = 0;
        for (uint32_t i = tid; i < slice.units; i += kThreads) {
            float x[Slice::kPer];
            slice.values(i, x);
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e) {
                const uint32_t b = bin_of(x[e]);
                if (b < kBins - 1) {
                    s += w(key_of<T>(x[e]));
                    atomicAdd(&sh.bins[b], 1u);
                }
            }
        }
        s = team.block_sum(s);
        team.exchange(s, 0, [&](uint32_t, uint64_t part, uint64_t) { all_weight += part; });
        // (the exchange has all CTAs' bins complete)  A thread takes eight bins, then a prefix over the threads.
        float sum = 0.0f, part[kBins / kThreads];
#pragma unroll
        for (int j = 0; j < kBins / kThreads; ++j) {
            const uint32_t b = tid * (kBins / kThreads) + j;
            uint32_t in_bin = 0;
            for (uint32_t c = 0; c < team.ctas; ++c) in_bin += cluster.map_shared_rank(sh.bins, c)[b];
            part[j] = sum += (float)in_bin * exp2f(-(float)(b + 1) / 32.0f);
        }
        float run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float up = __shfl_up_sync(kFull, run, o);
            if (lane >= o) run += up;
        }
        float* const sums = reinterpret_cast<float*>(sh.red);
        if (lane == 31) sums[warp] = run;
        __syncthreads();
        float before = run - sum;
        for (int j = 0; j < warp; ++j) before += sums[j];
        const float goal = (float)((double)max(p, 0.0f) * (double)all_weight / kOne) * 1.001f;      // bins and sums in f32: a thousandth covers what they lose
        uint32_t b = kBins - 1;
#pragma unroll
        for (int j = kBins / kThreads - 1; j >= 0; --j)
            if (before + part[j] >= goal) b = tid * (kBins / kThreads) + j;
        bound = kBins - 1 - team.block_max(kBins - 1 - b);
    }

    // What lies above it, in order: count, then places.
    const uint32_t len = ((slice.units + kWarps - 1) / kWarps + 31) / 32 * 32;
    const uint32_t u0 = min(slice.units, warp * len), u1 = min(slice.units, u0 + len);
    uint32_t candidates = 0;
    auto chosen = [&](float x) { return x > -INFINITY && (!ordinary || bin_of(x) <= bound); };
    for (uint32_t i = u0 + lane; i < u1; i += 32) {
        float x[Slice::kPer];
        slice.values(i, x);
#pragma unroll
        for (int e = 0; e < Slice::kPer; ++e) candidates += chosen(x[e]);
    }
    candidates = __reduce_add_sync(kFull, candidates);
    __syncthreads();
    if (lane == 0) sh.red[warp] = candidates;
    __syncthreads();
    uint32_t place = 0, own = 0;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) {
        if (j == warp) place = own;
        own += (uint32_t)sh.red[j];
    }
    if (own <= kLocal && candidates)
        for (uint32_t i = u0; i < u1; i += 32) {
            float x[Slice::kPer];
            uint32_t count = 0;
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e) x[e] = -INFINITY;
            if (i + lane < u1) slice.values(i + lane, x);
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e) count += chosen(x[e]);
            if (!__any_sync(kFull, count != 0)) continue;
            uint32_t upto = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(kFull, upto, o);
                if (lane >= o) upto += up;
            }
            uint32_t at = place + upto - count;
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e)
                if (chosen(x[e])) sh.local[at++] = make_uint2(key_of<T>(x[e]), slice.column_of(i + lane, e));
            place += __shfl_sync(kFull, upto, 31);
        }
    bool fits = true;
    uint32_t offset = 0, listed = 0;
    team.exchange(own, 0, [&](uint32_t c, uint64_t count, uint64_t) {
        if (c == team.cta) offset = listed;
        listed += (uint32_t)min(count, (uint64_t)kGathered + 1);
        fits = fits && count <= kLocal;
    });
    if (fits && listed <= kGathered) {
        uint2* const list = reinterpret_cast<uint2*>(dynamic);      // nobody reads a slice any more
        uint2* const to = cluster.map_shared_rank(list, 0) + offset;
        for (uint32_t i = tid; i < own; i += kThreads) to[i] = sh.local[i];
        cluster.sync();
        if (team.cta) return;
        const List source{list, listed};
        uint32_t smallest = 0;
        for (uint32_t i = tid; i < listed; i += kThreads) smallest = max(smallest, ~list[i].x);
        const uint32_t kmin = ~team.block_max(smallest);
        filter_and_draw<false>(team, source, w, kmin, listed, all_weight, by_k ? k : 0, p, least, u, token, prob);
        return;
    }
    uint32_t smallest = 0;
    uint64_t count = 0;
    for (uint32_t i = tid; i < slice.units; i += kThreads) {
        uint32_t key[Slice::kPer];
        slice.keys(i, key);
#pragma unroll
        for (int e = 0; e < Slice::kPer; ++e)
            if (key[e]) { smallest = max(smallest, ~key[e]); ++count; }
    }
    smallest = team.block_max(smallest);
    count = team.block_sum(count);
    uint64_t count_all = 0;
    uint32_t inverse = 0;
    team.exchange(smallest, count, [&](uint32_t, uint64_t x, uint64_t y) { inverse = max(inverse, (uint32_t)x); count_all += y; });
    filter_and_draw<true>(team, slice, w, ~inverse, count_all, 0, by_k ? k : 0, p, least, u, token, prob);
    cluster.sync();
}

template <typename T, bool kHeld>
int32_t launch_sample(fg_ctx* ctx, const SampleArgs& a, unsigned ctas, size_t bytes) {
    if (bytes > 16 * 1024) FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(sample_kernel<T, kHeld>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    fg_launch_cluster(ctx, sample_kernel<T, kHeld>, a.rows * ctas, kThreads, bytes, ctas, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T>
int32_t sample(fg_ctx* ctx, SampleArgs a) {
    // Slices of up to 32 KB, so that an SM works on four at a time and loads one while it computes on another; few rows are spread further.
    const uint64_t row = (uint64_t)a.cols * sizeof(T);
    unsigned ctas = 1;
    while (ctas < kMaxCtas && (row > 32768ull * ctas || (a.cols > 2048u * ctas && (uint64_t)a.rows * ctas < (uint64_t)ctx->sm_count))) ctas *= 2;
    a.slice = ((a.cols + ctas - 1) / ctas + 7) / 8 * 8;
    const size_t held = ((size_t)a.slice * sizeof(T) + 31) / 16 * 16, list = sizeof(uint2) * (a.cols < kGathered ? a.cols : kGathered);
    FG_REQUIRE(ctx, (uint64_t)a.rows * ctas < (1ull << 31), "fg_sample: too many rows");
    if (held <= 180 * 1024) return launch_sample<T, true>(ctx, a, ctas, held < list ? list : held);
    return launch_sample<T, false>(ctx, a, ctas, list);
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
