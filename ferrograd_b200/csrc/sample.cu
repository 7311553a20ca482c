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

#include <atomic>

#include "rows.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxCtas = 8;
constexpr int kSteps = 2048;                  // 64ths of an octave of weight that a bound is looked for in
constexpr int kBins = 512;                    // 16ths of an octave that a row's weight is added up in
constexpr uint32_t kLocal = 1024, kGathered = 4096;      // candidates of a CTA, of a row
constexpr unsigned kFull = 0xffffffffu;
constexpr double kOne = 4398046511104.0;      // 2^42
constexpr size_t kHeldBytes = 180 * 1024;     // of a slice in shared memory

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

// 2^(i / 256)
__device__ const double kRoots[256] = {
    1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175, 1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738,
    1.0218971486541166, 1.0246677928971357, 1.0274459491187637, 1.030231637686041, 1.0330248790212284, 1.0358256936019572, 1.0386341019613787, 1.041450124688316,
    1.0442737824274138, 1.0471050958792898, 1.0499440858006872, 1.0527907730046264, 1.0556451783605572, 1.0585073227945128, 1.061377227289262, 1.0642549128844645,
    1.0671404006768237, 1.0700337118202419, 1.0729348675259756, 1.075843889062791, 1.0787607977571199, 1.0816856149932152, 1.0846183622133092, 1.0875590609177697,
    1.0905077326652577, 1.0934643990728858, 1.0964290818163769, 1.099401802630222, 1.102382583307841, 1.1053714457017412, 1.1083684117236787, 1.1113735033448175,
    1.1143867425958924, 1.1174081515673693, 1.1204377524096067, 1.12347556733302, 1.1265216186082418, 1.129575928566288, 1.1326385195987192, 1.1357094141578055,
    1.1387886347566916, 1.1418762039695616, 1.1449721444318042, 1.148076478840179, 1.1511892299529827, 1.154310420590216, 1.1574400736337511, 1.1605782120274988,
    1.1637248587775775, 1.1668800369524817, 1.1700437696832502, 1.1732160801636373, 1.1763969916502812, 1.1795865274628758, 1.182784710984341, 1.1859915656609938,
    1.189207115002721, 1.1924313825831512, 1.1956643920398273, 1.1989061670743806, 1.202156731452703, 1.2054161090051239, 1.2086843236265816, 1.2119613992768012,
    1.215247359980469, 1.2185422298274085, 1.2218460329727576, 1.2251587936371455, 1.22848053610687, 1.2318112847340759, 1.2351510639369334, 1.2384998981998165,
    1.241857812073484, 1.245224830175258, 1.2486009771892048, 1.2519862778663162, 1.255380757024691, 1.2587844395497165, 1.2621973503942507, 1.2656195145788063,
    1.2690509571917332, 1.2724917033894028, 1.275941778396392, 1.2794012075056693, 1.2828700160787783, 1.2863482295460256, 1.2898358734066657, 1.2933329732290895,
    1.2968395546510096, 1.3003556433796506, 1.3038812651919358, 1.3074164459346773, 1.3109612115247644, 1.3145155879493546, 1.318079601266064, 1.3216532776031575,
    1.3252366431597413, 1.3288297242059544, 1.3324325470831615, 1.3360451382041458, 1.339667524053303, 1.3432997311868353, 1.3469417862329458, 1.3505937158920345,
    1.3542555469368927, 1.3579273062129011, 1.3616090206382248, 1.365300717204012, 1.3690024229745905, 1.3727141650876684, 1.3764359707545302, 1.380167867260238,
    1.383909881963832, 1.387662042298529, 1.3914243757719262, 1.3951969099662003, 1.3989796725383112, 1.4027726912202048, 1.4065759938190154, 1.4103896082172707,
    1.4142135623730951, 1.4180478843204152, 1.4218926021691656, 1.4257477441054942, 1.42961333839197, 1.433489413367789, 1.4373759974489824, 1.4412731191286257,
    1.4451808069770467, 1.449099089642035, 1.4530279958490526, 1.4569675544014438, 1.460917794180647, 1.4648787441464057, 1.4688504333369818, 1.4728328908693675,
    1.4768261459394993, 1.4808302278224719, 1.4848451658727524, 1.488870989524397, 1.4929077282912648, 1.4969554117672355, 1.5010140696264256, 1.5050837316234065,
    1.5091644275934228, 1.5132561874526098, 1.5173590411982147, 1.5214730189088146, 1.5255981507445384, 1.529734466947287, 1.533881997840956, 1.5380407738316568,
    1.5422108254079407, 1.5463921831410214, 1.550584877685, 1.5547889397770887, 1.559004400237837, 1.5632312899713576, 1.567469639965553, 1.5717194812923414,
    1.5759808451078865, 1.5802537626528246, 1.5845382652524937, 1.588834384317164, 1.593142151342267, 1.597461597908627, 1.6017927556826934, 1.606135656416771,
    1.6104903319492543, 1.6148568142048607, 1.6192351351948637, 1.6236253270173289, 1.6280274218573478, 1.632441451987275, 1.6368674497669644, 1.6413054476440063,
    1.645755478153965, 1.6502175739206177, 1.6546917676561943, 1.6591780921616162, 1.6636765803267364, 1.6681872651305825, 1.6727101796415966, 1.6772453570178785,
    1.681792830507429, 1.6863526334483934, 1.6909247992693053, 1.6955093614893326, 1.7001063537185235, 1.7047158096580513, 1.709337763100463, 1.713972247929926,
    1.718619298122478, 1.723278947746274, 1.7279512309618377, 1.732636182022311, 1.7373338352737062, 1.7420442251551564, 1.746767386199169, 1.7515033530318782,
    1.7562521603732995, 1.761013843037584, 1.7657884359332727, 1.7705759740635547, 1.7753764925265212, 1.7801900265154245, 1.785016611318935, 1.789856282321401,
    1.7947090750031072, 1.7995750249405351, 1.804454167806624, 1.809346539371032, 1.8142521755003989, 1.8191711121586085, 1.8241033854070534, 1.8290490314048973,
    1.8340080864093424, 1.8389805867758937, 1.843966568958626, 1.8489660695104508, 1.8539791250833855, 1.8590057724288205, 1.864046048397789, 1.8690999899412386,
    1.8741676341103, 1.8792490180565602, 1.8843441790323345, 1.8894531543909392, 1.8945759815869656, 1.8997126981765553, 1.9048633418176741, 1.9100279502703899,
    1.9152065613971474, 1.9203992131630474, 1.925605943636125, 1.930826790987627, 1.9360617934922943, 1.9413109895286405, 1.9465744175792332, 1.9518521162309783,
    1.9571441241754002, 1.9624504802089273, 1.9677712232331759, 1.9731063922552343, 1.978456026387951, 1.9838201648502194, 1.9891988469672663, 1.9945921121709402};

// round(2^42 exp(t)) with t = (x - m) / T: exp(t) = 2^(n / 256) exp(r) for the n that leaves |r| <= ln(2) / 512, and four terms of the series
// of exp(r), off by 2^-42.7 at most (1/6 is cut to 20 bits, which is 2^-52 of the result, so that it fits an instruction).  Of the
// 44 instructions that a logit of a row with a temperature alone takes, ten are 64-bit ones; a table of 64 and six terms needs two more.
template <typename T>
struct Weights {
    const double* roots;
    double m, c, mc;          // the largest logit; 1 / T; their product
    float top, rate, bottom;  // in f32, and log2(e) / T; 44 octaves below the largest: nothing that counts is lower
    uint32_t kmax;
    bool ordinary;            // nothing overflows in f32, and mc is good to 2^-33: the short cuts hold
    // 2^42 w, not rounded, for a w of 2^-44 or more
    __device__ __forceinline__ double series(float x) const {
        constexpr double kMagic = 6755399441055744.0;      // 1.5 * 2^52: a sum with it has its whole part in the low word
        const double t = __fma_rn((double)x, c, -mc);      // (mc's rounding scales all weights alike)
        const double y = __fma_rn(t, __hiloint2double(0x40771547, 0), kMagic);      // 256 / ln(2)
        const int j = __double2loint(y);
        const double r = __fma_rn(y - kMagic, -0.69314718055994530942 / 256, t);
        double p = __fma_rn(r, __hiloint2double(0x3fc55555, 0), 0.5);
        p = __fma_rn(r, p, 1.0);
        p = __fma_rn(r, p, 1.0);
        const double root = roots[j & 255];      // 2^42 times it, less what j's low bits add to the exponent here
        return __hiloint2double(__double2hiint(root) + (j << 12), __double2loint(root)) * p;
    }
    // The same for any x of an ordinary row, without a branch: what lies below `bottom`, -inf and NaN are taken for it, a quarter of 2^-42.
    __device__ __forceinline__ double usual(float x) const { return series(fmaxf(x, bottom)); }
    // Its rounded value as the low bits of a sum with 2^52; kBias too much.
    static constexpr uint64_t kBias = 0x4330000000000000ull;
    __device__ __forceinline__ uint64_t biased(float x) const { return (uint64_t)__double_as_longlong(usual(x) + 4503599627370496.0); }
    __device__ __forceinline__ double scaled(float x) const {
        if (ordinary) return usual(x);
        if (x == top) return kOne;
        const double t = ((double)x - m) * c;
        return x > -INFINITY && t > -30.0 ? exp(t) * kOne : 0.0;      // 2^-43
    }
    static __device__ __forceinline__ uint64_t whole(double v) { return (uint64_t)__double_as_longlong(v + 4503599627370496.0) & 0xfffffffffffffull; }
    __device__ __forceinline__ uint64_t operator()(float x) const { return whole(scaled(x)); }
    __device__ __forceinline__ uint64_t of_key(uint32_t key) const { return whole(scaled(logit_of<T>(key))); }
    // How far x lies below the largest, in 64ths of an octave of weight; NaN or infinite for what is never drawn.  Grows as x falls.
    __device__ __forceinline__ float below(float x) const { return (top - x) * (rate * 64.0f); }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

struct Border { uint32_t key; uint64_t above, at; };      // the sum over larger keys, and over this one

struct Shared {
    double roots[256];
    alignas(8) uint32_t hist[2][3][256];  // parts of sums
    uint64_t slots[2][2];                 // what a CTA tells the others
    uint64_t red[kWarps], red2[kWarps];
    alignas(16) uint32_t bins[kBins];
    uint2 local[kLocal];                  // (key, column)
    Border border;
    uint32_t next_lo, next_hi;
};

// What the functions below go over: units of kPer logits, in the order of the columns; a thread owns `stretch` units in a row.
template <typename T>
struct HeldSlice {      // a slice in shared memory, by 16-byte words; masked where a word reaches over the slice's ends
    static constexpr int kPer = FgPack<T>::E;
    static constexpr bool kLong = false;  // 180 KB: fewer than 2^17 elements
    const uint4* words;
    uint32_t units, column;               // of the first word's first element (it may lie before the slice)
    __device__ __forceinline__ void values(uint32_t u, float (&x)[kPer]) const { FgPack<T>::widen(words[u], x); }
    __device__ __forceinline__ float value(uint32_t i) const { return fg_widen(reinterpret_cast<const T*>(words)[i]); }
    __device__ __forceinline__ uint32_t column_of(uint32_t i) const { return column + i; }
    __device__ __forceinline__ uint32_t stretch() const { return ((units + kThreads - 1) / kThreads) | 1; }      // odd: no two lanes on one bank
};
template <typename T>
struct FarSlice {       // a slice that shared memory does not hold
    static constexpr int kPer = 1;
    static constexpr bool kLong = true;
    const T* data;
    uint32_t units, column;
    __device__ __forceinline__ void values(uint32_t u, float (&x)[1]) const { x[0] = fg_widen(data[u]); }
    __device__ __forceinline__ float value(uint32_t i) const { return fg_widen(data[i]); }
    __device__ __forceinline__ uint32_t column_of(uint32_t i) const { return column + i; }
    __device__ __forceinline__ uint32_t stretch() const { return (units + kThreads - 1) / kThreads; }
};
template <typename T>
struct List {           // entries (key, column)
    static constexpr int kPer = 1;
    static constexpr bool kLong = false;
    const uint2* entries;
    uint32_t units;
    __device__ __forceinline__ void values(uint32_t u, float (&x)[1]) const { x[0] = logit_of<T>(entries[u].x); }
    __device__ __forceinline__ float value(uint32_t i) const { return logit_of<T>(entries[i].x); }
    __device__ __forceinline__ uint32_t column_of(uint32_t i) const { return entries[i].y; }
    __device__ __forceinline__ uint32_t stretch() const { return ((units + kThreads - 1) / kThreads) | 1; }
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
    // Sums of a and b over the threads before this one; the block's in all_a and all_b.
    __device__ __forceinline__ void prefix(uint64_t& a, uint64_t& b, uint64_t& all_a, uint64_t& all_b) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        uint64_t x = a, y = b;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = __shfl_up_sync(kFull, x, o), up2 = __shfl_up_sync(kFull, y, o);
            if (lane >= o) { x += up; y += up2; }
        }
        __syncthreads();
        if (lane == 31) { sh.red[warp] = x; sh.red2[warp] = y; }
        __syncthreads();
        a = x - a;
        b = y - b;
        all_a = all_b = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) { a += all_a; b += all_b; }
            all_a += sh.red[w];
            all_b += sh.red2[w];
        }
    }
    // Every CTA's pair, to every thread: f(cta, a, b) in the order of the CTAs.
    template <typename F>
    __device__ __forceinline__ void exchange(uint64_t a, uint64_t b, F f) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) { sh.slots[turn][0] = a; sh.slots[turn][1] = b; }
        cluster.sync();
        uint64_t x = 0, y = 0;
        const uint32_t lane = threadIdx.x & 31;
        if (lane < ctas) {
            const uint64_t* const p = cluster.map_shared_rank(&sh.slots[turn][0], lane);
            x = p[0];
            y = p[1];
        }
        for (uint32_t c = 0; c < ctas; ++c) f(c, __shfl_sync(kFull, x, c), __shfl_sync(kFull, y, c));
        turn ^= 1;
    }
};

// The border at which `above` and the sum over the keys from hi down to lo (counts, or weights) reach `target`; all of them together do.
template <bool kAll, typename S, typename T>
__device__ Border find_border(Team& team, const S& source, const Weights<T>& w, uint32_t lo, uint32_t hi, uint64_t above, uint64_t target, bool by_weight) {
    Shared& sh = team.sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Border at{};
    target = max(target, above + 1);               // one thread finds the border in any case: should `above` be there already, among the highest keys
    for (int round = 0; round < 5; ++round) {      // 32 bits of range, eight less after each
        const int bits = 32 - __clz(hi - lo), shift = bits > 8 ? bits - 8 : 0;
        uint32_t (*const hist)[256] = sh.hist[team.round ^= 1];
        hist[0][tid] = hist[1][tid] = hist[2][tid] = 0;
        __syncthreads();
        for (uint32_t u = tid; u < source.units; u += kThreads) {
            float x[S::kPer];
            source.values(u, x);
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) {
                const uint32_t k = key_of<T>(x[e]);
                if (k >= lo && k <= hi) {
                    // A 64-bit addition in shared memory is a loop (a top-k of 3000 of 256 x 128003 took 1308 us with it, 182 with 32 bits), so a weight
                    // is added in parts of 15, 15 and 13 bits, which 2^17 elements do not carry over.
                    const uint32_t at = (k - lo) >> shift;
                    if (!by_weight) {
                        atomicAdd(&hist[0][at], 1u);
                    } else if (const uint64_t v = w(x[e])) {
                        if constexpr (S::kLong) atomicAdd(reinterpret_cast<unsigned long long*>(hist) + at, (unsigned long long)v);      // over the first two planes
                        else {
                            if (const uint32_t part = (uint32_t)v & 0x7fffu) atomicAdd(&hist[0][at], part);
                            if (const uint32_t part = (uint32_t)(v >> 15) & 0x7fffu) atomicAdd(&hist[1][at], part);
                            if (const uint32_t part = (uint32_t)(v >> 30)) atomicAdd(&hist[2][at], part);
                        }
                    }
                }
            }
        }
        auto sum_of = [&](const uint32_t* planes) {
            if (!by_weight) return (uint64_t)planes[tid];
            if constexpr (S::kLong) return reinterpret_cast<const uint64_t*>(planes)[tid];
            else return planes[tid] + ((uint64_t)planes[256 + tid] << 15) + ((uint64_t)planes[512 + tid] << 30);
        };
        uint64_t v = 0;
        if (kAll) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
#pragma unroll
            for (uint32_t c = 0; c < kMaxCtas; ++c) v += c < team.ctas ? sum_of(cluster.map_shared_rank(&hist[0][0], c)) : 0;
        } else {
            __syncthreads();
            v = sum_of(&hist[0][0]);
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
// The nucleus ends at `at`: as many ties as it takes to reach the target, of at most `most`.
template <typename T>
__device__ __forceinline__ uint64_t ties_to_reach(const Weights<T>& w, const Border& at, uint64_t target, uint64_t most) {
    const uint64_t each = w.of_key(at.key);
    return each && at.above < target ? min(most, (target - at.above + each - 1) / each) : 0;
}
// f times n, f from [0, 1), rounded down or up from the exact product: n has up to 63 bits, and in 64-bit floating point a border that the product
// hits exactly moves by a token.  f goes in parts of 2^-64, which is all of it from 2^-40 on; below that f n is less than 2^23, the largest weight 2^42.
template <bool kUp>
__device__ __forceinline__ uint64_t part_of(float f, uint64_t n) {
    const uint64_t parts = __float2ull_rz(f * 18446744073709551616.0f);
    return __umul64hi(parts, n) + (kUp && parts * n != 0);
}
__device__ __forceinline__ uint64_t nucleus(float p, uint64_t weight) { return max((uint64_t)1, part_of<true>(p > 0.0f ? p : 0.0f, weight)); }

// What is kept: keys above `cut` and the first `ties` of those at it, of weight `least` (in parts of 2^42) or more.
struct Kept { uint32_t cut; uint64_t ties; double least; };

// The first at which the running sum over what is kept exceeds u times the total.  mass and same: the kept weight above the cut, and the
// keys at it, of the thread's stretch.
template <bool kAll, typename S, typename T>
__device__ void locate(Team& team, const S& source, const Weights<T>& w, const Kept& keep, uint64_t mass, uint64_t same, float u, uint32_t* token, float* prob) {
    const int lane = threadIdx.x & 31;
    const double cut_scaled = keep.cut ? w.scaled(logit_of<T>(keep.cut)) : 0.0;
    const uint64_t at_cut = cut_scaled >= keep.least ? w.whole(cut_scaled) : 0;
    uint64_t m = mass, t = same, all_m, all_t;
    team.prefix(m, t, all_m, all_t);
    if (kAll) {
        uint64_t sum_m = 0, sum_t = 0, before_m = 0, before_t = 0;
        team.exchange(all_m, all_t, [&](uint32_t c, uint64_t x, uint64_t y) {
            if (c == team.cta) { before_m = sum_m; before_t = sum_t; }
            sum_m += x;
            sum_t += y;
        });
        m += before_m; t += before_t;
        all_m = sum_m; all_t = sum_t;
        cg::this_cluster().barrier_arrive();      // nobody reads another's memory from here on
    }
    auto upto = [&](uint64_t x, uint64_t y) { return x + min(keep.ties, y) * at_cut; };
    const uint64_t total = upto(all_m, all_t), goal = part_of<false>(u > 0.0f ? min(u, 0.99999994f) : 0.0f, total), before = upto(m, t);
    const unsigned holds = __ballot_sync(kFull, before <= goal && goal < upto(m + mass, t + same));
    if (holds) {      // the warp goes over that thread's stretch once more
        const int from = __ffs(holds) - 1;
        const uint32_t stretch = source.stretch(), u0 = (threadIdx.x - lane + from) * stretch;
        const uint32_t i1 = min(source.units, u0 + stretch) * S::kPer;
        uint64_t sum = __shfl_sync(kFull, before, from), ties = __shfl_sync(kFull, t, from);
        for (uint32_t i = u0 * S::kPer; i < i1; i += 32) {
            const float x = i + lane < i1 ? source.value(i + lane) : -INFINITY;
            const uint32_t key = key_of<T>(x);
            const unsigned tied = __ballot_sync(kFull, key == keep.cut && key);
            uint64_t v = 0;
            if (key > keep.cut) {
                const double s = w.scaled(x);
                v = s >= keep.least ? w.whole(s) : 0;
            } else if (key && key == keep.cut && ties + __popc(tied & ((1u << lane) - 1)) < keep.ties) v = at_cut;
            uint64_t run = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t up = __shfl_up_sync(kFull, run, o);
                if (lane >= o) run += up;
            }
            const unsigned over = __ballot_sync(kFull, sum + run > goal);
            if (over) {
                if (lane == __ffs(over) - 1) {
                    *token = source.column_of(i + lane);
                    if (prob) *prob = (float)((double)v / (double)total);
                }
                break;
            }
            sum += __shfl_sync(kFull, run, 31);
            ties += __popc(tied);
        }
    }
    if (kAll) cg::this_cluster().barrier_wait();
}
template <bool kAll, typename S, typename T>
__device__ void draw(Team& team, const S& source, const Weights<T>& w, const Kept& keep, float u, uint32_t* token, float* prob) {
    const uint32_t stretch = source.stretch(), u0 = min(source.units, threadIdx.x * stretch), u1 = min(source.units, u0 + stretch);
    uint64_t mass = 0, same = 0;
    if (keep.cut == 0 && keep.least == 0.0 && w.ordinary) {      // all of it
        for (uint32_t i = u0; i < u1; ++i) {
            float x[S::kPer];
            source.values(i, x);
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) mass += w.biased(x[e]);
        }
        mass -= (u1 - u0) * (uint64_t)S::kPer * w.kBias;
    } else
        for (uint32_t i = u0; i < u1; ++i) {
            float x[S::kPer];
            source.values(i, x);
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) {
                const uint32_t key = key_of<T>(x[e]);
                if (key > keep.cut) {
                    const double s = w.scaled(x[e]);
                    if (s >= keep.least) mass += w.whole(s);
                }
                same += key == keep.cut && key;
            }
        }
    locate<kAll>(team, source, w, keep, mass, same, u, token, prob);
}

// The filters on what `source` holds: all that can be drawn, and with kAll all of the row.  `count`: of keys.
template <bool kAll, typename S, typename T>
__device__ void filter_and_draw(Team& team, const S& source, const Weights<T>& w, uint32_t kmin, uint64_t count, uint32_t k, float p, double least, float u, uint32_t* token,
                                float* prob) {
    Kept keep{0, 0, least};
    if (k != 0 && k < count) {
        const Border at = find_border<kAll>(team, source, w, kmin, w.kmax, 0, k, false);
        keep.cut = at.key;
        keep.ties = k - at.above;
    }
    if (p < 1.0f) {
        uint64_t s = 0, t = 0;
        for (uint32_t i = threadIdx.x; i < source.units; i += kThreads) {
            float x[S::kPer];
            source.values(i, x);
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) {
                const uint32_t key = key_of<T>(x[e]);
                if (key > keep.cut) s += w(x[e]);
                t += key == keep.cut && key;
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
        const uint64_t target = nucleus(p, s + (keep.cut ? min(t, keep.ties) * w.of_key(keep.cut) : 0));
        const Border at = find_border<kAll>(team, source, w, keep.cut ? keep.cut : kmin, w.kmax, 0, target, true);
        keep.ties = ties_to_reach(w, at, target, at.key == keep.cut ? keep.ties : ~0ull);
        keep.cut = at.key;
    }
    draw<kAll>(team, source, w, keep, u, token, prob);
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
    sh.roots[tid] = __hiloint2double(__double2hiint(kRoots[tid]) + (42 << 20) - (tid << 12), __double2loint(kRoots[tid]));
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
                float x[Slice::kPer];
                slice.values(u, x);
#pragma unroll
                for (int e = 0; e < Slice::kPer; ++e)
                    if (key_of<T>(x[e]) == kmax) first = max(first, ~slice.column_of(u * Slice::kPer + e));
            }
        first = team.block_max(first);
        team.exchange(first, 0, [&](uint32_t, uint64_t inverse, uint64_t) { first = max(first, (uint32_t)inverse); });
        if (team.cta == 0 && tid == 0) { *token = ~first; if (prob) *prob = 1.0f; }
        cluster.sync();
        return;
    }
    const float top = logit_of<T>(kmax);
    const double per_unit = 1.0 / (double)temperature;
    const Weights<T> w{sh.roots, (double)top, per_unit, (double)top * per_unit, top, (float)(1.4426950408889634 * per_unit), (float)((double)top - 30.5 / per_unit), kmax,
                       fabs((double)top * per_unit) < 1e6 && per_unit < 1e30 && per_unit > 1e-30};
    const float u = a.u[r], p = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
    const uint32_t k = a.top_k && a.top_k[r] < a.cols ? a.top_k[r] : 0;
    // The largest logit itself comes out up to |mc| 2^-53 and a rounding off 2^42, which must not put it below a min_p of 1; |mc| 2^-52 lets in no other,
    // whose distance is 2^-24 of it at least.  (Its own computed weight as the bound takes 38.8 us where this takes 38.3: 512 x 32000 f32.)
    const double least = mp > 0.0f ? (double)min(mp, 1.0f) * (w.ordinary ? kOne - fabs(w.mc) * 0x1p-10 : kOne) : 0.0;
    if (!k && !(p < 1.0f)) {
        draw<true>(team, slice, w, Kept{0, 0, least}, u, token, prob);
        return;
    }
    const uint32_t stretch = slice.stretch(), u0 = min(slice.units, tid * stretch), u1 = min(slice.units, u0 + stretch);

    if (w.ordinary && k) {
        // k threads with a value of a bin or above it say that the k-th largest is not below it; so do k / ctas threads in each CTA.
        const float own_below = w.below(mine);
        const uint32_t own_bin = own_below < (float)kSteps ? (uint32_t)own_below : kSteps;
        auto reached = [&](uint32_t want) {
            uint32_t b = kSteps;      // not by any bin
            if (want <= kThreads)
                for (uint32_t lo = 0, hi = kSteps - 1; lo <= hi;) {      // 11 steps
                    const uint32_t mid = (lo + hi) / 2;
                    if ((uint32_t)__syncthreads_count(own_bin <= mid) >= want) {
                        b = mid;
                        if (mid == 0) break;
                        hi = mid - 1;
                    } else lo = mid + 1;
                }
            return b;
        };
        const uint32_t share = reached((k + team.ctas - 1) / team.ctas), whole = team.ctas > 1 ? reached(k) : share;
        uint32_t worst = 0, best = kSteps;
        team.exchange(share, whole, [&](uint32_t, uint64_t x, uint64_t y) { worst = max(worst, (uint32_t)x); best = min(best, (uint32_t)y); });
        const uint32_t bound = min(worst, best);
        const float limit = bound < (uint32_t)kSteps ? (float)(bound + 1) : INFINITY;
        // What is not below it goes to the first CTA, in order: count, then places.
        auto candidate = [&](float x) { return w.below(x) < limit; };
        uint64_t count = 0, none = 0, own, unused, where = 0;      // where: the units with candidates, of a stretch of up to 64
        for (uint32_t i = u0; i < u1; ++i) {
            float x[Slice::kPer];
            uint32_t found = 0;
            slice.values(i, x);
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e) found += candidate(x[e]);
            count += found;
            where |= (uint64_t)(found != 0) << ((i - u0) & 63);
        }
        team.prefix(count, none, own, unused);
        if (where && own <= kLocal)
            for (uint32_t i = u0; i < u1; ++i) {
                if (stretch <= 64) {
                    const uint64_t more = where >> (i - u0);
                    if (!more) break;
                    i += __ffsll(more) - 1;
                }
                float x[Slice::kPer];
                slice.values(i, x);
#pragma unroll
                for (int e = 0; e < Slice::kPer; ++e)
                    if (candidate(x[e])) sh.local[count++] = make_uint2(key_of<T>(x[e]), slice.column_of(i * Slice::kPer + e));
            }
        bool fits = true;
        uint32_t offset = 0, listed = 0;
        team.exchange(own, 0, [&](uint32_t c, uint64_t n_c, uint64_t) {
            if (c == team.cta) offset = listed;
            listed += (uint32_t)min(n_c, (uint64_t)kGathered + 1);
            fits = fits && n_c <= kLocal;
        });
        if (fits && listed <= kGathered) {
            uint2* const list = reinterpret_cast<uint2*>(dynamic);      // nobody reads a slice any more
            uint2* const to = cluster.map_shared_rank(list, 0) + offset;
            for (uint32_t i = tid; i < (uint32_t)own; i += kThreads) to[i] = sh.local[i];
            cluster.sync();
            if (team.cta) return;
            uint32_t inverse = 0;
            for (uint32_t i = tid; i < listed; i += kThreads) inverse = max(inverse, ~list[i].x);
            inverse = team.block_max(inverse);
            filter_and_draw<false>(team, List<T>{list, listed}, w, ~inverse, listed, k, p, least, u, token, prob);
            return;
        }
    } else if (w.ordinary) {
        // The weight of the row, exactly; then that of each bin, to 6e-5.  That says in which one or two bins the nucleus ends: what lies above them is
        // kept for sure, what lies in them is listed.
        for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
        uint64_t weight = 0, all_weight = 0;
        for (uint32_t i = tid; i < slice.units; i += kThreads) {
            float x[Slice::kPer];
            slice.values(i, x);
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e) weight += w.biased(x[e]) - w.kBias;
        }
        weight = team.block_sum(weight);
        team.exchange(weight, 0, [&](uint32_t, uint64_t part, uint64_t) { all_weight += part; });
        const uint64_t target = nucleus(p, all_weight);
        // All tokens of a weight below (1 - p) / cols of the row's together do not reach the 1 - p of it that may be left out: the nucleus ends above them.
        // An SM adds to shared memory one lane at a time, so binning them too took as long as everything else.
        const double rest = ((double)all_weight - (double)target) / kOne / a.cols;
        const float far = rest > 1e-9 ? fminf(kBins - 1.0f, 16.0f * -log2f((float)rest) + 1.0f) : kBins - 1.0f;
        for (uint32_t i = tid; i < slice.units; i += kThreads) {
            float x[Slice::kPer];
            slice.values(i, x);
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e) {
                const float d = w.below(x[e]) * 0.25f;
                if (d < far) {      // 2^13 of its weight over the middle of its bin: 2^(r / 16) for |r| <= 1/2, by two terms (off by 2e-6)
                    constexpr float l = 0.693147181f / 16.0f, kRound = 12582912.0f;      // 1.5 * 2^23: a sum with it has its whole part in the low bits
                    const float y = d + kRound, r = (y - kRound) - d;
                    const uint32_t b = __float_as_uint(y) & 0xfffu;
                    atomicAdd(&sh.bins[b], __float_as_uint(__fmaf_rn(r, __fmaf_rn(r, 4096.0f * l * l, 8192.0f * l), 8192.0f + 8388608.0f)) - 0x4b000000u);
                }
            }
        }
        cluster.sync();
        constexpr int kEach = kBins / kThreads;      // a thread takes two bins
        float sum = 0.0f, part[kEach];
        uint64_t in_bin[kEach] = {};      // a CTA's part fits in 32 bits (2^18 columns of 8371 at most), eight of them do not
#pragma unroll
        for (uint32_t c = 0; c < kMaxCtas; ++c)
            if (c < team.ctas) {
                const uint2 v = reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.bins, c))[tid];
                in_bin[0] += v.x;
                in_bin[1] += v.y;
            }
#pragma unroll
        for (int j = 0; j < kEach; ++j) part[j] = sum += (float)in_bin[j] * (exp2f(-(float)(tid * kEach + j) / 16.0f) / 8192.0f);
        float run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float up = __shfl_up_sync(kFull, run, o);
            if (lane >= o) run += up;
        }
        float* const sums = reinterpret_cast<float*>(sh.red2);
        if (lane == 31) sums[warp] = run;
        __syncthreads();
        float before = run - sum;
        for (int j = 0; j < warp; ++j) before += sums[j];
        // a weight in a bin is off by 6e-5 of it at most, the f32 sums by some 1e-6
        const float goal = (float)((double)target / kOne);
        uint32_t first = kBins - 1, last = kBins - 1;
#pragma unroll
        for (int j = kEach - 1; j >= 0; --j) {
            if (before + part[j] >= goal * 0.9999f) first = tid * kEach + j;
            if (before + part[j] >= goal * 1.0001f) last = tid * kEach + j;
        }
        first = kBins - 1 - team.block_max(kBins - 1 - first);
        last = kBins - 1 - team.block_max(kBins - 1 - last);
        // Bin b reaches from b - 1/2 to b + 1/2, in 64ths four times that.  What the f32 distance is off by decides between sure and listed at most.
        const float sure_end = 4.0f * (float)first - 2.01f, list_end = last < (uint32_t)kBins - 1 ? 4.0f * (float)last + 2.01f : INFINITY;
        uint64_t sure = 0, kept = 0, count = 0, none = 0, own, unused, where = 0;      // weight above the bins; of it, what min_p keeps; candidates, and their units
        for (uint32_t i = u0; i < u1; ++i) {
            float x[Slice::kPer];
            slice.values(i, x);
            unsigned above = 0;
            uint32_t found = 0;
#pragma unroll
            for (int e = 0; e < Slice::kPer; ++e) {
                const float d = w.below(x[e]);
                if (d < sure_end) above |= 1u << e;
                else if (d < list_end) ++found;
            }
            count += found;
            where |= (uint64_t)(found != 0) << ((i - u0) & 63);
            for (; above; above &= above - 1) {      // few: one at a time
                const double v = w.usual(slice.value(i * Slice::kPer + __ffs(above) - 1));
                const uint64_t q = w.whole(v);
                sure += q;
                if (v >= least) kept += q;
            }
        }
        uint32_t place = (uint32_t)count, end;
        team.prefix(count, none, own, unused);
        end = (uint32_t)count + place;
        place = (uint32_t)count;
        if (where && own <= kLocal)
            for (uint32_t i = u0, at = place; i < u1; ++i) {
                if (stretch <= 64) {
                    const uint64_t more = where >> (i - u0);
                    if (!more) break;
                    i += __ffsll(more) - 1;
                }
                float x[Slice::kPer];
                slice.values(i, x);
#pragma unroll
                for (int e = 0; e < Slice::kPer; ++e) {
                    const float d = w.below(x[e]);
                    if (!(d < sure_end) && d < list_end) sh.local[at++] = make_uint2(key_of<T>(x[e]), slice.column_of(i * Slice::kPer + e));
                }
            }
        const uint64_t own_sure = team.block_sum(sure);
        bool fits = true;
        uint64_t all_sure = 0, listed = 0;
        team.exchange(own_sure, own, [&](uint32_t, uint64_t s, uint64_t n_c) {
            all_sure += s;
            listed += n_c;
            fits = fits && n_c <= kLocal;
        });
        if (fits && listed) {
            const List<T> list{sh.local, (uint32_t)own};
            // its keys lie between those half a bin further out
            const float per_bin = 1.0f / (w.rate * 64.0f), lowest = top - (list_end + 0.5f) * per_bin, highest = top - fmaxf(sure_end - 0.5f, 0.0f) * per_bin;
            const uint32_t low = max(1u, key_of<T>(lowest)), high = min(kmax, key_of<T>(highest));
            const Border at = find_border<true>(team, list, w, low, high, all_sure, target, true);
            const Kept keep{at.key, ties_to_reach(w, at, target, ~0ull), least};
            uint64_t same = 0;
            for (uint32_t i = place; i < end; ++i) {
                const uint32_t key = sh.local[i].x;
                same += key == keep.cut;
                if (key > keep.cut) {
                    const double v = w.scaled(logit_of<T>(key));
                    if (v >= least) kept += w.whole(v);
                }
            }
            locate<true>(team, slice, w, keep, kept, same, u, token, prob);
            return;
        }
        if (listed) {      // the border among the row's keys that would be in the lists; starting over took 525 us where this takes 362 (256 x 128003 bf16, 0.9999)
            uint32_t largest_listed = 0, inverse = 0;
            for (uint32_t i = tid; i < slice.units; i += kThreads) {
                float x[Slice::kPer];
                slice.values(i, x);
#pragma unroll
                for (int e = 0; e < Slice::kPer; ++e) {
                    const float d = w.below(x[e]);
                    if (!(d < sure_end) && d < list_end) {
                        const uint32_t key = key_of<T>(x[e]);
                        largest_listed = max(largest_listed, key);
                        inverse = max(inverse, ~key);
                    }
                }
            }
            largest_listed = team.block_max(largest_listed);
            inverse = team.block_max(inverse);
            uint32_t high = 0, low = 0;
            team.exchange(largest_listed, inverse, [&](uint32_t, uint64_t a, uint64_t b) { high = max(high, (uint32_t)a); low = max(low, (uint32_t)b); });
            const Border at = find_border<true>(team, slice, w, ~low, high, all_sure, target, true);
            draw<true>(team, slice, w, Kept{at.key, ties_to_reach(w, at, target, ~0ull), least}, u, token, prob);
            return;
        }
    }
    // Too many candidates: on the row as it lies.
    uint32_t inverse = 0;
    uint64_t count = 0, count_all = 0;
    for (uint32_t i = tid; i < slice.units; i += kThreads) {
        float x[Slice::kPer];
        slice.values(i, x);
#pragma unroll
        for (int e = 0; e < Slice::kPer; ++e) {
            const uint32_t key = key_of<T>(x[e]);
            if (key) { inverse = max(inverse, ~key); ++count; }
        }
    }
    inverse = team.block_max(inverse);
    count = team.block_sum(count);
    const uint32_t own_inverse = inverse;
    team.exchange(own_inverse, count, [&](uint32_t, uint64_t x, uint64_t y) { inverse = max(inverse, (uint32_t)x); count_all += y; });
    filter_and_draw<true>(team, slice, w, ~inverse, count_all, k, p, least, u, token, prob);
}

template <typename T, bool kHeld>
int32_t launch_sample(fg_ctx* ctx, const SampleArgs& a, unsigned ctas, size_t bytes) {
    static std::atomic<uint64_t> attr_done{0};      // one bit per device; never less than the largest, which another thread's call may be about to use
    if (!(attr_done.load(std::memory_order_acquire) >> (ctx->device & 63) & 1ull)) {
        FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(sample_kernel<T, kHeld>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kHeld ? kHeldBytes : sizeof(uint2) * kGathered)));
        attr_done.fetch_or(1ull << (ctx->device & 63), std::memory_order_release);
    }
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
    if (held <= kHeldBytes) return launch_sample<T, true>(ctx, a, ctas, held < list ? list : held);
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
    const uint64_t line = 4ull * rows;
    for (const void* out : {(const void*)token_out, (const void*)prob_out}) {
        bool meets = fg_ranges_meet(out, line, logits, (uint64_t)rows * cols * fg_dtype_size(dtype)) || fg_ranges_meet(out, line, u, line);
        for (const void* in : {(const void*)temperature, (const void*)top_k, (const void*)top_p, (const void*)min_p}) meets = meets || fg_ranges_meet(out, line, in, line);
        FG_REQUIRE(ctx, !meets, "fg_sample: an output overlaps an input");
    }
    FG_REQUIRE(ctx, !fg_ranges_meet(token_out, line, prob_out, line), "fg_sample: token_out overlaps prob_out");
    if (rows == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, sample, ctx, SampleArgs{logits, u, temperature, top_k, top_p, min_p, token_out, prob_out, rows, cols});
}
