// Embedding lookup with scaling, and the gradient of its table.
//
// The lookup copies rows and is bound by memory.  The gradient is a sum over the tokens of each id.  The tokens are sorted by id
// (stably, so that the tokens of an id stand in their order), the sorted list is cut into chunks of one length, and a warp sums a chunk
// for 16 bytes of columns per lane: however the ids fall, every warp has the same work.  Ids that lie in one chunk are done with that;
// for an id that reaches over a border each chunk leaves its part in memory (f32), and the warp that brings the last part adds
// them in their order: only arrivals are counted atomically.
#include <cooperative_groups.h>

#include <atomic>

#include "rows.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kPacks = 4;      // of the lookup

struct EmbedArgs {
    uint32_t tokens, vocab, dim;
    const uint32_t* ids;
    const void* src;
    float scale;
    void* dst;
    int accumulate;
};


// ---- the tokens in order of their ids ----
// Least significant digit first, up to 9 bits a pass, by the CTAs of one cluster: a warp holds a stretch of the list and counts its digits
// in shared memory, the counts become places (over the warps of a CTA, over the CTAs by distributed shared memory), and the warp goes
// over its stretch again, 32 entries at a time, and puts each at its digit's next place.  The list stays in the L2; what a
// pass costs is its steps one after the other (some 3 us), which a grid's worth of CTAs and a launch per step would not shorten.
// The grid's other CTAs write the zeros meanwhile: each looks through the ids for those of its rows and clears the rest.
constexpr int kSortThreads = 1024, kSortWarps = 32, kMaxBins = 512, kHeldEntries = 4096;      // entries that a CTA holds in registers
constexpr uint32_t kFillRows = 1u << 17;      // rows that a CTA marks at a time
struct SortArgs {
    uint32_t tokens, vocab;
    const uint32_t* ids;
    uint2 *a, *b;             // (id, token): pass 0 writes a, pass 1 b, ...
    uint32_t* used;           // how many tokens have an id of the table
    int passes, digit, group, shares;
    char* dtable;             // rows that no token has, of those from `first_row` on, are cleared
    uint64_t row_bytes;
    uint32_t first_row;
    uint32_t* arrived;        // counters of the second launch
    uint64_t borders;
};

constexpr uint32_t kMaxGroup = 2048;     // rows that a block of the second launch marks
constexpr uint32_t kSegment = 2048;      // bytes that a warp clears at a time
__device__ __forceinline__ void clear_bytes(char* p, uint32_t bytes, int lane) {
    const uint32_t before = min((uint32_t)(-reinterpret_cast<uintptr_t>(p) & 15u), bytes), words = (bytes - before) / 16;
    uint4* const q = reinterpret_cast<uint4*>(p + before);
#pragma unroll
    for (uint32_t k = 0; k < kSegment / 512; ++k)
        if (32 * k + lane < words) q[32 * k + lane] = make_uint4(0, 0, 0, 0);
    if (2 * lane < before) *reinterpret_cast<uint16_t*>(p + 2 * lane) = 0;
    if (2 * lane < bytes - before - 16 * words) *reinterpret_cast<uint16_t*>(p + before + 16 * words + 2 * lane) = 0;
}
// The rows are dealt out in groups of 2^group (64 KB, where there are many), since the ids of a batch crowd together, to 2^shares CTAs.
__device__ void clear_absent(const SortArgs& s, uint32_t part, uint32_t* marks) {
    const uint32_t parts = 1u << s.shares;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rows = s.vocab - s.first_row, groups = (uint32_t)(((uint64_t)rows + (1u << s.group) - 1) >> s.group);
    const uint32_t own = part < groups ? (groups - part + parts - 1) / parts : 0;      // groups part, part + parts, ...
    const uint32_t step = kFillRows >> s.group;      // groups marked at a time
    const uint64_t segments = (s.row_bytes + kSegment - 1) / kSegment;
    for (uint32_t g = 0; g < own; g += min(step, own - g)) {
        const uint32_t n = min(step, own - g) << s.group;
        for (uint32_t i = tid; i < (n + 31) / 32; i += kSortThreads) marks[i] = 0;
        __syncthreads();
        const uint32_t head = min(s.tokens, (uint32_t)(-reinterpret_cast<uintptr_t>(s.ids) & 15u) / 4), words = (s.tokens - head) / 4;
        auto mark = [&](uint32_t id) {
            id -= s.first_row;      // ids below it come out behind all rows
            const uint32_t q = id >> s.group, at = (q >> s.shares) - g;
            if ((q & (parts - 1)) == part && at < (n >> s.group)) {
                const uint32_t k = (at << s.group) + (id & ((1u << s.group) - 1));
                atomicOr(&marks[k >> 5], 1u << (k & 31));
            }
        };
        const uint4* const ids = reinterpret_cast<const uint4*>(s.ids + head);
#pragma unroll 4
        for (uint32_t i = tid; i < words; i += kSortThreads) {
            const uint4 q = __ldg(ids + i);
            mark(q.x); mark(q.y); mark(q.z); mark(q.w);
        }
        if (tid < head) mark(s.ids[tid]);
        if (tid < s.tokens - head - 4 * words) mark(s.ids[head + 4 * words + tid]);
        __syncthreads();
        const uint64_t units = n * segments;      // the warps side by side
        for (uint64_t k = warp; k < units; k += kSortWarps) {
            const uint32_t i = (uint32_t)(k / segments);
            const uint64_t v = (((uint64_t)(g + (i >> s.group)) * parts + part) << s.group) + (i & ((1u << s.group) - 1));
            const uint64_t from = k % segments * kSegment;
            if (v < rows && !(marks[i >> 5] >> (i & 31) & 1u))
                clear_bytes(s.dtable + (s.first_row + v) * s.row_bytes + from, (uint32_t)min((uint64_t)kSegment, s.row_bytes - from), lane);
        }
        __syncthreads();
    }
}

// Leaves in same[j] the lanes whose entry has this lane's digit.  Without a test per set of 32 entries: the ballots of several
// bits are in flight together (a pass's placing of up to 32 entries per warp 2130 cycles, with the tests 3300; of 128 6150 and 6500).
template <int kSets>
__device__ __forceinline__ void same_digit(const uint2* e, unsigned* same, int shift, int digit) {
    uint32_t d[kSets];
#pragma unroll
    for (int j = 0; j < kSets; ++j) d[j] = e[j].x >> shift;
#pragma unroll 4
    for (int b = 0; b < digit; ++b)
#pragma unroll
        for (int j = 0; j < kSets; ++j) {
            const bool bit = d[j] >> b & 1u;
            const unsigned ones = __ballot_sync(kFull, bit);
            same[j] &= bit ? ones : ~ones;
        }
}

// kHeld: a lane's entries (four at most) stay in registers from the counting to the placing.
template <bool kHeld>
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const SortArgs s) {
    extern __shared__ __align__(16) uint32_t counts[];      // [warp][bin], then (kHeld) the CTA's entries in order
    __shared__ uint32_t totals[kMaxBins], bases[kMaxBins], begins[kMaxBins], fours[kSortThreads], red[kSortWarps + 1], red_cta[kSortWarps];
    fg_grid_enter();
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), cta = cluster.block_rank();
    if (blockIdx.x >= ctas) {
        if (blockIdx.x - ctas < 1u << s.shares) clear_absent(s, blockIdx.x - ctas, counts);
        return;
    }
    constexpr int kAhead = 4, kMaxCtas = 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << s.digit;
    const uint64_t stretch = ((uint64_t)s.tokens + ctas * kSortWarps - 1) / (ctas * kSortWarps);
    const uint32_t i0 = (uint32_t)min((uint64_t)s.tokens, (cta * kSortWarps + warp) * stretch), i1 = (uint32_t)min((uint64_t)s.tokens, i0 + stretch);
    uint32_t* const mine = counts + warp * bins;
    uint2* const staged = reinterpret_cast<uint2*>(counts + kSortWarps * bins);
    for (uint64_t i = cta * kSortThreads + tid; i < s.borders; i += ctas * kSortThreads) s.arrived[i] = 0;
    for (int pass = 0; pass < s.passes; ++pass) {
        const uint2* const from = pass & 1 ? s.a : s.b;
        uint2* const to = pass & 1 ? s.b : s.a;
        const int shift = pass * s.digit;
        uint2 e[kAhead];
        auto load = [&](uint32_t i) {      // padding becomes the last id
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const uint32_t k = i + 32 * j + lane;
                e[j] = k >= i1 ? make_uint2(0, 0) : pass ? __ldcg(from + k) : make_uint2(min(s.ids[k], s.vocab), k);
            }
        };
        if (kHeld) load(i0);
        for (int i = 4 * tid; i < kSortWarps * bins; i += 4 * kSortThreads) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        uint32_t inside = 0;
        for (uint32_t i = i0; i < i1; i += 32 * kAhead) {
            if (!kHeld) load(i);
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (i + 32 * j + lane < i1) {
                    atomicAdd(&mine[e[j].x >> shift & (bins - 1)], 1u);
                    inside += e[j].x < s.vocab;
                }
        }
        if (pass == 0) {
            inside = __reduce_add_sync(kFull, inside);
            if (lane == 0) red[warp] = inside;
        }
        __syncthreads();
        // over the warps: a thread takes a digit of kSortWarps / groups warps, then adds the groups before its own
        const int groups = bins >= kSortThreads / 2 ? 2 : 4, each = kSortWarps / groups, bin = tid & (bins - 1), group = tid >> s.digit;
        uint32_t sum = 0;
        if (group < groups) {
#pragma unroll 8
            for (int w = group * each; w < (group + 1) * each; ++w) {
                const uint32_t c = counts[w * bins + bin];
                counts[w * bins + bin] = sum;
                sum += c;
            }
            fours[tid] = sum;
        }
        if (pass == 0 && warp == 0) {
            inside = __reduce_add_sync(kFull, red[lane]);
            if (lane == 0) red[kSortWarps] = inside;
        }
        __syncthreads();
        if (group < groups) {
            uint32_t before = 0;
            for (int g = 0; g < group; ++g) before += fours[g * bins + bin];
            if (group == groups - 1) totals[bin] = before + sum;
            if (before)
#pragma unroll 8
                for (int w = group * each; w < (group + 1) * each; ++w) counts[w * bins + bin] += before;
        }
        cluster.sync();
        uint32_t before = 0, all = 0;
        if (tid < bins) {
#pragma unroll
            for (uint32_t c = 0; c < kMaxCtas; ++c) {
                const uint32_t t = c < ctas ? cluster.map_shared_rank(totals, c)[tid] : 0;
                before += c < cta ? t : 0;
                all += t;
            }
        }
        if (pass == 0 && cta == 0 && tid == 0) {
            uint32_t n = 0;
            for (uint32_t c = 0; c < ctas; ++c) n += cluster.map_shared_rank(red, c)[kSortWarps];
            *s.used = n;
        }
        const uint32_t here = tid < bins ? totals[tid] : 0;
        uint32_t run = all, run_cta = here;      // where each digit begins in the list, and among the CTA's entries
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(kFull, run, o), up_cta = __shfl_up_sync(kFull, run_cta, o);
            if (lane >= o) { run += up; run_cta += up_cta; }
        }
        if (lane == 31) { red[warp] = run; red_cta[warp] = run_cta; }
        __syncthreads();
        if (tid < bins) {
            uint32_t base = run - all + before, begin = run_cta - here;
            for (int w = 0; w < warp; ++w) { base += red[w]; begin += red_cta[w]; }
            bases[tid] = kHeld ? base - begin : base;
            begins[tid] = begin;
        }
        __syncthreads();
        for (uint32_t i = i0; i < i1; i += 32 * kAhead) {
            if (!kHeld) load(i);
            unsigned same[kAhead];      // the lanes with this digit, a bit at a time (one matching instruction takes as long as it finds values)
#pragma unroll
            for (int j = 0; j < kAhead; ++j) same[j] = __ballot_sync(kFull, i + 32 * j + lane < i1);
            const uint32_t sets = (min(i1 - i, 32u * kAhead) + 31) / 32;
            if (sets == 1) same_digit<1>(e, same, shift, s.digit);
            else if (sets == 2) same_digit<2>(e, same, shift, s.digit);
            else same_digit<kAhead>(e, same, shift, s.digit);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (i + 32 * j >= i1) break;
                const bool there = i + 32 * j + lane < i1;
                const uint32_t d = e[j].x >> shift & (bins - 1), rank = __popc(same[j] & ((1u << lane) - 1));
                uint32_t place = 0;
                if (there) place = (kHeld ? begins[d] : bases[d]) + mine[d] + rank;
                __syncwarp();
                if (there && rank == 0) mine[d] += __popc(same[j]);
                __syncwarp();
                if (there) (kHeld ? staged : to)[place] = e[j];
            }
        }
        if (kHeld) {      // entries of a digit lie together now: written one by one from the registers, each costs two cycles of the SM
            __syncthreads();
            const uint32_t c0 = (uint32_t)min((uint64_t)s.tokens, cta * kSortWarps * stretch), own = (uint32_t)min((uint64_t)s.tokens, c0 + kSortWarps * stretch) - c0;
            for (uint32_t i = tid; i < own; i += kSortThreads) {
                const uint2 v = staged[i];
                to[bases[v.x >> shift & (bins - 1)] + i] = v;
            }
        }
        cluster.sync();      // the list is there, and nobody reads these totals any more
    }
}

// ---- sums over the sorted list ----
struct SumArgs {
    uint32_t tokens, dim, length, tiles;      // entries per warp, tiles of 32 packs per row
    uint64_t chunks;
    const uint2* list;
    const uint32_t* used;
    const void *dout, *dout_end;
    void *dtable, *dtable_end;
    float* parts;             // [chunks][2][pitch]: of the id that reaches in from the chunk before, and of the one that goes on in the next
    uint64_t pitch;
    uint32_t* arrived;        // [chunks][tiles], zero at the start: parts there of the id that goes on behind the chunk
    float scale;
    uint32_t blocks, fills, group, fill_rows;      // blocks that sum, and blocks among them that clear 2^group rows each of the first fill_rows
    uint64_t row_bytes;
};

// Index of the first entry whose id is not below `id`: 32 probes at a time, by a whole warp.
__device__ __forceinline__ uint32_t first_not_below(const uint2* list, uint32_t n, uint64_t id, int lane) {
    uint32_t lo = 0;
    while (n > 0) {
        const uint32_t step = (n + 31) / 32, at = (uint32_t)lane * step;
        const int c = __popc(__ballot_sync(kFull, at < n && list[lo + at].x < id));
        if (c == 0) return lo;
        const uint32_t past = (uint32_t)(c - 1) * step + 1;
        lo += past;
        n = min(step - 1, n - past);
    }
    return lo;
}
// A block of 8 warps clears those of n rows from `rows` on that are not marked.
__device__ __forceinline__ void clear_unmarked(char* rows, uint32_t n, uint64_t row_bytes, const uint32_t* marks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t segments = (row_bytes + kSegment - 1) / kSegment, units = n * segments;
    for (uint64_t k = warp; k < units; k += 8) {
        const uint32_t i = (uint32_t)(k / segments);
        const uint64_t from = k % segments * kSegment;
        if (!(marks[i >> 5] >> (i & 31) & 1u)) clear_bytes(rows + i * row_bytes + from, (uint32_t)min((uint64_t)kSegment, row_bytes - from), lane);
    }
}
// A block clears the rows of its group that the sorted list does not name.
__device__ void clear_group(const SumArgs& s, uint32_t fill, uint32_t* marks, uint32_t* ends) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint64_t v0 = (uint64_t)fill << s.group, v1 = min((uint64_t)s.fill_rows, v0 + (1u << s.group));
    for (uint32_t i = tid; i < ((1u << s.group) + 31) / 32; i += 256) marks[i] = 0;
    if (warp < 2) {
        const uint32_t at = first_not_below(s.list, *s.used, warp ? v1 : v0, lane);
        if (lane == 0) ends[warp] = at;
    }
    __syncthreads();
    for (uint64_t i = ends[0] + tid; i < ends[1]; i += 256) {
        const uint32_t k = s.list[i].x - (uint32_t)v0;
        atomicOr(&marks[k >> 5], 1u << (k & 31));
    }
    __syncthreads();
    clear_unmarked(static_cast<char*>(s.dtable) + v0 * s.row_bytes, (uint32_t)(v1 - v0), s.row_bytes, marks);
}
template <typename T, bool kShift>
__device__ __forceinline__ uint4 load_old(const SumArgs& s, uint32_t v, uint64_t col, uint32_t left) {
    return fg_load_pack<T, kShift>(static_cast<const T*>(s.dtable) + (uint64_t)v * s.dim + col, left, (const T*)s.dtable, (const T*)s.dtable_end);
}
template <typename T, bool kShift, bool kAdd>
__device__ __forceinline__ void store_sum(const SumArgs& s, uint32_t v, uint64_t col, uint32_t left, const float (&x)[FgPack<T>::E], const uint4& old) {
    constexpr int E = FgPack<T>::E;
    float y[E];
    if (kAdd) {
        FgPack<T>::widen(old, y);
        if (kShift) __syncwarp();      // a lane writes words that others have read
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = __fmaf_rn(s.scale, x[e], y[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = s.scale * x[e];
    }
    fg_store_pack<T, kShift>(static_cast<T*>(s.dtable) + (uint64_t)v * s.dim + col, FgPack<T>::narrow(y), left);
}
template <typename T, bool kShift, bool kAdd>
__device__ __forceinline__ void store_sum(const SumArgs& s, uint32_t v, uint64_t col, uint32_t left, const float (&x)[FgPack<T>::E]) {
    store_sum<T, kShift, kAdd>(s, v, col, left, x, kAdd && left ? load_old<T, kShift>(s, v, col, left) : make_uint4(0, 0, 0, 0));
}
template <int E>
__device__ __forceinline__ void store_part(float* p, const float (&x)[E]) {
#pragma unroll
    for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
}

// A part of an id that reaches over chunks, from `first` to `end`, is written.  The warp that brings the last one adds them, in their order
// whoever it is, and nobody waits.  A launch of its own for that took 1.9 us of 31.1 (8192 tokens, 1024 f32 columns) and 2.1 of 114.0
// (32768 tokens, 4096 bf16 columns).
template <typename T, bool kShift, bool kAdd>
__device__ __forceinline__ void join_parts(const SumArgs& s, uint32_t id, uint64_t first, uint64_t end, uint32_t tile, uint64_t col, uint32_t left, int lane) {
    constexpr int E = FgPack<T>::E;
    __threadfence();      // the part, before its arrival
    __syncwarp();
    uint32_t there = 0;
    if (lane == 0) there = atomicAdd(&s.arrived[first * s.tiles + tile], 1u);
    const uint64_t more = end - first;
    if (__shfl_sync(kFull, there, 0) != more) return;
    __threadfence();
    float acc[E] = {};
    if (left) {
        const float* p = s.parts + (2 * first + 1) * s.pitch + col;      // its end of the first chunk, then the beginnings of the next ones
        for (uint64_t j = 0; j <= more; j += 4) {
            float4 v[4][E / 4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < E / 4; ++e)
                    v[k][e] = j + k <= more ? __ldcg(reinterpret_cast<const float4*>(p + (j + k ? 2 * (j + k) - 1 : 0) * s.pitch + 4 * e)) : make_float4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < E / 4; ++e) {
                    acc[4 * e] += v[k][e].x; acc[4 * e + 1] += v[k][e].y; acc[4 * e + 2] += v[k][e].z; acc[4 * e + 3] += v[k][e].w;
                }
        }
    }
    store_sum<T, kShift, kAdd>(s, id, col, left, acc);
}
// The last chunk that the id behind chunk c's end reaches into; the first one that the id which reaches into chunk c began in.
__device__ __forceinline__ uint64_t last_chunk_of(const SumArgs& s, uint32_t id, uint64_t c, int lane) {
    const uint64_t size = 8ull * s.length;
    while (true) {
        const uint64_t at = (c + 1 + lane) * size;
        const unsigned on = __ballot_sync(kFull, at < s.tokens && s.list[at].x == id);
        if (on != kFull) return c + __ffs(~on) - 1;
        c += 32;
    }
}
__device__ __forceinline__ uint64_t first_chunk_of(const SumArgs& s, uint32_t id, uint64_t c, int lane) {
    const uint64_t size = 8ull * s.length;
    while (true) {
        const uint64_t at = c > (uint64_t)lane ? (c - lane) * size : 0;      // 0: the list's beginning
        const unsigned on = __ballot_sync(kFull, at && s.list[at - 1].x == id);
        if (on != kFull) return c - (__ffs(~on) - 1);
        c -= 32;
    }
}

// A warp takes `length` entries and a tile of columns, with eight rows on their way while they are added one by one; the eight warps of a
// block take the same columns of entries that follow each other and join their parts in shared memory, so a chunk is eight stretches.
template <typename T, bool kShift, bool kAdd>
__global__ void __launch_bounds__(256, 3) embed_sum_kernel(const SumArgs s) {
    constexpr int E = FgPack<T>::E, kAhead = kAdd ? 4 : 8;
    __shared__ float4 ends[8][E / 4][32];         // a warp's part of the id that reaches in
    __shared__ bool through[8];                   // the warp has one id alone, which reaches in and goes on
    fg_grid_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t block = blockIdx.x;
    if constexpr (!kAdd) {      // the blocks that clear are spread evenly among the others: writes alone run at two thirds of the rate of reads and writes
        const uint32_t all = s.blocks + s.fills, before = (uint32_t)((uint64_t)block * s.fills / all), past = (uint32_t)((uint64_t)(block + 1) * s.fills / all);
        if (past != before) {
            uint32_t* const room = reinterpret_cast<uint32_t*>(&ends[0][0][0]);      // 4 KB at least
            clear_group(s, before, room + 2, room);
            return;
        }
        block -= before;
    }
    const uint64_t chunk = block / s.tiles, i0 = min((uint64_t)s.tokens, (chunk * 8 + warp) * s.length), i1 = min((uint64_t)s.tokens, i0 + s.length);
    const uint64_t col = ((uint64_t)(block % s.tiles) * 32 + lane) * E;
    const uint32_t left = col < s.dim ? (uint32_t)min((uint64_t)E, s.dim - col) : 0;
    const T* const dout = static_cast<const T*>(s.dout);
    constexpr uint32_t kNone = 0xffffffffu;      // no id of the table
    const uint32_t before = i0 ? s.list[i0 - 1].x : kNone, after = i1 < s.tokens ? s.list[i1].x : kNone;
    uint2 mine = i0 + lane < i1 ? s.list[i0 + lane] : make_uint2(0, 0);
    uint32_t behind = i0 + lane + 1 < i1 ? s.list[i0 + lane + 1].x : after;      // the id after each entry's
    const uint32_t used = *s.used;      // padding has the last places
    if (chunk * 8 * s.length >= used) return;
    const uint32_t n = (uint32_t)(min((uint64_t)used, i1) - min((uint64_t)used, i0));
    bool reaches_in = n && __shfl_sync(kFull, mine.x, 0) == before, open = false;      // open: the id of the last entry goes on
    const bool enters = warp == 0 && reaches_in;
    float acc[E] = {};
    auto leave = [&] {
#pragma unroll
        for (int e = 0; e < E / 4; ++e) ends[warp][e][lane] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
    };
    // `kAhead` rows are on their way: as one is added, the one `kAhead` entries behind it is asked for.
    uint4 v[kAhead], old[kAdd ? kAhead : 1];
    auto ask = [&](int k, uint32_t j, const uint2& from, unsigned ending) {      // entry j, one of the 32 in `from`
        const uint32_t t = __shfl_sync(kFull, from.y, j), id = kAdd ? __shfl_sync(kFull, from.x, j) : 0;
        if (left) v[k] = fg_load_pack<T, kShift>(dout + (uint64_t)t * s.dim + col, left, dout, (const T*)s.dout_end);
        if (kAdd && left && (ending >> j & 1u)) old[kAdd ? k : 0] = load_old<T, kShift>(s, id, col, left);
    };
    unsigned ending = __ballot_sync(kFull, behind != mine.x);      // the last of their id
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        v[k] = make_uint4(0, 0, 0, 0);
        if (kAdd) old[k] = v[k];
        if ((uint32_t)k < n) ask(k, k, mine, ending);
    }
    for (uint32_t j0 = 0; j0 < n; j0 += 32) {
        const uint64_t i = i0 + j0 + 32 + lane;      // the next 32
        const uint2 next = i < i1 ? s.list[i] : make_uint2(0, 0);
        const uint32_t next_behind = i + 1 < i1 ? s.list[i + 1].x : after;
        const unsigned next_ending = __ballot_sync(kFull, next_behind != next.x);
        const uint32_t m = min(32u, n - j0);
        open = !(ending >> (m - 1) & 1u);
#pragma unroll 1
        for (uint32_t j = 0; j < m; j += kAhead) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (j + k >= m) break;
                float x[E];
                FgPack<T>::widen(v[k], x);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += x[e];
                if (ending >> (j + k) & 1u) {
                    const uint32_t id = __shfl_sync(kFull, mine.x, j + k);
                    if (reaches_in) leave();
                    else store_sum<T, kShift, kAdd>(s, id, col, left, acc, old[kAdd ? k : 0]);
                    reaches_in = false;
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
                }
                if (j0 + j + k + kAhead < n) {
                    const bool here = j + kAhead < 32;
                    ask(k, (j + k + kAhead) & 31, here ? mine : next, here ? ending : next_ending);
                }
            }
        }
        mine = next;
        ending = next_ending;
    }
    if (open && reaches_in) leave();
    if (lane == 0) through[warp] = open && reaches_in;
    __syncthreads();
    // Now the ids that cross a stretch's end.  The warp that one begins in adds what the next ones left of it; the block's first warp does so for
    // the id that reaches into the block.
    if (enters) {
        float sum[E] = {};
        bool on = true;      // it goes on behind the chunk
        for (int w = 0; w < 8; ++w) {
#pragma unroll
            for (int e = 0; e < E / 4; ++e) {
                const float4 p = ends[w][e][lane];
                sum[4 * e] += p.x; sum[4 * e + 1] += p.y; sum[4 * e + 2] += p.z; sum[4 * e + 3] += p.w;
            }
            on = through[w];
            if (!on) break;
        }
        if (left) store_part(s.parts + 2 * chunk * s.pitch + col, sum);
        join_parts<T, kShift, kAdd>(s, before, first_chunk_of(s, before, chunk, lane), on ? last_chunk_of(s, before, chunk, lane) : chunk, block % s.tiles, col, left, lane);
    }
    if (open && !reaches_in) {
        bool out = warp == 7;
        for (int w = warp + 1; w < 8; ++w) {
#pragma unroll
            for (int e = 0; e < E / 4; ++e) {
                const float4 p = ends[w][e][lane];
                acc[4 * e] += p.x; acc[4 * e + 1] += p.y; acc[4 * e + 2] += p.z; acc[4 * e + 3] += p.w;
            }
            if (!through[w]) break;
            out = w == 7;
        }
        if (out) {
            if (left) store_part(s.parts + (2 * chunk + 1) * s.pitch + col, acc);
            join_parts<T, kShift, kAdd>(s, after, chunk, last_chunk_of(s, after, chunk, lane), block % s.tiles, col, left, lane);
        } else store_sum<T, kShift, kAdd>(s, after, col, left, acc);
    }
}

// ---- few tokens ----
// Up to kFew of them need no sorting: a block takes a token and two tiles of columns, finds by ballots where else its id stands, and if nowhere
// before, adds those rows, four warps a quarter of them each where there are many.  Blocks behind these clear the other rows.  One launch
// instead of several, added to the table: 129 tokens of 1024 f32 columns 16 -> 4 us, 256 of 777 25 -> 7, 512 of 1024 17 -> 10; from there on the
// blocks of tokens that are not their id's first cost more than the sort.
constexpr uint32_t kFew = 512;
template <typename T, bool kShift, bool kAdd>
__global__ void __launch_bounds__(256) embed_few_kernel(const SumArgs s, const uint32_t* ids) {
    constexpr int E = FgPack<T>::E, kAhead = 8, kWords = kFew / 32;
    __shared__ uint32_t marks[kMaxGroup / 32];
    __shared__ unsigned where[kWords];
    __shared__ float4 parts[8][E / 4][32];
    fg_grid_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (!kAdd && blockIdx.x >= s.blocks) {
        const uint64_t v0 = (uint64_t)(blockIdx.x - s.blocks) << s.group;
        const uint32_t n = (uint32_t)(min((uint64_t)s.fill_rows, v0 + (1u << s.group)) - v0);
        for (uint32_t i = threadIdx.x; i < (n + 31) / 32; i += 256) marks[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < s.tokens; i += 256) {
            const uint32_t k = ids[i] - (uint32_t)v0;
            if (k < n) atomicOr(&marks[k >> 5], 1u << (k & 31));
        }
        __syncthreads();
        clear_unmarked(static_cast<char*>(s.dtable) + v0 * s.row_bytes, n, s.row_bytes, marks);
        return;
    }
    const uint32_t pairs = (s.tiles + 1) / 2, t = blockIdx.x / pairs, tile = blockIdx.x % pairs * 2 + (warp >> 2), quarter = warp & 3;
    const uint64_t col = ((uint64_t)tile * 32 + lane) * E;
    const uint32_t left = col < s.dim ? (uint32_t)min((uint64_t)E, s.dim - col) : 0, id = ids[t];
    if (id >= s.fill_rows) return;      // padding
    uint4 old = make_uint4(0, 0, 0, 0);
    if (kAdd && left && quarter == 0) old = load_old<T, kShift>(s, id, col, left);
#pragma unroll
    for (int j = warp; j < kWords; j += 8) {
        const unsigned found = __ballot_sync(kFull, 32 * j + lane < s.tokens && ids[min(32 * j + lane, s.tokens - 1)] == id);
        if (lane == 0) where[j] = found;
    }
    __syncthreads();
    uint32_t count = 0, first = kFew;
#pragma unroll
    for (int j = kWords - 1; j >= 0; --j) {
        count += __popc(where[j]);
        if (where[j]) first = 32 * j + __ffs(where[j]) - 1;
    }
    if (first < t) return;      // its first token adds
    const bool shared = count >= 8;
    const uint32_t from = shared ? count * quarter / 4 : 0, n = shared ? count * (quarter + 1) / 4 - from : quarter ? 0 : count;
    uint32_t word = 0, skip = from;
    while (n && skip >= (uint32_t)__popc(where[word])) skip -= __popc(where[word++]);
    unsigned bits = n ? where[word] : 0;
    for (; skip; --skip) bits &= bits - 1;
    const T* const dout = static_cast<const T*>(s.dout);
    float acc[E] = {};
    for (uint32_t i = 0; i < n; i += kAhead) {
        uint4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            v[k] = make_uint4(0, 0, 0, 0);
            if (i + k < n) {
                while (!bits) bits = where[++word];
                const uint64_t row = 32 * word + __ffs(bits) - 1;
                bits &= bits - 1;
                if (left) v[k] = fg_load_pack<T, kShift>(dout + row * s.dim + col, left, dout, (const T*)s.dout_end);
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i + k < n) {
                float x[E];
                FgPack<T>::widen(v[k], x);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += x[e];
            }
    }
    if (shared) {
#pragma unroll
        for (int e = 0; e < E / 4; ++e) parts[warp][e][lane] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
        __syncthreads();
        for (int q = 1; q < 4 && quarter == 0; ++q)
#pragma unroll
            for (int e = 0; e < E / 4; ++e) {
                const float4 p = parts[warp + q][e][lane];
                acc[4 * e] += p.x; acc[4 * e + 1] += p.y; acc[4 * e + 2] += p.z; acc[4 * e + 3] += p.w;
            }
    }
    if (quarter == 0) store_sum<T, kShift, kAdd>(s, id, col, left, acc, old);
}

// ---- lookup ----
// A warp takes a token and a tile of columns, `kPacks` packs of 16 bytes per lane or, off 16-byte boundaries, as many single elements side by side
// (words turned by a row's distance from the boundary took more instructions than the elements do).
template <typename T, bool kStraight>
__global__ void __launch_bounds__(256) embed_kernel(uint32_t tokens, uint32_t vocab, uint32_t dim, uint32_t tiles, const uint32_t* ids, const T* table, float scale, T* out) {
    using Unit = std::conditional_t<kStraight, uint4, T>;
    constexpr int E = sizeof(Unit) / sizeof(T), kUnits = kStraight ? kPacks : kPacks * 4;
    fg_grid_enter();
    const int lane = threadIdx.x & 31;
    const uint32_t units = dim / E;      // of a row
    const uint64_t work = (uint64_t)tokens * tiles;
    for (uint64_t k = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); k < work; k += (uint64_t)gridDim.x * 8) {
        const uint32_t t = (uint32_t)(k / tiles), first = (uint32_t)(k % tiles) * (32 * kUnits) + lane, id = ids[t];
        const bool inside = id < vocab;
        const Unit* const from = reinterpret_cast<const Unit*>(table + (uint64_t)id * dim);
        Unit* const to = reinterpret_cast<Unit*>(out + (uint64_t)t * dim);
        Unit v[kUnits];
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            v[j] = Unit{};
            if (inside && first + 32 * j < units) v[j] = from[first + 32 * j];
        }
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            if constexpr (kStraight) {
                float x[E];
                FgPack<T>::widen(v[j], x);
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] *= scale;
                v[j] = FgPack<T>::narrow(x);
            } else v[j] = fg_narrow<T>(fg_widen(v[j]) * scale);
            if (!inside) v[j] = Unit{};
            if (first + 32 * j < units) to[first + 32 * j] = v[j];
        }
    }
}

template <typename T>
int32_t embed_fwd(fg_ctx* ctx, const EmbedArgs& a) {
    const bool straight = fg_rows_lie_straight(a.dim, sizeof(T), a.src, a.dst);
    const uint32_t tile = 32 * kPacks * (straight ? FgPack<T>::E : 4), tiles = (uint32_t)(((uint64_t)a.dim + tile - 1) / tile);
    const uint64_t blocks = ((uint64_t)a.tokens * tiles + 7) / 8, cap = 32ull * ctx->sm_count;
    fg_launch(ctx, straight ? embed_kernel<T, true> : embed_kernel<T, false>, (unsigned)(blocks < cap ? blocks : cap), 256, 0, a.tokens, a.vocab, a.dim, tiles, a.ids,
              (const T*)a.src, a.scale, (T*)a.dst);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

template <typename T>
int32_t embed_bwd(fg_ctx* ctx, const EmbedArgs& a) {
    constexpr uint32_t E = FgPack<T>::E;
    SumArgs s{};
    s.tokens = a.tokens;
    s.dim = a.dim;
    s.tiles = (uint32_t)(((uint64_t)a.dim + 32 * E - 1) / (32 * E));
    s.pitch = (uint64_t)s.tiles * 32 * E;
    s.scale = a.scale;
    s.dout = a.src;
    s.dout_end = (const T*)a.src + (uint64_t)a.tokens * a.dim;
    s.dtable = a.dst;
    s.dtable_end = (T*)a.dst + (uint64_t)a.vocab * a.dim;
    const bool straight = fg_rows_lie_straight(a.dim, sizeof(T), a.src, a.dst), add = a.accumulate != 0;
    if (a.tokens <= kFew) {
        s.row_bytes = (uint64_t)a.dim * sizeof(T);
        s.fill_rows = a.vocab;
        while (1u << s.group < kMaxGroup && s.row_bytes << (s.group + 1) <= 32768) ++s.group;
        const uint64_t work = (uint64_t)a.tokens * ((s.tiles + 1) / 2), fills = add ? 0 : ((uint64_t)a.vocab + (1ull << s.group) - 1) >> s.group;
        FG_REQUIRE(ctx, work + fills < (1ull << 31), "fg_embedding_bwd: tensor too large");
        s.blocks = (uint32_t)work;
        fg_launch(ctx, add ? straight ? embed_few_kernel<T, false, true> : embed_few_kernel<T, true, true>
                           : straight ? embed_few_kernel<T, false, false> : embed_few_kernel<T, true, false>, (unsigned)(work + fills), 256, 0, s, a.ids);
        FG_LAUNCHED(ctx);
        return FG_OK;
    }
    // Stretches for four waves of warps, of 8 to 128 entries; a chunk is the eight stretches of a block.
    const uint64_t want = (uint64_t)a.tokens * s.tiles / (96ull * ctx->sm_count);
    s.length = (uint32_t)(want < 8 ? 8 : want > 128 ? 128 : (want + 7) / 8 * 8);
    s.chunks = ((uint64_t)a.tokens + 8ull * s.length - 1) / (8ull * s.length);
    const uint64_t list = ((uint64_t)a.tokens * 8 + 255) / 256 * 256;
    void* p;
    const uint64_t parts = 8 * s.chunks * s.pitch, blocks = s.chunks * s.tiles;
    const int32_t st = fg_ws_alloc(ctx, 2 * list + 256 + parts + 4 * blocks, &p);
    if (st != FG_OK) return st;
    SortArgs o{};
    o.tokens = a.tokens;
    o.vocab = a.vocab;
    o.ids = a.ids;
    o.a = (uint2*)p;
    o.b = (uint2*)((char*)p + list);
    o.used = (uint32_t*)((char*)p + 2 * list);
    s.parts = (float*)((char*)p + 2 * list + 256);
    s.arrived = o.arrived = (uint32_t*)((char*)s.parts + parts);
    o.borders = blocks;
    int bits = 1;      // of the largest key, vocab
    while (bits < 32 && a.vocab >> bits) ++bits;
    o.passes = (bits + 8) / 9;
    o.digit = (bits + o.passes - 1) / o.passes;
    s.list = o.passes & 1 ? o.a : o.b;
    s.used = o.used;
    unsigned ctas = 1;
    while (ctas < 8 && (uint64_t)ctas * 1024 < a.tokens) ctas *= 2;
    const bool held = (uint64_t)ctas * kHeldEntries >= a.tokens;
    uint64_t fill = 0;
    if (!a.accumulate) {
        // While the tokens are sorted (10 to 20 us) there is time to clear some 40 MB, beginning with the last rows, which are the rarest; the
        // other rows are cleared while the sums are made.
        const uint64_t row = (uint64_t)a.dim * sizeof(T), room = (40u << 20) / row, rows = room < a.vocab ? (room ? room : 1) : a.vocab;
        o.dtable = (char*)a.dst;
        o.row_bytes = s.row_bytes = row;
        o.first_row = s.fill_rows = (uint32_t)(a.vocab - rows);
        while (o.group < 11 && row << (o.group + 1) <= 65536 && rows >> (o.group + 10)) ++o.group;
        const uint64_t groups = (rows + (1ull << o.group) - 1) >> o.group;
        while (o.shares < 8 && (1ull << o.shares) < groups && rows * row >> (o.shares + 14)) ++o.shares;      // from 16 KB each
        fill = ((1ull << o.shares) + ctas - 1) / ctas * ctas;
        while (1u << s.group < kMaxGroup && row << (s.group + 1) <= 131072) ++s.group;
        s.fills = (uint32_t)(((uint64_t)s.fill_rows + (1ull << s.group) - 1) >> s.group);
    }
    FG_REQUIRE(ctx, blocks + s.fills < (1ull << 31), "fg_embedding_bwd: tensor too large");
    s.blocks = (uint32_t)blocks;
    const size_t most = sizeof(uint32_t) * kSortWarps * kMaxBins + sizeof(uint2) * kHeldEntries, marks = kFillRows / 8;
    size_t bytes = (sizeof(uint32_t) * kSortWarps << o.digit) + (held ? sizeof(uint2) * kHeldEntries : 0);
    bytes = bytes < marks ? marks : bytes;
    static std::atomic<uint64_t> attr_done{0};      // one bit per device
    if (!(attr_done.load(std::memory_order_acquire) >> (ctx->device & 63) & 1ull)) {
        FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(embed_sort_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(embed_sort_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        attr_done.fetch_or(1ull << (ctx->device & 63), std::memory_order_release);
    }
    fg_launch_cluster(ctx, held ? embed_sort_kernel<true> : embed_sort_kernel<false>, (unsigned)(ctas + fill), kSortThreads, bytes, ctas, o);
    FG_LAUNCHED(ctx);
    fg_launch(ctx, add ? straight ? embed_sum_kernel<T, false, true> : embed_sum_kernel<T, true, true>
                       : straight ? embed_sum_kernel<T, false, false> : embed_sum_kernel<T, true, false>, (unsigned)(blocks + s.fills), 256, 0, s);
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
    FG_REQUIRE(ctx, !fg_ranges_meet(ids, 4ull * tokens, out, (uint64_t)tokens * dim * size), "fg_embedding_fwd: out overlaps ids");
    if (tokens == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, embed_fwd, ctx, EmbedArgs{tokens, vocab, dim, ids, table, scale, out, 0});
}

int32_t fg_embedding_bwd(fg_ctx* ctx, int32_t dtype, uint32_t tokens, uint32_t vocab, uint32_t dim, const uint32_t* ids, const void* dout,
                         float scale, void* dtable, int32_t accumulate) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_embedding_bwd: unknown dtype");
    FG_REQUIRE(ctx, ids && dout && dtable, "fg_embedding_bwd: NULL pointer");
    FG_REQUIRE(ctx, vocab >= 1 && dim >= 1, "fg_embedding_bwd: vocab and dim must be >= 1");
    FG_REQUIRE(ctx, tokens < (1u << 31) && (uint64_t)tokens * dim < (1ull << 40) && (uint64_t)vocab * dim < (1ull << 40),
               "fg_embedding_bwd: tensor too large");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(ids, 4) && fg_at_element(dout, size) && fg_at_element(dtable, size),
               "fg_embedding_bwd: a tensor does not start at an element");
    FG_REQUIRE(ctx, !fg_ranges_meet(dtable, (uint64_t)vocab * dim * size, dout, (uint64_t)tokens * dim * size), "fg_embedding_bwd: dtable overlaps dout");
    FG_REQUIRE(ctx, !fg_ranges_meet(ids, 4ull * tokens, dtable, (uint64_t)vocab * dim * size), "fg_embedding_bwd: dtable overlaps ids");
    if (tokens == 0) {      // empty sums
        if (!accumulate) FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(dtable, 0, (uint64_t)vocab * dim * size, ctx->stream));
        return FG_OK;
    }
    return FG_BY_DTYPE(dtype, embed_bwd, ctx, EmbedArgs{tokens, vocab, dim, ids, dout, scale, dtable, accumulate});
}

}  // extern "C"
