// Rows that a group of threads holds: what the norms' kernels share.
#pragma once
#include <atomic>

#include "rows.cuh"

namespace {

// ---- rows that a group of threads holds ----
// A group of warps takes a row at a time, a thread the same columns of each.  What bounds these kernels beside the memory is instructions:
// 400 to 600 per warp and row of 16 columns a thread in a first form, most of them addresses and zeros for columns that are not there,
// so rows that fill their threads have code of their own (kFull), two f32 operations go in one instruction and the two sums of a
// row share their shuffles.
constexpr int kMaxGroups = 8, kMaxThreads = 512;
struct Group {
    int index, threads, thread, warps, warp, lane;      // of the block's groups; a group's threads; within the group
    __device__ __forceinline__ explicit Group(int threads_) : threads(threads_) {
        warps = threads >> 5;
        index = (threadIdx.x >> 5) / warps;
        thread = threadIdx.x - index * threads;
        warp = thread >> 5;
        lane = threadIdx.x & 31;
    }
    // The sum of a in lanes 0 to 15, of b in 16 to 31.
    __device__ __forceinline__ float halves(float a, float b) const {
        const float mine = lane < 16 ? a : b, other = lane < 16 ? b : a;
        float v = mine + __shfl_xor_sync(0xffffffffu, other, 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    // Two sums over the group, in all of its threads.  `red` is the group's [32] floats, others from one call to the next; 16 warps at most.
    __device__ __forceinline__ float2 sum(float a, float b, float* red) const {
        float v = halves(a, b);
        if (warps > 1) {
            if ((lane & 15) == 0) red[lane + warp] = v;
            fg_group_barrier(index, threads);
            v = (lane & 15) < warps ? red[lane] : 0.0f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        }
        return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
    }
    __device__ __forceinline__ float max(float a, float* red) const {      // of numbers >= 0
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (warps == 1) return a;
        if (lane == 0) red[warp] = a;
        fg_group_barrier(index, threads);
        a = (lane & 15) < warps ? red[lane & 15] : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        return a;
    }
    __device__ __forceinline__ float sum(float a, float* red) const {
        a = fg_warp_sum(a);
        if (warps == 1) return a;
        if (lane == 0) red[warp] = a;
        fg_group_barrier(index, threads);
        a = (lane & 15) < warps ? red[lane & 15] : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        return a;
    }
};

// Rows that lie straight: a thread has packs `thread`, `thread` + threads, ... of 16 bytes, asked for one to four rows ahead by asynchronous
// copies into slots of shared memory that are the thread's own.
__host__ __device__ constexpr int stages_of(int packs) { return packs > 8 ? 1 : packs > 4 ? 3 : 4; }      // by the packs of all tensors in a stage: 512 threads fit
template <typename T_, int kPacks, bool kFull, int kTensors>
struct Straight {
    using T = T_;
    static constexpr int E = FgPack<T>::E, P = E / 2, N = kPacks * E, kStages = stages_of(kTensors * kPacks);
    static constexpr bool kAhead = true, kTight = false, kApart = false;
    uint32_t slots, block, offset, pitch, have;      // shared address of the thread's first slot, bytes of a block's packs, of the thread, of a group's packs
    uint32_t put = 0, take = 0;                      // stages
    __device__ __forceinline__ Straight(const Group& g, uint32_t cols, uint32_t, const void* shared) {
        slots = (uint32_t)__cvta_generic_to_shared(shared) + threadIdx.x * 16;
        block = blockDim.x * 16;
        offset = g.thread * 16;
        pitch = g.threads * 16;
        const uint32_t packs = cols / E;
        have = (uint32_t)g.thread < packs ? min((uint32_t)kPacks, (packs - g.thread + g.threads - 1) / g.threads) : 0;
    }
    __device__ __forceinline__ bool has(int k) const { return kFull || k < have; }
    __device__ __forceinline__ uint32_t slot(uint32_t stage, int t, int k) const { return slots + ((stage * kTensors + t) * kPacks + k) * block; }
    __device__ __forceinline__ void ask(int t, const T* row) {
        const char* const p = reinterpret_cast<const char*>(row) + offset;
#pragma unroll
        for (int k = 0; k < kPacks; ++k)
            if (has(k)) fg_copy_async(slot(put, t, k), p + k * pitch);
    }
    __device__ __forceinline__ void asked() {
        fg_copies_end();
        put = put == kStages - 1 ? 0 : put + 1;
    }
    __device__ __forceinline__ void arrived() const { fg_copies_wait<kStages - 1>(); }
    __device__ __forceinline__ void taken() { take = take == kStages - 1 ? 0 : take + 1; }
    __device__ __forceinline__ void spread(int k, const uint4& w, float2* v) const {
        float2 x[P];
        FgPack<T>::widen(w, x);
#pragma unroll
        for (int e = 0; e < P; ++e) v[k * P + e] = has(k) ? x[e] : make_float2(0.0f, 0.0f);
    }
    __device__ __forceinline__ void get(int t, const T*, float2 (&v)[N / 2]) const {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) spread(k, fg_load_shared(slot(take, t, k)), v);
    }
    __device__ __forceinline__ void load(const T* row, float2 (&v)[N / 2]) const {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (has(k)) w = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row) + offset + k * pitch);
            spread(k, w, v);
        }
    }
    __device__ __forceinline__ void parameter(const T* p, float2 (&v)[N / 2]) const { load(p, v); }
    // A parameter's columns, kept for all rows (of up to 4 packs: read from the L1 and, where slots leave it little room, from the L2 for every
    // row, they cost a fifth of the time).
    static constexpr bool kKeep = kPacks <= 4;
    struct Kept { uint4 w[kKeep ? kPacks : 1]; };
    __device__ __forceinline__ void keep(const T* p, Kept& kept) const {
        if (!kKeep) return;
#pragma unroll
        for (int k = 0; k < (kKeep ? kPacks : 0); ++k) {
            kept.w[k] = make_uint4(0, 0, 0, 0);
            if (has(k)) kept.w[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) + offset + k * pitch);
        }
    }
    __device__ __forceinline__ void kept(const Kept& kept, const T* p, float2 (&v)[N / 2]) const {
        if constexpr (kKeep) {
#pragma unroll
            for (int k = 0; k < kPacks; ++k) spread(k, kept.w[k], v);
        } else load(p, v);
    }
    __device__ __forceinline__ void mask(float2 (&v)[N / 2]) const {      // columns that are not there count for nothing
        if (!kFull)
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (!has(i / P)) v[i] = make_float2(0.0f, 0.0f);
    }
    __device__ __forceinline__ void store(T* row, const float2 (&v)[N / 2]) const {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            float2 x[P];
#pragma unroll
            for (int e = 0; e < P; ++e) x[e] = v[k * P + e];
            if (has(k)) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(row) + offset + k * pitch) = FgPack<T>::narrow(x);
        }
    }
    __device__ __forceinline__ void store_sums(float* row, const float2 (&v)[N / 2]) const {
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
            if (has(i / P)) *reinterpret_cast<float2*>(row + (offset + (i / P) * pitch) / sizeof(T) + 2 * (i % P)) = v[i];
    }
};

// Rows of any length in tensors that start on 16-byte boundaries.  The distance of a row's start from a boundary comes back every E rows at the
// latest, so if the rows of a group, and of all groups of a block, lie a multiple of that apart (kApart: they are a grid apart), it is one number
// for them, and the thread's words hold the same columns of every row.  The words at a row's ends are shared with other rows.
// Against single elements, forward and backward, us: 4099 x 1001 f16 9.4 and 14.2 (10.3 and 18.0), 30000 x 777 f16 34.5 and 49.1 (53.6 and
// 72.1), 3000 x 5001 f32 35.9 and 45.5 (73.6 and 162), 10000 x 4097 bf16 80.6 and 91.9 (137 and 178), 3000 x 12001 f32 120 and 178
// (210 and 223).  What is over the time of rows that lie straight (30000 x 776: 24.7 and 41.8) are the ends: the warps that have one mask it
// and store it by elements (a lane per element was no faster).
template <typename T_, int kPacks, int kTensors>
struct Shifted {
    using T = T_;
    static constexpr int E = FgPack<T>::E, P = E / 2, N = kPacks * E, kStages = stages_of(kTensors * kPacks);
    static constexpr bool kAhead = true, kTight = false, kApart = true;
    static constexpr uint32_t kAll = N == 32 ? ~0u : (1u << (N & 31)) - 1, kWord = (1u << E) - 1;
    uint32_t slots, block, pitch, valid = 0, tail, tail_bytes;      // valid: a bit per element that belongs to the row; tail: which pack is the row's last word
    uint32_t head[4];                                               // what the first pack has of the row
    int32_t column;                                                 // of the first element; negative where it belongs to the row before
    uint32_t put = 0, take = 0;
    __device__ __forceinline__ Shifted(const Group& g, uint32_t cols, uint32_t first, const void* shared) {
        slots = (uint32_t)__cvta_generic_to_shared(shared) + threadIdx.x * 16;
        block = blockDim.x * 16;
        pitch = g.threads * E;
        const uint32_t off = (uint32_t)((uint64_t)first * cols % E), last = (off + cols - 1) / E;
        column = (int32_t)(g.thread * E) - (int32_t)off;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            const uint32_t w = g.thread + k * g.threads;
            uint32_t bits = w > last ? 0 : w == last ? (2u << ((off + cols - 1) & (E - 1))) - 1 : kWord;
            if (w == 0) bits &= ~((1u << off) - 1);
            valid |= bits << (k * E);
        }
        tail = last % g.threads == (uint32_t)g.thread ? last / g.threads : kPacks;
        tail_bytes = (((off + cols - 1) & (E - 1)) + 1) * sizeof(T);
        const uint32_t cut = g.thread == 0 ? off * sizeof(T) : 0;      // bytes of the row before
#pragma unroll
        for (int i = 0; i < 4; ++i) head[i] = cut <= 4 * i ? ~0u : cut >= 4 * i + 4 ? 0u : 0xffff0000u;
#pragma unroll
        for (int k = 0; k < kPacks; ++k)
            if (!has(k))
                for (int i = 0; i < kStages * kTensors; ++i) fg_store_shared(slots + (i * kPacks + k) * block, make_uint4(0, 0, 0, 0));
    }
    __device__ __forceinline__ bool has(int k) const { return valid >> (k * E) & kWord; }
    __device__ __forceinline__ bool whole(int k) const { return (valid >> (k * E) & kWord) == kWord; }
    __device__ __forceinline__ bool bit(int i) const { return valid >> i & 1u; }
    __device__ __forceinline__ uint32_t slot(uint32_t stage, int t, int k) const { return slots + ((stage * kTensors + t) * kPacks + k) * block; }
    __device__ __forceinline__ void ask(int t, const T* row) {      // nothing behind the row, which may be the tensor's last
        const T* const p = row + column;
#pragma unroll
        for (int k = 0; k < kPacks; ++k)
            if (has(k)) fg_copy_async(slot(put, t, k), p + k * pitch, (uint32_t)k == tail ? tail_bytes : 16);
    }
    __device__ __forceinline__ void asked() {
        fg_copies_end();
        put = put == kStages - 1 ? 0 : put + 1;
    }
    __device__ __forceinline__ void arrived() const { fg_copies_wait<kStages - 1>(); }
    __device__ __forceinline__ void taken() { take = take == kStages - 1 ? 0 : take + 1; }
    __device__ __forceinline__ void spread(const uint4& w, int k, float2 (&v)[N / 2]) const {
        float2 x[P];
        FgPack<T>::widen(w, x);
#pragma unroll
        for (int e = 0; e < P; ++e) v[k * P + e] = x[e];
    }
    __device__ __forceinline__ void mask(float2 (&v)[N / 2]) const {
        if (valid != kAll)      // the ends of rows
#pragma unroll
            for (int k = 0; k < kPacks; ++k)
                if (!whole(k))
#pragma unroll
                    for (int i = k * P; i < (k + 1) * P; ++i) v[i] = make_float2(bit(2 * i) ? v[i].x : 0.0f, bit(2 * i + 1) ? v[i].y : 0.0f);
    }
    __device__ __forceinline__ void get(int t, const T*, float2 (&v)[N / 2]) const {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {      // zero outside of the row: packs and parts of packs behind it never arrive
            uint4 w = fg_load_shared(slot(take, t, k));
            if (k == 0) w = make_uint4(w.x & head[0], w.y & head[1], w.z & head[2], w.w & head[3]);
            spread(w, k, v);
        }
    }
    __device__ __forceinline__ void elements(const T* p, int k, float2 (&v)[N / 2]) const {      // p: the pack's first
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float x = bit(k * E + e) ? fg_widen(p[e]) : 0.0f;
            if (e & 1) v[k * P + e / 2].y = x;
            else v[k * P + e / 2].x = x;
        }
    }
    __device__ __forceinline__ void load(const T* row, float2 (&v)[N / 2]) const {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            const T* const p = row + column + (int64_t)(k * pitch);
            if (whole(k)) spread(*reinterpret_cast<const uint4*>(p), k, v);
            else elements(p, k, v);
        }
    }
    // Parameters lie as they like; of up to 4 packs they are read once.
    __device__ __forceinline__ void parameter(const T* p, float2 (&v)[N / 2]) const {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) elements(p + column + (int64_t)(k * pitch), k, v);
    }
    static constexpr bool kKeep = kPacks <= 4;
    struct Kept { uint4 w[kKeep ? kPacks : 1]; };
    __device__ __forceinline__ void keep(const T* p, Kept& kept) const {
        if constexpr (kKeep) {
            float2 v[N / 2];
            parameter(p, v);
#pragma unroll
            for (int k = 0; k < kPacks; ++k) kept.w[k] = pack(v, k);
        }
    }
    __device__ __forceinline__ void kept(const Kept& kept, const T* p, float2 (&v)[N / 2]) const {
        if constexpr (kKeep) {
#pragma unroll
            for (int k = 0; k < kPacks; ++k) spread(kept.w[k], k, v);
        } else parameter(p, v);
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&v)[N / 2], int k) {
        float2 x[P];
#pragma unroll
        for (int e = 0; e < P; ++e) x[e] = v[k * P + e];
        return FgPack<T>::narrow(x);
    }
    __device__ __forceinline__ void store(T* row, const float2 (&v)[N / 2]) const {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
            T* const p = row + column + (int64_t)(k * pitch);
            if (whole(k)) *reinterpret_cast<uint4*>(p) = pack(v, k);
            else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (bit(k * E + e)) p[e] = fg_narrow<T>(e & 1 ? v[k * P + e / 2].y : v[k * P + e / 2].x);
        }
    }
    __device__ __forceinline__ void store_sums(float* row, const float2 (&v)[N / 2]) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (bit(i)) row[column + (int64_t)((i / E) * pitch) + i % E] = i & 1 ? v[i / 2].y : v[i / 2].x;
    }
};

// Any other row (tensors off 16-byte boundaries, and short rows forward): a thread has the elements `thread`, `thread` + threads, ... of it.
template <typename T_, int kCount, int kTensors>
struct Ragged {
    using T = T_;
    static constexpr int N = kCount, kStages = 1;
    static constexpr bool kAhead = kTensors * kCount <= 8;       // the next row's elements are on their way, in registers
    static constexpr bool kTight = kCount <= 8, kApart = false;  // kTight: 64 registers, for 1024 threads an SM
    uint32_t thread, threads, cols;
    T next[kAhead ? kTensors : 1][kAhead ? N : 1];
    __device__ __forceinline__ Ragged(const Group& g, uint32_t cols_, uint32_t, const void*) : thread(g.thread), threads(g.threads), cols(cols_) {}
    __device__ __forceinline__ void ask(int t, const T* row) {
        if constexpr (kAhead)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t c = thread + i * threads;
                next[t][i] = c < cols ? row[c] : fg_narrow<T>(0.0f);
            }
    }
    __device__ __forceinline__ void asked() {}
    __device__ __forceinline__ void arrived() const {}
    __device__ __forceinline__ void taken() {}
    __device__ __forceinline__ void get(int t, const T* row, float2 (&v)[N / 2]) const {
        if constexpr (kAhead) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) v[i] = make_float2(fg_widen(next[t][2 * i]), fg_widen(next[t][2 * i + 1]));
        } else load(row, v);
    }
    __device__ __forceinline__ void load(const T* row, float2 (&v)[N / 2]) const {
        T w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = thread + i * threads;
            w[i] = c < cols ? row[c] : fg_narrow<T>(0.0f);
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = make_float2(fg_widen(w[2 * i]), fg_widen(w[2 * i + 1]));
    }
    __device__ __forceinline__ void parameter(const T* p, float2 (&v)[N / 2]) const { load(p, v); }
    static constexpr bool kKeep = kCount <= 16;
    struct Kept { T w[kKeep ? N : 1]; };
    __device__ __forceinline__ void keep(const T* p, Kept& kept) const {
#pragma unroll
        for (int i = 0; i < (kKeep ? N : 0); ++i) {
            const uint32_t c = thread + i * threads;
            kept.w[i] = c < cols ? p[c] : fg_narrow<T>(0.0f);
        }
    }
    __device__ __forceinline__ void kept(const Kept& kept, const T* p, float2 (&v)[N / 2]) const {
        if constexpr (kKeep) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) v[i] = make_float2(fg_widen(kept.w[2 * i]), fg_widen(kept.w[2 * i + 1]));
        } else load(p, v);
    }
    __device__ __forceinline__ void mask(float2 (&v)[N / 2]) const {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if (thread + 2 * i * threads >= cols) v[i].x = 0.0f;
            if (thread + (2 * i + 1) * threads >= cols) v[i].y = 0.0f;
        }
    }
    template <typename U>
    __device__ __forceinline__ void put(U* row, const float2 (&v)[N / 2]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = thread + i * threads;
            if (c < cols) row[c] = fg_narrow<U>(i & 1 ? v[i / 2].y : v[i / 2].x);
        }
    }
    __device__ __forceinline__ void store(T* row, const float2 (&v)[N / 2]) const { put(row, v); }
    __device__ __forceinline__ void store_sums(float* row, const float2 (&v)[N / 2]) const { put(row, v); }
};

int rows_grid(const fg_ctx* ctx, uint32_t rows) { return (int)(rows < 8u * ctx->sm_count ? rows : 8u * ctx->sm_count); }

// How a kernel that holds rows is launched: a thread's packs (or elements, of ragged rows), the threads of a group, the groups of a block, the
// bytes of its slots, the blocks; threads = 0: not at all.
struct HeldPlan { int units, threads, groups; bool full; size_t bytes; int grid; };
// How many units a thread holds: `least`, doubled (to `most` at most) while the row would take more threads than are good for it.  us, forward of
// bf16 unless said otherwise, by packs:
//   two rows per SM or fewer      512 (a block): more threads answer sooner (296 x 4096 backward 8.9 by 1, 12.0 by 2; forward 64 x 1024 1.8 and 1.9,
//                                 but 296 x 4096 3.4 and 2.7)
//   below `usual`                 32 (a warp): its sums need no barrier, and less of a row is instructions (16384 x 512 7.7 by 2, 12.9 by 1; 600 x 4096
//                                 4.4 and 6.0; f32 16384 x 4096 82 to 86 by 4, 118 by 2), but no more than a warp is for (16384 x 256 5.8 by 1, 8.7 by 2)
//   2 packs, and 4 make a warp    32 (16384 x 1024 11.0 by 4, 16.5 by 2)
//   2 packs, longer rows          256: an SM has two rows to switch between then (7000 x 8192 44.1 by 4, 61.8 by 2)
//   4 packs and more              512: registers hold no more (f32 16384 x 4096 82 by 4, 101 by 8; 7000 x 12288 75 by 4, 68 by 8)
int units_of(uint64_t units, bool many, int least, int usual, int most) {
    int each = least;
    while (each < most) {
        const uint32_t enough = !many || (each >= usual && each >= 4) ? kMaxThreads : each < usual || units <= 128 ? 32 : 256;
        if (units <= (uint64_t)enough * each) break;
        each *= 2;
    }
    return each;
}
// A block has 256 threads or, for a longer row, up to 512.  `resident`: threads that an SM has registers for, at the usual units.
HeldPlan held_plan(const fg_ctx* ctx, uint32_t rows, uint64_t units, int least, int usual, int most, int tensors, int resident) {
    HeldPlan p{units_of(units, rows > 2u * ctx->sm_count, least, usual, most), 0, 1, false, 0, 0};
    if (units > (uint64_t)kMaxThreads * p.units) return p;
    p.threads = (int)((units + 32 * p.units - 1) / (32 * p.units) * 32);
    p.full = units == (uint64_t)p.threads * p.units;
    p.groups = 256 / p.threads < 1 ? 1 : 256 / p.threads;
    while (p.groups > 1 && (uint64_t)rows * 2 <= (uint64_t)p.groups * ctx->sm_count) p.groups /= 2;      // few rows: over the SMs first
    p.bytes = sizeof(uint4) * stages_of(tensors * p.units) * tensors * p.units * p.threads * p.groups;
    // What the SMs hold at once: threads by their registers, 220 KB with the static part.
    const uint64_t by_threads = (p.units <= usual ? resident : kMaxThreads) / (p.threads * p.groups), by_memory = 220 * 1024 / (p.bytes + 5 * 1024),
                   per_sm = by_threads < by_memory ? by_threads : by_memory;
    const uint64_t need = ((uint64_t)rows + p.groups - 1) / p.groups, cap = (uint64_t)ctx->sm_count * (per_sm ? per_sm : 1);
    p.grid = (int)(need < cap ? need : cap);
    return p;
}
// The same for rows that begin anywhere in a word: a grid of as many blocks as bring a row's start back to its place in one.
template <typename T>
HeldPlan shifted_plan(const fg_ctx* ctx, uint32_t rows, uint32_t cols, int least, int usual, int most, int tensors) {
    constexpr uint32_t E = FgPack<T>::E;
    HeldPlan p = held_plan(ctx, rows, ((uint64_t)cols + 2 * E - 2) / E, least, usual, most, tensors, 512);
    if (!p.threads) return p;
    int period = 1;
    while ((uint64_t)period * cols % E) period *= 2;
    const bool all = (uint64_t)p.grid * p.groups >= rows;      // a row each: some blocks more
    p.grid = (p.grid + (all ? period - 1 : 0)) / period * period;
    if (p.grid == 0) p.grid = period;
    return p;
}
// More shared memory than a kernel may have by default, once per kernel (`done`) and device.
template <typename K>
int32_t allow_shared(fg_ctx* ctx, std::atomic<uint64_t>& done, K kernel, size_t bytes) {
    if (bytes <= 32 * 1024 || done.load(std::memory_order_acquire) >> (ctx->device & 63) & 1ull) return FG_OK;
    FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 * 1024));
    done.fetch_or(1ull << (ctx->device & 63), std::memory_order_release);
    return FG_OK;
}

}  // namespace
