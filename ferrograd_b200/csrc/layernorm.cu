// Layer norm over the rows of a matrix, forward and backward.
//
// Forward: m = sum(x) / n; then, over d = x - m, r = sum(d) / n and q = sum(d * d) / n.  r is what rounding left of the mean, so the
// mean is m + r and the variance q - r * r: rows far from zero lose nothing to the subtraction.
// Backward, with h = (x - mean) * rstd and g = dy * gamma: dx = rstd * (g - mean(g) - h * mean(g * h)); dgamma and dbeta are column
// sums of dy * h and dy.
#include <atomic>

#include "rows.cuh"

namespace {

struct NormArgs {
    const void *x, *gamma, *beta;
    void* y;
    float *mean, *rstd;
    uint32_t rows, cols;
    float eps;
};
struct NormBwdArgs {
    const void *x, *dy, *gamma;
    const float *mean, *rstd;
    void *dx, *dgamma, *dbeta;
    uint32_t rows, cols;
    int accumulate_dx, accumulate_params;
};

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

template <typename C>
__global__ void __launch_bounds__(kMaxThreads, C::kTight && C::N <= 16 ? 2 : 1) norm_held_kernel(const NormArgs a, int threads) {
    using T = typename C::T;
    constexpr int H = C::N / 2;
    extern __shared__ uint4 shared[];
    __shared__ float red[kMaxGroups][4][32];
    fg_grid_enter();
    const Group group(threads);
    const uint32_t groups = blockDim.x / threads, step = gridDim.x * groups;
    const uint32_t first = C::kApart ? group.index * gridDim.x + blockIdx.x : blockIdx.x * groups + group.index;
    C columns(group, a.cols, first, shared);
    const float n = (float)a.cols, inv_n = 1.0f / n;
    const T *const gamma = static_cast<const T*>(a.gamma), *const beta = static_cast<const T*>(a.beta);
    typename C::Kept gammas, betas;
    if (gamma) columns.keep(gamma, gammas);
    if (beta) columns.keep(beta, betas);
    const uint64_t stride = (uint64_t)step * a.cols;
    const T *x = static_cast<const T*>(a.x) + (uint64_t)first * a.cols, *ahead = x;
    T* y = static_cast<T*>(a.y) + (uint64_t)first * a.cols;
    uint64_t next = first;      // the next row to ask for
    auto ask = [&] {
        if (next < a.rows) columns.ask(0, ahead);
        columns.asked();
        next += step;
        ahead += stride;
    };
    if (C::kAhead)
#pragma unroll
        for (int i = 0; i < C::kStages; ++i) ask();
    int turn = 0;
    for (uint64_t r = first; r < a.rows; r += step, x += stride, y += stride) {
        float2 v[H];
        columns.arrived();
        columns.get(0, x, v);
        columns.taken();
        if (C::kAhead) ask();
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < H; ++i) s = fg_add2(s, v[i]);
        const float m = group.sum(s.x + s.y, red[group.index][turn]) / n;
        const float2 less = make_float2(-m, -m);
#pragma unroll
        for (int i = 0; i < H; ++i) v[i] = fg_add2(v[i], less);
        columns.mask(v);
        float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
        for (int i = 0; i < H; ++i) {
            s1 = fg_add2(s1, v[i]);
            s2 = fg_fma2(v[i], v[i], s2);
        }
        const float2 t = group.sum(s1.x + s1.y, s2.x + s2.y, red[group.index][turn + 1]);
        const float rest = t.x * inv_n, rstd = 1.0f / sqrtf(fmaxf(__fmaf_rn(-rest, rest, t.y * inv_n), 0.0f) + a.eps);
        const float2 less_rest = make_float2(-rest, -rest), by = make_float2(rstd, rstd);
#pragma unroll
        for (int i = 0; i < H; ++i) v[i] = fg_mul2(fg_add2(v[i], less_rest), by);
        if (gamma) {
            float2 g[H];
            columns.kept(gammas, gamma, g);
#pragma unroll
            for (int i = 0; i < H; ++i) v[i] = fg_mul2(v[i], g[i]);
        }
        if (beta) {
            float2 b[H];
            columns.kept(betas, beta, b);
#pragma unroll
            for (int i = 0; i < H; ++i) v[i] = fg_add2(v[i], b[i]);
        }
        columns.store(y, v);
        if (group.thread == 0) {
            if (a.mean) a.mean[r] = m + rest;
            if (a.rstd) a.rstd[r] = rstd;
        }
        turn ^= 2;
    }
}

// The backward pass the same way, 16 columns at most per thread.  With the gradients of the parameters (kParams) a thread sums its columns
// over the rows of its group, a block adds its groups and leaves one row of parts: [block][2][pitch].
// With c = x - mean, dx = rstd * g + (-rstd * m1) + c * (-rstd^2 * m2), where m1 and m2 are the means of g and of g * h.
template <typename C, bool kParams>
__global__ void __launch_bounds__(kMaxThreads, C::kTight && C::N <= 4 ? 2 : 1) norm_bwd_held_kernel(const NormBwdArgs a, int threads, float* parts, uint32_t pitch) {
    using T = typename C::T;
    constexpr int H = C::N / 2;
    extern __shared__ uint4 shared[];      // the slots; at the end the groups' sums
    __shared__ float red[kMaxGroups][2][32];
    fg_grid_enter();
    const Group group(threads);
    const uint32_t groups = blockDim.x / threads, step = gridDim.x * groups;
    const uint32_t first = C::kApart ? group.index * gridDim.x + blockIdx.x : blockIdx.x * groups + group.index;
    C columns(group, a.cols, first, shared);
    const float inv_n = 1.0f / (float)a.cols;
    const T* const gamma = static_cast<const T*>(a.gamma);
    float2 gm[H];
    if (gamma) columns.parameter(gamma, gm);
    else
#pragma unroll
        for (int i = 0; i < H; ++i) gm[i] = make_float2(1.0f, 1.0f);
    const uint64_t stride = (uint64_t)step * a.cols, at = (uint64_t)first * a.cols;
    const T *x = static_cast<const T*>(a.x) + at, *dy = static_cast<const T*>(a.dy) + at, *x_ahead = x, *dy_ahead = dy;
    T* dx = a.dx ? static_cast<T*>(a.dx) + at : nullptr;
    uint64_t next = first;
    auto ask = [&] {
        if (next < a.rows) {
            columns.ask(0, x_ahead);
            columns.ask(1, dy_ahead);
        }
        columns.asked();
        next += step;
        x_ahead += stride;
        dy_ahead += stride;
    };
    if (C::kAhead)
#pragma unroll
        for (int i = 0; i < C::kStages; ++i) ask();
    float mean = 0.0f, rstd = 0.0f;
    if (first < a.rows) { mean = a.mean[first]; rstd = a.rstd[first]; }
    float2 dg[H], db[H];
#pragma unroll
    for (int i = 0; i < H; ++i) dg[i] = db[i] = make_float2(0.0f, 0.0f);
    int turn = 0;
    for (uint64_t r = first; r < a.rows; r += step, x += stride, dy += stride) {
        float2 c[H], g[H];
        const float sd = rstd;
        const float2 less = make_float2(-mean, -mean), by = make_float2(sd, sd);
        columns.arrived();
        columns.get(0, x, c);
        columns.get(1, dy, g);
        columns.taken();
        if (r + step < a.rows) { mean = a.mean[r + step]; rstd = a.rstd[r + step]; }
        if (C::kAhead) ask();
#pragma unroll
        for (int i = 0; i < H; ++i) c[i] = fg_add2(c[i], less);      // (columns that are not there: dy is zero)
        float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if (kParams) {
                dg[i] = fg_fma2(g[i], fg_mul2(c[i], by), dg[i]);
                db[i] = fg_add2(db[i], g[i]);
            }
            g[i] = fg_mul2(g[i], gm[i]);
            s1 = fg_add2(s1, g[i]);
            s2 = fg_fma2(g[i], c[i], s2);
        }
        if (dx) {
            const float2 t = group.sum(s1.x + s1.y, s2.x + s2.y, red[group.index][turn]);
            const float u1 = -sd * (t.x * inv_n), u2 = -sd * sd * (sd * (t.y * inv_n));
            const float2 add = make_float2(u1, u1), slope = make_float2(u2, u2);
#pragma unroll
            for (int i = 0; i < H; ++i) g[i] = fg_fma2(g[i], by, fg_fma2(c[i], slope, add));
            if (a.accumulate_dx) {
                columns.load(dx, c);
#pragma unroll
                for (int i = 0; i < H; ++i) g[i] = fg_add2(g[i], c[i]);
            }
            columns.store(dx, g);
            dx += stride;
        }
        turn ^= 1;
    }
    if constexpr (kParams) {
        float2* const sums = reinterpret_cast<float2*>(shared);      // the groups one after the other: [2][pair][thread]
        if (C::kAhead) fg_copies_wait<0>();
        for (uint32_t i = 0; i + 1 < groups; ++i) {
            __syncthreads();
            if (group.index == (int)i)
#pragma unroll
                for (int e = 0; e < H; ++e) {
                    float2 *const p = sums + e * threads + group.thread, *const q = p + H * threads;
                    *p = i ? fg_add2(*p, dg[e]) : dg[e];
                    *q = i ? fg_add2(*q, db[e]) : db[e];
                }
        }
        __syncthreads();
        if (group.index + 1 == (int)groups) {
            if (groups > 1)
#pragma unroll
                for (int e = 0; e < H; ++e) {
                    dg[e] = fg_add2(sums[e * threads + group.thread], dg[e]);
                    db[e] = fg_add2(sums[(H + e) * threads + group.thread], db[e]);
                }
            float* const mine = parts + (uint64_t)blockIdx.x * 2 * pitch;
            columns.store_sums(mine, dg);
            columns.store_sums(mine + pitch, db);
        }
    }
}

// Adds the blocks' parts: 128 columns per block, a warp takes every 32nd part.  pitch is a multiple of 128.
template <typename T>
__global__ void __launch_bounds__(1024) norm_parts_kernel(const NormBwdArgs a, const float* parts, uint32_t count, uint32_t pitch) {
    __shared__ float4 red[32][32];
    fg_grid_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t at = blockIdx.x * 128 + 4 * lane;      // dgamma's columns, then dbeta's
    T* const out = static_cast<T*>(at < pitch ? a.dgamma : a.dbeta);
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t i0 = warp; i0 < count; i0 += 32 * 8) {
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = i0 + 32 * j < count ? *reinterpret_cast<const float4*>(parts + (uint64_t)(i0 + 32 * j) * 2 * pitch + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 8; ++j) { s.x += v[j].x; s.y += v[j].y; s.z += v[j].z; s.w += v[j].w; }
    }
    red[warp][lane] = s;
    __syncthreads();
    if (threadIdx.x < 128) {
        const uint32_t c = blockIdx.x * 128 + threadIdx.x - (at < pitch ? 0 : pitch);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 32; ++w) sum += reinterpret_cast<const float*>(red[w])[threadIdx.x];
        if (out && c < a.cols) out[c] = fg_narrow<T>(a.accumulate_params ? fg_widen(out[c]) + sum : sum);
    }
}

// Any row: one block each, the row read once per sum.
template <typename T>
__global__ void __launch_bounds__(256) norm_stream_kernel(const NormArgs a) {
    __shared__ float red[64];
    fg_grid_enter();
    const float n = (float)a.cols;
    const T *gamma = static_cast<const T*>(a.gamma), *beta = static_cast<const T*>(a.beta);
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + (uint64_t)r * a.cols;
        T* y = static_cast<T*>(a.y) + (uint64_t)r * a.cols;
        float s = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) s += fg_widen(x[c]);
        const float m = fg_block_sum2(s, 0.0f, red).x / n;
        float s1 = 0.0f, s2 = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float d = fg_widen(x[c]) - m;
            s1 += d;
            s2 = __fmaf_rn(d, d, s2);
        }
        const float2 t = fg_block_sum2(s1, s2, red);
        const float rest = t.x / n, rstd = 1.0f / sqrtf(fmaxf(__fmaf_rn(-rest, rest, t.y / n), 0.0f) + a.eps);
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float h = ((fg_widen(x[c]) - m) - rest) * rstd;
            y[c] = fg_narrow<T>(__fmaf_rn(h, gamma ? fg_widen(gamma[c]) : 1.0f, beta ? fg_widen(beta[c]) : 0.0f));
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = m + rest;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_bwd_stream_kernel(const NormBwdArgs a) {
    __shared__ float red[64];
    fg_grid_enter();
    const float n = (float)a.cols;
    const T* gamma = static_cast<const T*>(a.gamma);
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const uint64_t at = (uint64_t)r * a.cols;
        const T *x = static_cast<const T*>(a.x) + at, *dy = static_cast<const T*>(a.dy) + at;
        T* dx = static_cast<T*>(a.dx) + at;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float g = fg_widen(dy[c]) * (gamma ? fg_widen(gamma[c]) : 1.0f);
            s1 += g;
            s2 = __fmaf_rn(g, (fg_widen(x[c]) - mean) * rstd, s2);
        }
        const float2 t = fg_block_sum2(s1, s2, red);
        const float m1 = t.x / n, m2 = t.y / n;
        for (uint64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
            const float g = fg_widen(dy[c]) * (gamma ? fg_widen(gamma[c]) : 1.0f), h = (fg_widen(x[c]) - mean) * rstd;
            const float v = rstd * __fmaf_rn(-h, m2, g - m1);
            dx[c] = fg_narrow<T>(a.accumulate_dx ? fg_widen(dx[c]) + v : v);
        }
    }
}

// Rows that are too long for a thread to keep its columns' sums beside them: the parameters' gradients first, by columns, over chunks of rows.
// A warp takes 32 columns, or as many packs of rows that lie straight, and every 8th row of the chunk.  part: [2][chunks][cols].
constexpr uint32_t kChunk = 256;
template <typename T, bool kPacked>
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormBwdArgs a, float* part) {
    constexpr int E = kPacked ? FgPack<T>::E : 1, kRows = 4;
    __shared__ float red[2][8][32][E];
    fg_grid_enter();
    const uint64_t c = ((uint64_t)blockIdx.x * 32 + threadIdx.x) * E, chunks = gridDim.y;
    const uint32_t r0 = blockIdx.y * kChunk, r1 = min(a.rows, r0 + kChunk);
    const T *const x = static_cast<const T*>(a.x) + c, *const dy = static_cast<const T*>(a.dy) + c;
    float s1[E] = {}, s2[E] = {};
    if (c < a.cols)
        for (uint32_t r = r0 + threadIdx.y; r < r1; r += 8 * kRows) {
            float u[kRows][E], v[kRows][E], mean[kRows], rstd[kRows];
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                const uint32_t row = r + 8 * j;
                const bool there = row < r1;
                mean[j] = there ? a.mean[row] : 0.0f;
                rstd[j] = there ? a.rstd[row] : 0.0f;
                if constexpr (kPacked) {
                    FgPack<T>::widen(there ? *reinterpret_cast<const uint4*>(x + (uint64_t)row * a.cols) : make_uint4(0, 0, 0, 0), u[j]);
                    FgPack<T>::widen(there ? *reinterpret_cast<const uint4*>(dy + (uint64_t)row * a.cols) : make_uint4(0, 0, 0, 0), v[j]);
                } else {
                    u[j][0] = there ? fg_widen(x[(uint64_t)row * a.cols]) : 0.0f;
                    v[j][0] = there ? fg_widen(dy[(uint64_t)row * a.cols]) : 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < kRows; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    s1[e] = __fmaf_rn(v[j][e], (u[j][e] - mean[j]) * rstd[j], s1[e]);
                    s2[e] += v[j][e];
                }
        }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        red[0][threadIdx.y][threadIdx.x][e] = s1[e];
        red[1][threadIdx.y][threadIdx.x][e] = s2[e];
    }
    __syncthreads();
    if (threadIdx.y < 2 && c < a.cols)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += red[threadIdx.y][i][threadIdx.x][e];
            part[(threadIdx.y * chunks + blockIdx.y) * a.cols + c + e] = s;
        }
}
template <typename T>
__global__ void __launch_bounds__(256) norm_fold_kernel(const NormBwdArgs a, const float* part, uint32_t chunks) {
    fg_grid_enter();
    const uint64_t c = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    T* out = static_cast<T*>(blockIdx.y == 0 ? a.dgamma : a.dbeta);
    if (c >= a.cols || !out) return;
    part += (uint64_t)blockIdx.y * chunks * a.cols;
    float s = 0.0f;
    for (uint32_t i = 0; i < chunks; ++i) s += part[(uint64_t)i * a.cols + c];
    out[c] = fg_narrow<T>(a.accumulate_params ? fg_widen(out[c]) + s : s);
}

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

template <typename C>
int32_t launch_held(fg_ctx* ctx, const NormArgs& a, HeldPlan p) {
    static std::atomic<uint64_t> done{0};
    const int32_t s = allow_shared(ctx, done, norm_held_kernel<C>, p.bytes);
    if (s != FG_OK) return s;
    fg_launch(ctx, norm_held_kernel<C>, p.grid, p.threads * p.groups, p.bytes, a, p.threads);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T, int kPacks>
int32_t launch_straight(fg_ctx* ctx, const NormArgs& a, HeldPlan p) {
    return p.full ? launch_held<Straight<T, kPacks, true, 1>>(ctx, a, p) : launch_held<Straight<T, kPacks, false, 1>>(ctx, a, p);
}
template <typename T>
int32_t norm_fwd(fg_ctx* ctx, const NormArgs& a) {
    constexpr int usual = 16 / FgPack<T>::E;      // 16 columns a thread
    if (fg_rows_lie_straight(a.cols, sizeof(T), a.x, a.y, a.gamma, a.beta)) {
        const HeldPlan p = held_plan(ctx, a.rows, a.cols / FgPack<T>::E, 1, usual, 8, 1, 512);
        if (p.threads)
            return p.units == 1 ? launch_straight<T, 1>(ctx, a, p) : p.units == 2 ? launch_straight<T, 2>(ctx, a, p)
                   : p.units == 4 ? launch_straight<T, 4>(ctx, a, p) : launch_straight<T, 8>(ctx, a, p);
    } else {
        // Rows that a warp holds by four elements a lane (eight of f32) are faster so: 20000 x 81 bf16 7.0 us against 9.6, 20000 x 201 f32 10.3 against 11.0.
        if (a.cols > 64 * sizeof(T) && fg_aligned16(a.x) && fg_aligned16(a.y)) {
            constexpr int most = 32 / FgPack<T>::E;      // a bit per column of a thread
            const HeldPlan p = shifted_plan<T>(ctx, a.rows, a.cols, 1, usual, most, 1);
            if (p.threads)
                return p.units == 1 ? launch_held<Shifted<T, 1, 1>>(ctx, a, p) : p.units == 2 ? launch_held<Shifted<T, 2, 1>>(ctx, a, p)
                       : p.units == 4 ? launch_held<Shifted<T, 4, 1>>(ctx, a, p) : launch_held<Shifted<T, most, 1>>(ctx, a, p);
        }
        HeldPlan p = held_plan(ctx, a.rows, a.cols, 4, 8, 32, 0, 1024);
        if (p.threads)
            return p.units == 4 ? launch_held<Ragged<T, 4, 1>>(ctx, a, p) : p.units == 8 ? launch_held<Ragged<T, 8, 1>>(ctx, a, p)
                   : p.units == 16 ? launch_held<Ragged<T, 16, 1>>(ctx, a, p) : launch_held<Ragged<T, 32, 1>>(ctx, a, p);
    }
    fg_launch(ctx, norm_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

template <typename C, bool kParams>
int32_t launch_bwd(fg_ctx* ctx, const NormBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch) {
    const size_t sums = kParams && p.groups > 1 ? 8ull * C::N * p.threads : 0, bytes = p.bytes < sums ? sums : p.bytes;
    static std::atomic<uint64_t> done{0};
    const int32_t s = allow_shared(ctx, done, norm_bwd_held_kernel<C, kParams>, bytes);
    if (s != FG_OK) return s;
    fg_launch(ctx, norm_bwd_held_kernel<C, kParams>, p.grid, p.threads * p.groups, bytes, a, p.threads, parts, pitch);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename C>
int32_t launch_bwd_held(fg_ctx* ctx, const NormBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch) {
    return parts ? launch_bwd<C, true>(ctx, a, p, parts, pitch) : launch_bwd<C, false>(ctx, a, p, parts, pitch);
}
template <typename T, int kPacks>
int32_t launch_bwd_straight(fg_ctx* ctx, const NormBwdArgs& a, HeldPlan p, float* parts, uint32_t pitch) {
    return p.full ? launch_bwd_held<Straight<T, kPacks, true, 2>>(ctx, a, p, parts, pitch) : launch_bwd_held<Straight<T, kPacks, false, 2>>(ctx, a, p, parts, pitch);
}

template <typename T>
int32_t norm_bwd(fg_ctx* ctx, const NormBwdArgs& a) {
    constexpr int usual = 16 / FgPack<T>::E;
    const bool straight = fg_rows_lie_straight(a.cols, sizeof(T), a.x, a.dy, a.gamma, a.dx);
    HeldPlan p{};
    if (straight) p = held_plan(ctx, a.rows, a.cols / FgPack<T>::E, 1, usual, usual, 2, 512);
    else if (fg_aligned16(a.x) && fg_aligned16(a.dy) && fg_aligned16(a.dx)) p = shifted_plan<T>(ctx, a.rows, a.cols, 1, usual, usual, 2);
    const bool shifted = !straight && p.threads;
    if (!straight && !shifted) p = held_plan(ctx, a.rows, a.cols, 4, 4, 16, 0, 1024);
    if (p.threads) {
        float* parts = nullptr;
        const uint32_t pitch = (a.cols + 127) / 128 * 128;
        if (a.dgamma || a.dbeta) {
            void* w;
            const int32_t s = fg_ws_alloc(ctx, 8ull * pitch * p.grid, &w);
            if (s != FG_OK) return s;
            parts = (float*)w;
        }
        int32_t s;
        if (straight) {
            if (p.units == 1) s = launch_bwd_straight<T, 1>(ctx, a, p, parts, pitch);
            else if (p.units == 2) s = launch_bwd_straight<T, 2>(ctx, a, p, parts, pitch);
            else s = launch_bwd_straight<T, usual>(ctx, a, p, parts, pitch);
        } else if (shifted) {
            if (p.units == 1) s = launch_bwd_held<Shifted<T, 1, 2>>(ctx, a, p, parts, pitch);
            else if (p.units == 2) s = launch_bwd_held<Shifted<T, 2, 2>>(ctx, a, p, parts, pitch);
            else s = launch_bwd_held<Shifted<T, usual, 2>>(ctx, a, p, parts, pitch);
        } else if (p.units == 4) s = launch_bwd_held<Ragged<T, 4, 2>>(ctx, a, p, parts, pitch);
        else if (p.units == 8) s = launch_bwd_held<Ragged<T, 8, 2>>(ctx, a, p, parts, pitch);
        else s = launch_bwd_held<Ragged<T, 16, 2>>(ctx, a, p, parts, pitch);
        if (s != FG_OK || !parts) return s;
        fg_launch(ctx, norm_parts_kernel<T>, pitch / 64, 1024, 0, a, (const float*)parts, (uint32_t)p.grid, pitch);
        FG_LAUNCHED(ctx);
        return FG_OK;
    }
    if (a.dgamma || a.dbeta) {      // before dx, which may be dy or x
        const uint32_t chunks = (a.rows + kChunk - 1) / kChunk, E = straight ? FgPack<T>::E : 1;
        void* w;
        const int32_t s = fg_ws_alloc(ctx, 8ull * chunks * a.cols, &w);
        if (s != FG_OK) return s;
        fg_launch(ctx, straight ? norm_columns_kernel<T, true> : norm_columns_kernel<T, false>, dim3((unsigned)(((uint64_t)a.cols + 32 * E - 1) / (32 * E)), chunks), dim3(32, 8), 0, a, (float*)w);
        FG_LAUNCHED(ctx);
        fg_launch(ctx, norm_fold_kernel<T>, dim3((unsigned)(((uint64_t)a.cols + 255) / 256), 2), 256, 0, a, (const float*)w, chunks);
        FG_LAUNCHED(ctx);
    }
    if (!a.dx) return FG_OK;
    // dx alone leaves a thread room for 32 columns.
    const HeldPlan q = straight ? held_plan(ctx, a.rows, a.cols / FgPack<T>::E, 2 * usual, 2 * usual, 2 * usual, 2, 512) : HeldPlan{};
    if (q.threads) return launch_bwd<Straight<T, 2 * usual, false, 2>, false>(ctx, a, q, nullptr, 0);
    if (!straight && fg_aligned16(a.x) && fg_aligned16(a.dy) && fg_aligned16(a.dx)) {
        const HeldPlan w = shifted_plan<T>(ctx, a.rows, a.cols, 2 * usual, 2 * usual, 2 * usual, 2);
        if (w.threads) return launch_bwd<Shifted<T, 2 * usual, 2>, false>(ctx, a, w, nullptr, 0);
    }
    const HeldPlan e = straight ? HeldPlan{} : held_plan(ctx, a.rows, a.cols, 32, 32, 32, 0, 512);
    if (e.threads) return launch_bwd<Ragged<T, 32, 2>, false>(ctx, a, e, nullptr, 0);
    fg_launch(ctx, norm_bwd_stream_kernel<T>, rows_grid(ctx, a.rows), 256, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

}  // namespace

extern "C" {

int32_t fg_layernorm_fwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* x, const void* gamma, const void* beta,
                         float eps, void* y, float* mean_out, float* rstd_out) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_layernorm_fwd: unknown dtype");
    FG_REQUIRE(ctx, x && y, "fg_layernorm_fwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1, "fg_layernorm_fwd: cols must be >= 1");
    FG_REQUIRE(ctx, eps >= 0.0f && eps <= 3.402823466e38f, "fg_layernorm_fwd: eps must be a number >= 0");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_layernorm_fwd: tensor too large");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(x, size) && fg_at_element(y, size) && fg_at_element(gamma, size) && fg_at_element(beta, size) &&
                        fg_at_element(mean_out, 4) && fg_at_element(rstd_out, 4), "fg_layernorm_fwd: a tensor does not start at an element");
    const uint64_t bytes = (uint64_t)rows * cols * size;
    FG_REQUIRE(ctx, y == x || !fg_ranges_meet(x, bytes, y, bytes), "fg_layernorm_fwd: y overlaps x but is not x");
    const uint64_t line = (uint64_t)cols * size;
    FG_REQUIRE(ctx, !fg_ranges_meet(y, bytes, gamma, line) && !fg_ranges_meet(y, bytes, beta, line), "fg_layernorm_fwd: y overlaps gamma or beta");
    const uint64_t column = 4ull * rows;
    for (const void* out : {(const void*)mean_out, (const void*)rstd_out})
        FG_REQUIRE(ctx, !fg_ranges_meet(out, column, x, bytes) && !fg_ranges_meet(out, column, y, bytes) && !fg_ranges_meet(out, column, gamma, line) &&
                            !fg_ranges_meet(out, column, beta, line), "fg_layernorm_fwd: statistics overlap another tensor");
    FG_REQUIRE(ctx, !fg_ranges_meet(mean_out, column, rstd_out, column), "fg_layernorm_fwd: mean_out overlaps rstd_out");
    if (rows == 0) return FG_OK;
    return FG_BY_DTYPE(dtype, norm_fwd, ctx, NormArgs{x, gamma, beta, y, mean_out, rstd_out, rows, cols, eps});
}

int32_t fg_layernorm_bwd(fg_ctx* ctx, int32_t dtype, uint32_t rows, uint32_t cols, const void* x, const void* dy, const void* gamma,
                         const float* mean, const float* rstd, void* dx, void* dgamma, void* dbeta, int32_t accumulate_dx,
                         int32_t accumulate_params) {
    FG_ENTER(ctx);
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "fg_layernorm_bwd: unknown dtype");
    FG_REQUIRE(ctx, x && dy && mean && rstd, "fg_layernorm_bwd: NULL pointer");
    FG_REQUIRE(ctx, cols >= 1, "fg_layernorm_bwd: cols must be >= 1");
    FG_REQUIRE(ctx, (uint64_t)rows * cols < (1ull << 40), "fg_layernorm_bwd: tensor too large");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(x, size) && fg_at_element(dy, size) && fg_at_element(gamma, size) && fg_at_element(dx, size) &&
                        fg_at_element(dgamma, size) && fg_at_element(dbeta, size) && fg_at_element(mean, 4) && fg_at_element(rstd, 4),
               "fg_layernorm_bwd: a tensor does not start at an element");
    FG_REQUIRE(ctx, dx || dgamma || dbeta, "fg_layernorm_bwd: no output");
    FG_REQUIRE(ctx, !accumulate_dx || (dx != dy && dx != x), "fg_layernorm_bwd: accumulate_dx needs a dx of its own");
    const uint64_t bytes = (uint64_t)rows * cols * size;
    FG_REQUIRE(ctx, (dx == x || !fg_ranges_meet(x, bytes, dx, bytes)) && (dx == dy || !fg_ranges_meet(dy, bytes, dx, bytes)),
               "fg_layernorm_bwd: dx overlaps x or dy but is neither");
    const uint64_t line = (uint64_t)cols * size;
    FG_REQUIRE(ctx, !fg_ranges_meet(dx, bytes, gamma, line), "fg_layernorm_bwd: dx overlaps gamma");
    for (const void* out : {dgamma, dbeta})
        FG_REQUIRE(ctx, !fg_ranges_meet(out, line, x, bytes) && !fg_ranges_meet(out, line, dy, bytes) && !fg_ranges_meet(out, line, gamma, line) &&
                            !fg_ranges_meet(out, line, dx, bytes), "fg_layernorm_bwd: a parameter's gradient overlaps another tensor");
    FG_REQUIRE(ctx, !fg_ranges_meet(dgamma, line, dbeta, line), "fg_layernorm_bwd: dgamma overlaps dbeta");
    const uint64_t column = 4ull * rows;
    for (const void* in : {(const void*)mean, (const void*)rstd})
        FG_REQUIRE(ctx, !fg_ranges_meet(in, column, dx, bytes) && !fg_ranges_meet(in, column, dgamma, line) && !fg_ranges_meet(in, column, dbeta, line),
                   "fg_layernorm_bwd: a gradient overlaps the statistics");
    if (rows == 0) {      // empty sums
        if (dgamma && !accumulate_params) FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(dgamma, 0, (uint64_t)cols * size, ctx->stream));
        if (dbeta && !accumulate_params) FG_CUDA(ctx, FG_ERR_FAILED_BUFFER_COPY, cudaMemsetAsync(dbeta, 0, (uint64_t)cols * size, ctx->stream));
        return FG_OK;
    }
    return FG_BY_DTYPE(dtype, norm_bwd, ctx,
                       NormBwdArgs{x, dy, gamma, mean, rstd, dx, dgamma, dbeta, rows, cols, accumulate_dx, accumulate_params});
}

}  // extern "C"
