// Attention over packed sequences with grouped heads, forward and backward: the entry points, and the kernels for f32 and for 16-bit tensors that the tensor
// cores do not take as they lie.
//
// Forward, per head: s_ij = scale * q_i . k_j for the keys j that row i sees, o_i = sum_j p_ij v_j with p_ij = exp(s_ij - m) / l, where m is the
// largest s_ij and l the sum of exp(s_ij - m).  One pass over the keys: when a tile of keys raises m, what was summed so far is multiplied by
// exp(old m - new m).  Exponents are powers of two (s * log2 e).  lse_i = m + log l is what the backward pass takes.
// Backward, with delta_i = dout_i . out_i: p_ij = exp(s_ij - lse_i); ds_ij = p_ij * (dout_i . v_j - delta_i); dq_i = scale * sum_j ds_ij k_j;
// dk_j = scale * sum_i ds_ij q_i; dv_j = sum_i p_ij dout_i.  A block has a tile of rows and goes over their keys for dq, or a tile of keys and goes over
// their rows, those of all heads of the group, for dk and dv: nothing is added atomically, so the order of sums is fixed.
#include <atomic>

#include "attention_tc.cuh"

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxDim = 256;
template <typename T> constexpr int32_t dtype_of = sizeof(T) == 4 ? FG_DTYPE_F32 : std::is_same_v<T, __half> ? FG_DTYPE_F16 : FG_DTYPE_BF16;

// Is x a number that stays one when it is rounded to 11 bits, as the products on the tensor cores below take it?
__device__ __forceinline__ bool has_halves(float x) { return fabsf(x) < __uint_as_float(0x7f7ff000u); }
// Was there one that is not, among those met (or a number within a thousandth of the largest)?  kByProduct: by two products, in a pipe that the gradients' kernels have room in, instead of a
// comparison (4000 tokens of 128 columns, all pairs: 6628 us and 6885; forward 4096 tokens, 8 heads: 1345 and 1315).
template <bool kByProduct>
struct Odd {
    float z = 0.0f;
    bool any = false;
    __device__ __forceinline__ void meet(float x) {
        if (kByProduct) z = __fmaf_rn(x * 1.001f, 0.0f, z);
        else any |= !has_halves(x);
    }
    __device__ __forceinline__ explicit operator bool() const { return kByProduct ? z != z : any; }
};

// ---- plain FMAs: few rows, and head_dim over 128 forward ----
// Threads are 16 x 16: thread (y, x) has rows y * RT .. and keys x, x + 16, .. of a tile's scores, and the same rows by columns 4 x .. + 64 j of a sum.  Rows of a tile are (query, head of the group) pairs, so the heads of a group share the keys' tile.
// Rows in shared memory are f32, padded by four words: 16 threads that read 16 bytes each of 16 rows take two passes, the least for 256 bytes.
// Rows [first, first + n) of a tensor's `dim` columns into shared memory, zeros behind the last row and column.  Has this thread met a number that has no usual halves?
template <typename T, int kRows, int DM, int kWarps = kThreads / 32, bool kByProduct = false, typename F>
__device__ __forceinline__ bool fetch(float* to, uint32_t n, uint32_t dim, F row) {
    constexpr int kPitch = DM + 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Odd<kByProduct> odd;
#pragma unroll 8
    for (int r = warp; r < kRows; r += kWarps) {
        const T* p = (uint32_t)r < n ? row((uint32_t)r) : nullptr;
#pragma unroll
        for (int c = 0; c < DM; c += 32) {
            const float x = p && (uint32_t)(c + lane) < dim ? fg_widen(p[c + lane]) : 0.0f;
            to[r * kPitch + c + lane] = x;
            odd.meet(x);
        }
    }
    return (bool)odd;
}
// RT x CT products of rows of two tiles: a's rows a0 + i, b's rows b0 + 16 * j.
template <int RT, int CT, int DM>
__device__ __forceinline__ void dots(const float* a, const float* b, uint32_t dim, int a0, int b0, float (&s)[RT][CT]) {
    constexpr int kPitch = DM + 4;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) s[i][j] = 0.0f;
#pragma unroll 4
    for (uint32_t d = 0; d < dim; d += 4) {
        float4 x[RT], y[CT];
#pragma unroll
        for (int i = 0; i < RT; ++i) x[i] = *reinterpret_cast<const float4*>(a + (a0 + i) * kPitch + d);
#pragma unroll
        for (int j = 0; j < CT; ++j) y[j] = *reinterpret_cast<const float4*>(b + (b0 + 16 * j) * kPitch + d);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < CT; ++j)
                s[i][j] = __fmaf_rn(x[i].w, y[j].w, __fmaf_rn(x[i].z, y[j].z, __fmaf_rn(x[i].y, y[j].y, __fmaf_rn(x[i].x, y[j].x, s[i][j]))));
    }
}
// acc[i] += w_i * row of b: one row of b's columns 4 x .. + 64 j.
template <int RT, int DM>
__device__ __forceinline__ void add_row(const float* b, int x, const float (&w)[RT], float4 (&acc)[RT][DM / 64]) {
#pragma unroll
    for (int j = 0; j < DM / 64; ++j) {
        const float4 v = *reinterpret_cast<const float4*>(b + 4 * x + 64 * j);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            acc[i][j].x = __fmaf_rn(w[i], v.x, acc[i][j].x);
            acc[i][j].y = __fmaf_rn(w[i], v.y, acc[i][j].y);
            acc[i][j].z = __fmaf_rn(w[i], v.z, acc[i][j].z);
            acc[i][j].w = __fmaf_rn(w[i], v.w, acc[i][j].w);
        }
    }
}
template <int DM>
__device__ __forceinline__ void put_row(float* to, int x, uint32_t dim, const float4 (&v)[DM / 64], float by) {
#pragma unroll
    for (int j = 0; j < DM / 64; ++j) {
        const float e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if ((uint32_t)(4 * x + 64 * j + c) < dim) to[4 * x + 64 * j + c] = e[c] * by;
    }
}
template <typename T, int DM>
__device__ __forceinline__ void put_row(T* to, int x, uint32_t dim, const float4 (&v)[DM / 64], float by) {
#pragma unroll
    for (int j = 0; j < DM / 64; ++j) {
        const float e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if ((uint32_t)(4 * x + 64 * j + c) < dim) to[4 * x + 64 * j + c] = fg_narrow<T>(e[c] * by);
    }
}
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// ---- f32 products on the tensor cores ----
// An f32 number is the sum of two tf32 numbers of 11 bits and 2^-22 of itself, and x y = hi hi + hi lo + lo hi within 3 * 2^-22 |x y|: three
// instructions of 16 x 8 x 8 products, whose sums are f32.  The instruction cuts what it adds to its sums, always towards zero, so every three start at
// zero and are added in plain f32 (a chain of them over a tile was three times as far off: 1.0e-6 of the gradients of 501 tokens, 3.4e-7 like this, for a
// twentieth of the gradients' time).
// kAny: x may be NaN, an infinity or a number that rounds to one.  The first two are their own high half and have no other, so that they meet the other side's number once, whole
// (half of an infinity times a low half of the other sign would be no number, nor would it be times a half that is zero); the last is cut.  NaN is written anew:
// added to, its bits could become those of a zero.  Tiles that hold such a number are known when they are fetched, and only those are multiplied in this way.
struct Tf32 { uint32_t hi, lo, cross; };      // cross: what meets the other side's low half
template <bool kAny>
__device__ __forceinline__ Tf32 tf32_halves(float x) {
    const uint32_t bits = __float_as_uint(x);
    if (kAny && !has_halves(x)) {
        const bool number = fabsf(x) < INFINITY;
        const uint32_t hi = number ? bits & 0xffffe000u : x != x ? 0x7fffe000u : bits;
        return Tf32{hi, number ? __float_as_uint(x - __uint_as_float(hi)) : 0u, number ? hi : 0u};
    }
    const uint32_t hi = (bits + 0x1000u) & 0xffffe000u;
    return Tf32{hi, __float_as_uint(x - __uint_as_float(hi)) + 0x1000u, hi};
}
__device__ __forceinline__ void mma_16x8x8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool kAny>
struct Left {      // a 16 x 8 block in halves: lane l has rows l / 4 and 8 more, columns l % 4 and 4 more
    uint32_t hi[4], lo[4], cross[4];
    __device__ __forceinline__ Left(float a0, float a1, float a2, float a3) {
        const float x[4] = {a0, a1, a2, a3};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Tf32 t = tf32_halves<kAny>(x[i]);
            hi[i] = t.hi;
            lo[i] = t.lo;
            cross[i] = t.cross;
        }
    }
    __device__ __forceinline__ void times(float b0, float b1, float (&d)[4]) const {
        const Tf32 x = tf32_halves<kAny>(b0), y = tf32_halves<kAny>(b1);
        float f[4] = {};
        mma_16x8x8(f, lo, x.cross, y.cross);
        mma_16x8x8(f, cross, x.lo, y.lo);
        mma_16x8x8(f, hi, x.hi, y.hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] += f[e];
    }
};
// 16 rows of a by 8 * NT rows of b, over dim columns (zeros behind): lane l has rows l / 4, + 8 and columns 8 t + 2 (l % 4), + 1.
template <bool kAny, int NT, int DM>
__device__ __forceinline__ void row_products(const float* a, const float* b, uint32_t dim, float (&s)[NT][4]) {
    constexpr int kPitch = DM + 4;
    const int g = (threadIdx.x & 31) >> 2, q = threadIdx.x & 3;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.0f;
#pragma unroll 2
    for (uint32_t d = q; d < dim + q; d += 8) {
        const float* const x = a + g * kPitch + d;
        const Left<kAny> left(x[0], x[8 * kPitch], x[4], x[8 * kPitch + 4]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float* const y = b + (8 * t + g) * kPitch + d;
            left.times(y[0], y[4], s[t]);
        }
    }
}
// acc += (16 x 8 * steps block given by `left`) times rows of b: 8 * NT columns of it from b on.
template <bool kAny, int NT, int DM, typename F>
__device__ __forceinline__ void add_products(F left, const float* b, int steps, float (&acc)[NT][4]) {
    constexpr int kPitch = DM + 4, kOnce = NT < 4 ? NT : 4;
    const int g = (threadIdx.x & 31) >> 2, q = threadIdx.x & 3;
#pragma unroll
    for (int t0 = 0; t0 < NT; t0 += kOnce)
#pragma unroll 2
        for (int k = 0; k < steps; ++k) {
            const Left<kAny> x = left(k);
            const float* const y = b + (8 * k + q) * kPitch + 8 * t0 + g;
#pragma unroll
            for (int t = 0; t < kOnce; ++t) x.times(y[8 * t], y[4 * kPitch + 8 * t], acc[t0 + t]);
        }
}
// The lane's columns of a row (e0 = 0: row l / 4; 2: the one 8 below) to memory.
template <typename T, int NT>
__device__ __forceinline__ void put_columns(T* to, int c0, uint32_t dim, const float (&v)[NT][4], int e0, float by) {
    const int c = c0 + 2 * (threadIdx.x & 3);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if ((uint32_t)(c + 8 * t) < dim) to[c + 8 * t] = fg_narrow<T>(v[t][e0] * by);
        if ((uint32_t)(c + 8 * t + 1) < dim) to[c + 8 * t + 1] = fg_narrow<T>(v[t][e0 + 1] * by);
    }
}
// Which query and head of the group rows of a tile are: one 64-bit division for a tile, a 32-bit one for a row.
struct RowPlace {
    uint32_t i0, g0, group;
    __device__ __forceinline__ RowPlace(uint64_t first, uint32_t group_) : group(group_) {
        i0 = (uint32_t)(first / group_);
        g0 = (uint32_t)(first - (uint64_t)i0 * group_);
    }
    __device__ __forceinline__ uint32_t query(uint32_t r) const { return group == 1 ? i0 + r : i0 + (g0 + r) / group; }
    __device__ __forceinline__ uint32_t head(uint32_t r) const { return group == 1 ? 0 : (g0 + r) % group; }
};

constexpr int kKeys = 64;
constexpr size_t rows_bytes(int rt, int dm) { return sizeof(float) * ((size_t)(16 * rt + 2 * kKeys) * (dm + 4) + 16 * rt * (kKeys + 4)); }
template <typename T, int RT, int DM>
__global__ void __launch_bounds__(kThreads) attn_rows_kernel(const FgAttnArgs a) {
    constexpr int R = 16 * RT, kPitch = DM + 4, kP = kKeys + 4;
    extern __shared__ float shared[];
    float *const qs = shared, *const ks = qs + R * kPitch, *const vs = ks + kKeys * kPitch, *const ps = vs + kKeys * kPitch;
    fg_grid_enter();
    uint32_t tile;
    const int b = fg_attn_find(a.q_starts, a.sequences, a.queries, a.group, R, gridDim.x - 1 - blockIdx.x, &tile);
    if (b < 0) return;
    const FgAttnSeq s(a, b);
    const uint64_t rows = (uint64_t)s.nq * a.group, first = (uint64_t)tile * R;
    if (first >= rows) return;
    const uint32_t n = rows - first < R ? (uint32_t)(rows - first) : R, kv = blockIdx.y, dim = a.dim;
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const T *const q = static_cast<const T*>(a.q), *const k = static_cast<const T*>(a.k) + (uint64_t)s.k0 * a.k_stride + (uint64_t)kv * dim,
                  *const v = static_cast<const T*>(a.v) + (uint64_t)s.k0 * a.v_stride + (uint64_t)kv * dim;
    const RowPlace place(first, a.group);
    fetch<T, R, DM>(qs, n, dim, [&](uint32_t r) { return q + (uint64_t)(s.q0 + place.query(r)) * a.q_stride + (uint64_t)(kv * a.group + place.head(r)) * dim; });
    uint32_t seen[RT];
    float top[RT], sum[RT];
    float4 acc[RT][DM / 64];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const uint32_t r = y * RT + i;
        seen[i] = r < n ? s.seen(a, place.query(r)) : 0;
        top[i] = -INFINITY;
        sum[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < DM / 64; ++j) acc[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    uint32_t lo, hi;
    if (!s.share(a, blockIdx.z, &lo, &hi)) return;
    hi = min(hi, s.seen(a, place.query(n - 1)));
    const float by = a.scale * kFgLog2e;
    for (uint32_t j0 = lo; j0 < hi; j0 += kKeys) {
        const uint32_t there = min((uint32_t)kKeys, s.nk - j0);
        __syncthreads();
        fetch<T, kKeys, DM>(ks, there, dim, [&](uint32_t r) { return k + (uint64_t)(j0 + r) * a.k_stride; });
        fetch<T, kKeys, DM>(vs, there, dim, [&](uint32_t r) { return v + (uint64_t)(j0 + r) * a.v_stride; });
        __syncthreads();
        float p[RT][4], fade[RT];
        dots<RT, 4, DM>(qs, ks, dim, y * RT, x, p);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t key = j0 + x + 16 * j;
                p[i][j] = key < seen[i] && key < hi ? p[i][j] * by : -INFINITY;
                most = fmaxf(most, p[i][j]);
            }
            most = fmaxf(half_warp_max(most), top[i]);
            const float base = most == -INFINITY ? 0.0f : most, less = fg_ex2_fast(top[i] - base);
            float l = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[i][j] = fg_ex2_fast(p[i][j] - base);
                l += p[i][j];
                ps[(y * RT + i) * kP + x + 16 * j] = p[i][j];
            }
            top[i] = most;
            sum[i] = __fmaf_rn(sum[i], less, half_warp_sum(l));
            fade[i] = less;
        }
        __syncwarp();
        float4 of_tile[RT][DM / 64];      // (added key by key to the sums of a long share: 4.7e-7 off at 3400 keys instead of 2.9e-7)
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < DM / 64; ++j) of_tile[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int c = 0; c < kKeys; c += 4) {
            float4 w[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) w[i] = *reinterpret_cast<const float4*>(ps + (y * RT + i) * kP + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float u[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) u[i] = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
                add_row<RT, DM>(vs + (c + e) * kPitch, x, u, of_tile);
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < DM / 64; ++j) {
                const float4 t = of_tile[i][j];
                float4& o = acc[i][j];
                o = make_float4(__fmaf_rn(o.x, fade[i], t.x), __fmaf_rn(o.y, fade[i], t.y), __fmaf_rn(o.z, fade[i], t.z), __fmaf_rn(o.w, fade[i], t.w));
            }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const uint32_t r = y * RT + i;
        if (r >= n) continue;
        const uint32_t row = s.q0 + place.query(r), head = kv * a.group + place.head(r);
        const uint64_t line = (uint64_t)row * a.heads + head;
        if (a.splits > 1) {
            const uint64_t part = (uint64_t)blockIdx.z * a.queries * a.heads + line;
            put_row<DM>(a.part_out + part * dim, x, dim, acc[i], 1.0f);
            if (x == 0) a.part_stat[part] = make_float2(top[i], sum[i]);
        } else {
            put_row<T, DM>(static_cast<T*>(a.out) + line * dim, x, dim, acc[i], sum[i] == 0.0f ? 0.0f : 1.0f / sum[i]);
            if (x == 0 && a.lse) a.lse[(uint64_t)head * a.queries + row] = (top[i] + __log2f(sum[i])) * kFgLn2;
        }
    }
}

// Many rows: a warp has 16 of a block's 128, and all keys of a tile.  The weights of a tile stay in registers as the left side of the product with v: the lane that has the
// scores of keys 2 (l % 4) and + 1 takes them for columns l % 4 and + 4, with v's rows in that order.
template <bool kAny, int NT, int NS, int DM>
__device__ __forceinline__ void add_weighted(const float (&p)[NT][4], const float* vs, float (&acc)[NS][4]) {
    constexpr int kPitch = DM + 4;
    const int g = (threadIdx.x & 31) >> 2, q = threadIdx.x & 3;
    // (sums of a tile's own: added straight to the rows' sums, 4096 tokens took 1838 us instead of 1686)
#pragma unroll
    for (int t0 = 0; t0 < NS; t0 += 4) {
        float f[4][4] = {};
#pragma unroll
        for (int k = 0; k < NT; ++k) {
            const Left<kAny> x(p[k][0], p[k][2], p[k][1], p[k][3]);
            const float* const y = vs + (8 * k + 2 * q) * kPitch + 8 * t0 + g;
#pragma unroll
            for (int t = 0; t < 4; ++t) x.times(y[8 * t], y[kPitch + 8 * t], f[t]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t0 + t][e] += f[t][e];
    }
}
// The products of tiles with odd numbers are functions of their own: inlined beside the usual ones, they took 4096 tokens of 128 columns from 1315 to 1407 us.  (What a function gets the
// address of does not stay in registers, so it is a copy.)
template <int N, int M>
__device__ __forceinline__ void copy(float (&to)[N][M], const float (&from)[N][M]) {
#pragma unroll
    for (int i = 0; i < N * M; ++i) to[i / M][i % M] = from[i / M][i % M];
}
template <int NT, int DM>
__noinline__ __device__ void odd_row_products(const float* a, const float* b, uint32_t dim, float (&s)[NT][4]) { row_products<true, NT, DM>(a, b, dim, s); }
template <int NT, int NS, int DM>
__noinline__ __device__ void odd_add_weighted(const float (&p)[NT][4], const float* vs, float (&acc)[NS][4]) { add_weighted<true, NT, NS, DM>(p, vs, acc); }
constexpr size_t many_bytes(int dm) { return sizeof(float) * (size_t)(128 + 2 * kKeys) * (dm + 4); }
template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) attn_many_kernel(const FgAttnArgs a) {
    constexpr int R = 128, kPitch = DM + 4, NT = kKeys / 8, NS = DM / 8;
    extern __shared__ float shared[];
    float *const qs = shared, *const ks = qs + R * kPitch, *const vs = ks + kKeys * kPitch;
    fg_grid_enter();
    uint32_t tile;
    const int b = fg_attn_find(a.q_starts, a.sequences, a.queries, a.group, R, gridDim.x - 1 - blockIdx.x, &tile);
    if (b < 0) return;
    const FgAttnSeq s(a, b);
    const uint64_t rows = (uint64_t)s.nq * a.group, first = (uint64_t)tile * R;
    if (first >= rows) return;
    const uint32_t n = rows - first < R ? (uint32_t)(rows - first) : R, kv = blockIdx.y, dim = a.dim, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint32_t block = (threadIdx.x >> 5) * 16;
    const T *const qp = static_cast<const T*>(a.q), *const kp = static_cast<const T*>(a.k) + (uint64_t)s.k0 * a.k_stride + (uint64_t)kv * dim,
                  *const vp = static_cast<const T*>(a.v) + (uint64_t)s.k0 * a.v_stride + (uint64_t)kv * dim;
    const RowPlace place(first, a.group);
    const bool odd_rows = fetch<T, R, DM>(qs, n, dim, [&](uint32_t r) { return qp + (uint64_t)(s.q0 + place.query(r)) * a.q_stride + (uint64_t)(kv * a.group + place.head(r)) * dim; });
    uint32_t seen[2];
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f}, acc[NS][4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) seen[h] = block + g + 8 * h < n ? s.seen(a, place.query(block + g + 8 * h)) : 0;
    const uint32_t hi = s.seen(a, place.query(n - 1));
    const float by = a.scale * kFgLog2e;
    for (uint32_t j0 = 0; j0 < hi; j0 += kKeys) {
        const uint32_t there = min((uint32_t)kKeys, s.nk - j0);
        __syncthreads();
        const bool odd_keys = fetch<T, kKeys, DM>(ks, there, dim, [&](uint32_t r) { return kp + (uint64_t)(j0 + r) * a.k_stride; });
        const bool odd_values = fetch<T, kKeys, DM>(vs, there, dim, [&](uint32_t r) { return vp + (uint64_t)(j0 + r) * a.v_stride; });
        const bool odd = __syncthreads_or(odd_rows | odd_keys | odd_values);
        float p[NT][4];
        if (odd) {
            float x[NT][4];
            odd_row_products<NT, DM>(qs + block * kPitch, ks, dim, x);
            copy(p, x);
        } else row_products<false, NT, DM>(qs + block * kPitch, ks, dim, p);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float most = -INFINITY;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 2 * h; e < 2 * h + 2; ++e) {
                    p[t][e] = j0 + 8 * t + 2 * q + (e & 1) < seen[h] ? p[t][e] * by : -INFINITY;
                    most = fmaxf(most, p[t][e]);
                }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2)), top[h]);
            const float base = most == -INFINITY ? 0.0f : most, less = fg_ex2_fast(top[h] - base);
            top[h] = most;
            sum[h] *= less;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 2 * h; e < 2 * h + 2; ++e) {
                    p[t][e] = fg_ex2_fast(p[t][e] - base);
                    sum[h] += p[t][e];
                }
#pragma unroll
            for (int t = 0; t < NS; ++t) { acc[t][2 * h] *= less; acc[t][2 * h + 1] *= less; }
        }
        // (A weight that is no number makes its row's sum none, and that the row, whatever its products are.)
        if (odd) {
            float w[NT][4], o[NS][4];
            copy(w, p);
            copy(o, acc);
            odd_add_weighted<NT, NS, DM>(w, vs, o);
            copy(acc, o);
        } else add_weighted<false, NT, NS, DM>(p, vs, acc);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        const uint32_t r = block + g + 8 * h;
        if (r >= n) continue;
        const uint32_t row = s.q0 + place.query(r), head = kv * a.group + place.head(r);
        put_columns<T, NS>(static_cast<T*>(a.out) + ((uint64_t)row * a.heads + head) * dim, 0, dim, acc, 2 * h, sum[h] == 0.0f ? 0.0f : 1.0f / sum[h]);
        if (q == 0 && a.lse) a.lse[(uint64_t)head * a.queries + row] = (top[h] + __log2f(sum[h])) * kFgLn2;
    }
}

// Shares of the keys joined: four warps a row (a query's head), each with every fourth share; the same numbering of rows as the kernel before it, 2 rows
// a block.  All of a warp's loads are independent of one another (128 shares of a row one after the other took 50 us).
constexpr uint32_t kMaxSplits = 128, kJoinRows = 2, kJoinWarps = 4;
template <typename T>
__global__ void __launch_bounds__(kThreads) attn_join_kernel(const FgAttnArgs a) {
    __shared__ float sums[kJoinRows][kJoinWarps][kMaxDim];
    fg_grid_enter();
    uint32_t tile;
    const int b = fg_attn_find(a.q_starts, a.sequences, a.queries, a.heads, kJoinRows, blockIdx.x, &tile);
    if (b < 0) return;
    const FgAttnSeq s(a, b);
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp / kJoinWarps, part = warp % kJoinWarps;
    const uint64_t at = (uint64_t)tile * kJoinRows + mine;
    const bool there = at < (uint64_t)s.nq * a.heads;
    const uint32_t row = s.q0 + (uint32_t)(at / a.heads), head = (uint32_t)(at % a.heads), splits = s.shares(a);
    const uint64_t line = (uint64_t)row * a.heads + head, pitch = (uint64_t)a.queries * a.heads;
    float2 st[kMaxSplits / 32];
    float top = -INFINITY, sum = 0.0f, acc[kMaxDim / 32];
#pragma unroll
    for (int i = 0; i < (int)kMaxSplits / 32; ++i) {
        const uint32_t z = lane + 32 * i;
        st[i] = there && z < splits ? a.part_stat[z * pitch + line] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, st[i].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < (int)kMaxSplits / 32; ++i) {
        st[i].x = st[i].y == 0.0f ? 0.0f : fg_ex2_fast(st[i].x - base);      // the share's factor; a share that saw nothing has none
        sum = __fmaf_rn(st[i].x, st[i].y, sum);
    }
    sum = fg_warp_sum(sum);
#pragma unroll
    for (int c = 0; c < (int)kMaxDim / 32; ++c) acc[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < (int)kMaxSplits / 32; ++i) {
        if (32u * i >= splits) break;
#pragma unroll 4
        for (uint32_t l = part; l < 32; l += kJoinWarps) {
            const float w = __shfl_sync(0xffffffffu, st[i].x, l);
            const float* const p = a.part_out + ((32 * i + l) * pitch + line) * a.dim;
            if (there && w != 0.0f)
#pragma unroll
                for (int c = 0; c < (int)kMaxDim / 32; ++c)
                    if (lane + 32 * c < a.dim) acc[c] = __fmaf_rn(w, __ldcg(p + lane + 32 * c), acc[c]);
        }
    }
#pragma unroll
    for (int c = 0; c < (int)kMaxDim / 32; ++c)
        if (lane + 32 * c < a.dim) sums[mine][part][lane + 32 * c] = acc[c];
    __syncthreads();
    if (!there) return;
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* const out = static_cast<T*>(a.out) + line * a.dim;
    for (uint32_t d = part * 32 + lane; d < a.dim; d += 32 * kJoinWarps) {
        float v = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kJoinWarps; ++w) v += sums[mine][w][d];
        out[d] = fg_narrow<T>(v * by);
    }
    if (part == 0 && lane == 0 && a.lse) a.lse[(uint64_t)head * a.queries + row] = (top + __log2f(sum)) * kFgLn2;
}

// delta_i = dout_i . out_i, a warp per row; [heads][queries].
template <typename T>
__global__ void __launch_bounds__(kThreads) attn_delta_kernel(const T* out, const T* dout, float* delta, uint32_t queries, uint32_t heads, uint32_t dim) {
    fg_grid_enter();
    const uint64_t line = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (line >= (uint64_t)queries * heads) return;
    const uint32_t lane = threadIdx.x & 31;
    float s = 0.0f;
    for (uint32_t d = lane; d < dim; d += 32) s = __fmaf_rn(fg_widen(out[line * dim + d]), fg_widen(dout[line * dim + d]), s);
    s = fg_warp_sum(s);
    if (lane == 0) delta[(line % heads) * queries + line / heads] = s;
}

constexpr size_t bwd_bytes(int dm, int n) { return sizeof(float) * (4 * (size_t)n * (dm + 4) + 2 * n * (n + 4) + 2 * n); }
// The weights and the gradients of the scores of a tile of rows and keys, in shared memory by row.
// A block of 64 rows and 64 keys of 128 columns has an SM to itself, and 16 warps: 4000 tokens, 8 heads over one, all pairs, 6578 us (a tenth more with 8).
constexpr int bwd_warps(int dm, int n) { return dm == 128 && n == 64 ? 16 : 8; }
// Blocks that an SM has registers for.  (32 rows of 64 columns: four, with some registers spilled, take 501 tokens 53.5 us instead of 50.4, and 1900 tokens 460 instead of 474.)
constexpr int bwd_blocks(int dm, int n) { return dm == 64 && n == 32 ? 3 : dm == 64 || n == 32 ? 2 : 1; }
template <typename T, int DM, int N_>
struct BwdTile {
    static constexpr int N = N_, kWarps = bwd_warps(DM, N), kPitch = DM + 4, kP = N + 4;
    float *qs, *dos, *ks, *vs, *ps, *ds, *stat;      // stat: lse in powers of two, delta
    __device__ __forceinline__ explicit BwdTile(float* shared) {
        qs = shared;
        dos = qs + N * kPitch;
        ks = dos + N * kPitch;
        vs = ks + N * kPitch;
        ps = vs + N * kPitch;
        ds = ps + N * kP;
        stat = ds + N * kP;
    }
    // Both, like fetch(), say whether this thread has met a number that has no usual halves.
    __device__ __forceinline__ bool keys(const FgAttnArgs& a, const FgAttnSeq& s, uint32_t kv, uint32_t j0) {
        const uint32_t n = s.nk - j0;
        const bool odd = fetch<T, N, DM, kWarps, true>(ks, n, a.dim, [&](uint32_t r) { return static_cast<const T*>(a.k) + (uint64_t)(s.k0 + j0 + r) * a.k_stride + (uint64_t)kv * a.dim; });
        return odd | fetch<T, N, DM, kWarps, true>(vs, n, a.dim, [&](uint32_t r) { return static_cast<const T*>(a.v) + (uint64_t)(s.k0 + j0 + r) * a.v_stride + (uint64_t)kv * a.dim; });
    }
    __device__ __forceinline__ bool rows(const FgAttnArgs& a, const FgAttnSeq& s, uint32_t kv, const RowPlace& at, uint32_t n) {
        auto place = [&](uint32_t r, uint32_t* i, uint32_t* head) {
            *i = s.q0 + at.query(r);
            *head = kv * a.group + at.head(r);
        };
        bool odd = fetch<T, N, DM, kWarps, true>(qs, n, a.dim, [&](uint32_t r) {
            uint32_t i, h;
            place(r, &i, &h);
            return static_cast<const T*>(a.q) + (uint64_t)i * a.q_stride + (uint64_t)h * a.dim;
        });
        odd |= fetch<T, N, DM, kWarps, true>(dos, n, a.dim, [&](uint32_t r) {
            uint32_t i, h;
            place(r, &i, &h);
            return static_cast<const T*>(a.dout) + ((uint64_t)i * a.heads + h) * a.dim;
        });
        if (threadIdx.x < N) {
            uint32_t i = 0, h = 0;
            float lse = 0.0f, delta = 0.0f;
            if (threadIdx.x < n) {
                place(threadIdx.x, &i, &h);
                lse = a.lse_in[(uint64_t)h * a.queries + i];
                delta = a.delta[(uint64_t)h * a.queries + i];
            }
            stat[threadIdx.x] = lse == -INFINITY ? INFINITY : lse * kFgLog2e;      // a row that saw nothing weighs nothing
            stat[N + threadIdx.x] = delta;
        }
        return odd;
    }
    // The warps: kBlocks of 16 rows (of the sums: rows, or keys) by kSides shares of the columns.
    static constexpr int kBlocks = N / 16, kSides = kWarps / kBlocks, NT = N / 8 / kSides, NS = DM / 8 / kSides;
    static __device__ __forceinline__ int block() { return (threadIdx.x >> 5) / kSides * 16; }
    static __device__ __forceinline__ int side() { return (threadIdx.x >> 5) % kSides; }
    // n rows from `at` on against keys from j0 on; p is left out where it is not wanted.  Has this thread left a number that has no usual halves?
    template <bool kP_, bool kAny>
    __device__ __forceinline__ bool weights(const FgAttnArgs& a, const FgAttnSeq& s, const RowPlace& at, uint32_t n, uint32_t j0) {
        const int g = (threadIdx.x & 31) >> 2, q = threadIdx.x & 3, c0 = side() * NT * 8;
        float p[NT][4], dp[NT][4];
        row_products<kAny, NT, DM>(qs + block() * kPitch, ks + c0 * kPitch, a.dim, p);
        row_products<kAny, NT, DM>(dos + block() * kPitch, vs + c0 * kPitch, a.dim, dp);
        Odd<true> odd;
        const float by = a.scale * kFgLog2e;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = block() + g + 8 * h, seen = r < n ? s.seen(a, at.query(r)) : 0;
            const float lse = stat[r], delta = stat[N + r];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float w[2], d[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    w[e] = j0 + c0 + 8 * t + 2 * q + e < seen ? fg_ex2_fast(__fmaf_rn(p[t][2 * h + e], by, -lse)) : 0.0f;
                    d[e] = w[e] == 0.0f ? 0.0f : w[e] * (dp[t][2 * h + e] - delta);
                    odd.meet(w[e]);
                    odd.meet(d[e]);
                }
                const uint32_t to = r * kP + c0 + 8 * t + 2 * q;
                if (kP_) *reinterpret_cast<float2*>(ps + to) = make_float2(w[0], w[1]);
                *reinterpret_cast<float2*>(ds + to) = make_float2(d[0], d[1]);
            }
        }
        return (bool)odd;
    }
    // acc += w (this warp's 16 rows of ds, or columns of ps or ds) times rows of `tile`.
    template <bool kAny>
    __device__ __forceinline__ void add_rows(const float* w, const float* tile, float (&acc)[NS][4]) const {
        const float* const x = w + (block() + ((threadIdx.x & 31) >> 2)) * kP + (threadIdx.x & 3);
        add_products<kAny, NS, DM>([&](int k) { return Left<kAny>(x[8 * k], x[8 * kP + 8 * k], x[8 * k + 4], x[8 * kP + 8 * k + 4]); }, tile + side() * NS * 8, N / 8, acc);
    }
    template <bool kAny>
    __device__ __forceinline__ void add_columns(const float* w, const float* tile, float (&acc)[NS][4]) const {
        const float* const x = w + (threadIdx.x & 3) * kP + block() + ((threadIdx.x & 31) >> 2);
        add_products<kAny, NS, DM>([&](int k) { return Left<kAny>(x[8 * k * kP], x[8 * k * kP + 8], x[(8 * k + 4) * kP], x[(8 * k + 4) * kP + 8]); }, tile + side() * NS * 8, N / 8, acc);
    }
};

template <typename T, int DM, int N>
__device__ __forceinline__ void dq_tile(const FgAttnArgs& a, float* shared, uint64_t number) {
    using B = BwdTile<T, DM, N>;
    B t(shared);
    uint32_t tile;
    const int b = fg_attn_find(a.q_starts, a.sequences, a.queries, a.group, N, number, &tile);
    if (b < 0) return;
    const FgAttnSeq s(a, b);
    const uint64_t rows = (uint64_t)s.nq * a.group, first = (uint64_t)tile * N;
    if (first >= rows) return;
    const uint32_t n = rows - first < N ? (uint32_t)(rows - first) : N, kv = blockIdx.y;
    const RowPlace place(first, a.group);
    const bool odd_rows = t.rows(a, s, kv, place, n);
    float acc[B::NS][4] = {};
    const uint32_t hi = s.seen(a, place.query(n - 1));
    for (uint32_t j0 = 0; j0 < hi; j0 += N) {
        __syncthreads();
        const bool odd_keys = t.keys(a, s, kv, j0);
        bool odd = __syncthreads_or(odd_rows | odd_keys);
        odd |= odd ? t.template weights<false, true>(a, s, place, n, j0) : t.template weights<false, false>(a, s, place, n, j0);
        odd = __syncthreads_or(odd);
        if (odd) t.template add_rows<true>(t.ds, t.ks, acc);
        else t.template add_rows<false>(t.ds, t.ks, acc);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t r = B::block() + ((threadIdx.x & 31) >> 2) + 8 * h;
        if (r >= n) continue;
        T* const to = static_cast<T*>(a.dq) + (uint64_t)(s.q0 + place.query(r)) * a.q_stride + (uint64_t)(kv * a.group + place.head(r)) * a.dim;
        put_columns<T, B::NS>(to, B::side() * B::NS * 8, a.dim, acc, 2 * h, a.scale);
    }
}

template <typename T, int DM, int N>
__device__ __forceinline__ void dkv_tile(const FgAttnArgs& a, float* shared, uint64_t number, uint32_t share) {
    using B = BwdTile<T, DM, N>;
    B t(shared);
    uint32_t tile;
    const int b = fg_attn_find(a.k_starts, a.sequences, a.keys, 1, N, number, &tile);
    if (b < 0) return;
    const FgAttnSeq s(a, b);
    const uint64_t j0_ = (uint64_t)tile * N;
    if (j0_ >= s.nk) return;
    const uint32_t j0 = (uint32_t)j0_, kv = blockIdx.y;
    const bool odd_keys = t.keys(a, s, kv, j0);
    float dk[B::NS][4] = {}, dv[B::NS][4] = {};
    const uint64_t start = (uint64_t)s.first_query(a, j0) * a.group, all = (uint64_t)s.nq * a.group;
    const uint64_t each = ((all - start + N - 1) / N + a.row_shares - 1) / a.row_shares * N, rows = min(all, start + (share + 1) * each);
    for (uint64_t first = start + share * each; first < rows; first += N) {
        const uint32_t n = rows - first < N ? (uint32_t)(rows - first) : N;
        const RowPlace place(first, a.group);
        __syncthreads();
        const bool odd_rows = t.rows(a, s, kv, place, n);
        bool odd = __syncthreads_or(odd_rows | odd_keys);
        odd |= odd ? t.template weights<true, true>(a, s, place, n, j0) : t.template weights<true, false>(a, s, place, n, j0);
        odd = __syncthreads_or(odd);
        if (odd) {
            t.template add_columns<true>(t.ps, t.dos, dv);
            t.template add_columns<true>(t.ds, t.qs, dk);
        } else {
            t.template add_columns<false>(t.ps, t.dos, dv);
            t.template add_columns<false>(t.ds, t.qs, dk);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t j = j0 + B::block() + ((threadIdx.x & 31) >> 2) + 8 * h;
        if (j >= s.nk) continue;
        if (a.row_shares > 1) {
            put_columns<float, B::NS>(fg_attn_part(a, share, 0, s.k0 + j, kv), B::side() * B::NS * 8, a.dim, dk, 2 * h, a.scale);
            put_columns<float, B::NS>(fg_attn_part(a, share, 1, s.k0 + j, kv), B::side() * B::NS * 8, a.dim, dv, 2 * h, 1.0f);
            continue;
        }
        put_columns<T, B::NS>(static_cast<T*>(a.dk) + (uint64_t)(s.k0 + j) * a.k_stride + (uint64_t)kv * a.dim, B::side() * B::NS * 8, a.dim, dk, 2 * h, a.scale);
        put_columns<T, B::NS>(static_cast<T*>(a.dv) + (uint64_t)(s.k0 + j) * a.v_stride + (uint64_t)kv * a.dim, B::side() * B::NS * 8, a.dim, dv, 2 * h, 1.0f);
    }
}

// Tiles of keys first (they have more to do), then tiles of rows, the longest of either first.
template <typename T, int DM, int N>
__global__ void __launch_bounds__(32 * bwd_warps(DM, N), bwd_blocks(DM, N)) attn_bwd_kernel(const FgAttnArgs a, uint32_t key_tiles, uint32_t row_tiles) {
    extern __shared__ float shared[];
    fg_grid_enter();
    const uint32_t key_blocks = key_tiles * a.row_shares;
    if (blockIdx.x < key_blocks) dkv_tile<T, DM, N>(a, shared, blockIdx.x / a.row_shares, blockIdx.x % a.row_shares);
    else dq_tile<T, DM, N>(a, shared, row_tiles - 1 - (blockIdx.x - key_blocks));
}

// The shares' sums of the sequences' keys, added in order: 8 keys a block.
template <typename T>
__global__ void __launch_bounds__(kThreads) attn_fold_kernel(const FgAttnArgs a) {
    fg_grid_enter();
    uint32_t tile;
    const int b = fg_attn_find(a.k_starts, a.sequences, a.keys, 1, 8, blockIdx.x, &tile);
    if (b < 0) return;
    const FgAttnSeq s(a, b);
    const uint32_t line = a.kv_heads * a.dim;
    const uint64_t pitch = 2ull * a.keys * line;
    for (uint64_t j = (uint64_t)tile * 8 + (threadIdx.x >> 5); j < s.nk && j < ((uint64_t)tile + 1) * 8; j += 8)
        for (uint32_t c = threadIdx.x & 31; c < 2 * line; c += 32) {
            const uint32_t which = c >= line, d = c - (which ? line : 0);
            const float* const from = a.part_kv + ((uint64_t)which * a.keys + s.k0 + j) * line + d;
            float v = 0.0f;
#pragma unroll 4
            for (uint32_t z = 0; z < a.row_shares; ++z) v += from[z * pitch];
            if (which) static_cast<T*>(a.dv)[(s.k0 + j) * a.v_stride + d] = fg_narrow<T>(v);
            else static_cast<T*>(a.dk)[(s.k0 + j) * a.k_stride + d] = fg_narrow<T>(v);
        }
}

// More shared memory than a kernel may have by default, to the most it is ever given: once per kernel (`done`) and device.
template <typename K>
int32_t allow_shared(fg_ctx* ctx, std::atomic<uint64_t>& done, K kernel, size_t bytes) {
    if (bytes <= 48 * 1024 || done.load(std::memory_order_acquire) >> (ctx->device & 63) & 1ull) return FG_OK;
    FG_CUDA(ctx, FG_ERR_INTERNAL, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done.fetch_or(1ull << (ctx->device & 63), std::memory_order_release);
    return FG_OK;
}
template <typename T, int RT, int DM>
int32_t rows_launch(fg_ctx* ctx, const FgAttnArgs& a) {
    static std::atomic<uint64_t> done{0};
    const dim3 grid((unsigned)fg_attn_tiles(a.sequences, a.queries, a.group, 16 * RT), a.kv_heads, a.splits);
    const int32_t s = allow_shared(ctx, done, attn_rows_kernel<T, RT, DM>, rows_bytes(RT, DM));
    if (s != FG_OK) return s;
    fg_launch(ctx, attn_rows_kernel<T, RT, DM>, grid, kThreads, rows_bytes(RT, DM), a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T, int DM>
int32_t many_launch(fg_ctx* ctx, const FgAttnArgs& a) {
    static std::atomic<uint64_t> done{0};
    const int32_t s = allow_shared(ctx, done, attn_many_kernel<T, DM>, many_bytes(DM));
    if (s != FG_OK) return s;
    fg_launch(ctx, attn_many_kernel<T, DM>, dim3((unsigned)fg_attn_tiles(a.sequences, a.queries, a.group, 128), a.kv_heads), kThreads, many_bytes(DM), a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}
template <typename T, int DM, int N>
int32_t bwd_launch(fg_ctx* ctx, const FgAttnArgs& a) {
    static std::atomic<uint64_t> done{0};
    const uint32_t key_tiles = a.dk && a.keys ? (uint32_t)fg_attn_tiles(a.sequences, a.keys, 1, N) : 0;
    const uint32_t row_tiles = a.dq && a.queries ? (uint32_t)fg_attn_tiles(a.sequences, a.queries, a.group, N) : 0;
    if (!key_tiles && !row_tiles) return FG_OK;
    const int32_t s = allow_shared(ctx, done, attn_bwd_kernel<T, DM, N>, bwd_bytes(DM, N));
    if (s != FG_OK) return s;
    fg_launch(ctx, attn_bwd_kernel<T, DM, N>, dim3(key_tiles * a.row_shares + row_tiles, a.kv_heads), 32 * bwd_warps(DM, N), bwd_bytes(DM, N), a, key_tiles, row_tiles);
    FG_LAUNCHED(ctx);
    return a.row_shares > 1 ? fg_attn_fold(ctx, dtype_of<T>, a) : FG_OK;
}
// Are there fewer than two blocks of 64 rows for an SM?  Smaller tiles then.
bool few_tiles(const fg_ctx* ctx, const FgAttnArgs& a) { return fg_attn_tiles(a.sequences, a.queries, a.group, 64) * a.kv_heads < 2ull * ctx->sm_count; }

// Few queries per sequence leave few blocks of rows, so their keys go in shares.  A block costs some 3 us beside its keys (0.4 us for 64 of 128 columns), so a
// share has 512 keys or more, up to 16384 where there are enough for 16 blocks an SM (shares of sequences of different lengths even out then); fewer, but 128
// at least, only while there are not two blocks for every SM, which run at a time.  One sequence is cut for those two.  4 sequences of 5000 keys, 8 heads of 128:
// 40 us in shares of 128, 28 like this.
int32_t in_shares(fg_ctx* ctx, FgAttnArgs& a) {
    const uint64_t all = (uint64_t)a.keys * a.kv_heads, once = all / (2ull * ctx->sm_count) + 63, usual = a.keys / a.sequences + 1;
    uint64_t chunk = all / (16ull * ctx->sm_count);
    chunk = chunk < 512 ? 512 : chunk > 16384 ? 16384 : chunk;
    if (a.sequences == 1 || chunk > once) chunk = once;
    chunk = (chunk < 128 ? 128 : chunk) / 64 * 64;
    uint64_t splits = (a.sequences == 1 ? usual : 4 * usual) / chunk + 1;
    if (splits > kMaxSplits) splits = kMaxSplits;
    a.chunk = (uint32_t)chunk;
    a.splits = (uint32_t)splits;
    if (splits == 1) return FG_OK;
    const uint64_t lines = splits * a.queries * a.heads;
    void* w;
    const int32_t s = fg_ws_alloc(ctx, lines * (4ull * a.dim + 8), &w);
    if (s != FG_OK) return s;
    a.part_stat = (float2*)w;
    a.part_out = (float*)w + 2 * lines;
    return FG_OK;
}

// Few rows of a sequence, on average: its keys go in shares.  Otherwise tiles of rows have all of their keys.  Both sides of the border, us, in shares (and in tiles), 32 heads over 8 of 128 columns:
//   bf16, rows        16            48            64            96            128
//   1 x 100000 keys   82 (1475)     145 (1466)    146 (1441)    277 (1438)    280 (1235)
//   8 x 20000         149 (458)     294 (455)     310 (447)     559 (446)     592 (386)
//   64 x 4000         214 (267)     457 (266)     489 (261)     882 (261)     945 (232)
//   64 x 500          67 (48)       141 (48)      165 (47)      270 (48)      319 (48)
//   f32, rows         8             16            32            64
//   1 x 100000 keys   610 (14353)   611 (14357)   1187 (14388)  2113 (14386)
//   64 x 4000         1565 (3949)   1577 (3957)   2779 (3970)   5352 (3977)
//   64 x 500          251 (534)     265 (538)     449 (541)     849 (548)
// 64 rows are right for some sequences with long caches; where there are enough sequences for all SMs, tiles would be from 32 rows on, and for short caches from 16.
template <typename T>
int32_t attention_fwd(fg_ctx* ctx, FgAttnArgs a) {
    const uint64_t rows = ((uint64_t)a.queries * a.group + a.sequences - 1) / a.sequences;      // of a sequence, on average
    const bool tc = fg_attn_tc_suits(ctx, dtype_of<T>, a), few = rows <= (tc ? 64 : 16);
    a.splits = 1;
    if (tc && !few) return fg_attn_tc_fwd(ctx, dtype_of<T>, a);
    if (few) {
        const int32_t s = in_shares(ctx, a);
        if (s != FG_OK) return s;
    }
    int32_t s;
    if (tc) s = fg_attn_few(ctx, dtype_of<T>, a, (uint32_t)rows);
    else if (few || few_tiles(ctx, a)) s = a.dim <= 64 ? rows_launch<T, 1, 64>(ctx, a) : a.dim <= 128 ? rows_launch<T, 1, 128>(ctx, a) : rows_launch<T, 1, 256>(ctx, a);
    else s = a.dim <= 64 ? many_launch<T, 64>(ctx, a) : a.dim <= 128 ? many_launch<T, 128>(ctx, a) : rows_launch<T, 4, 256>(ctx, a);
    if (s != FG_OK || a.splits == 1) return s;
    fg_launch(ctx, attn_join_kernel<T>, (unsigned)fg_attn_tiles(a.sequences, a.queries, a.heads, kJoinRows), kThreads, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

template <typename T>
int32_t attention_bwd(fg_ctx* ctx, FgAttnArgs a) {
    a.splits = 1;
    if (fg_attn_tc_suits(ctx, dtype_of<T>, a)) return fg_attn_tc_bwd(ctx, dtype_of<T>, a);
    const uint64_t lines = (uint64_t)a.queries * a.heads;
    const bool small = a.dim > 128 || few_tiles(ctx, a);
    const int32_t s = fg_attn_bwd_room(ctx, a, small ? 32 : 64, false);
    if (s != FG_OK) return s;
    if (lines) {
        fg_launch(ctx, attn_delta_kernel<T>, (unsigned)((lines + 7) / 8), kThreads, 0, (const T*)a.out, (const T*)a.dout, const_cast<float*>(a.delta), a.queries, a.heads, a.dim);
        FG_LAUNCHED(ctx);
    }
    if (a.dim > 128) return bwd_launch<T, 256, 32>(ctx, a);
    if (small) return a.dim <= 64 ? bwd_launch<T, 64, 32>(ctx, a) : bwd_launch<T, 128, 32>(ctx, a);
    return a.dim <= 64 ? bwd_launch<T, 64, 64>(ctx, a) : bwd_launch<T, 128, 64>(ctx, a);
}

// Bytes from the first to behind the last element of a tensor of `rows` tokens.
uint64_t extent(uint64_t rows, uint64_t stride, uint64_t line, uint32_t size) { return rows ? ((rows - 1) * stride + line) * size : 0; }

// What both passes ask of their arguments; strides of 0 become those of dense tensors.
int32_t check(fg_ctx* ctx, int32_t dtype, FgAttnArgs& a) {
    FG_REQUIRE(ctx, fg_dtype_known(dtype), "attention: unknown dtype");
    FG_REQUIRE(ctx, a.heads >= 1 && a.kv_heads >= 1 && a.heads % a.kv_heads == 0, "attention: heads must be a multiple of kv_heads");
    FG_REQUIRE(ctx, a.kv_heads <= 65535, "attention: too many heads");
    FG_REQUIRE(ctx, a.dim >= 1 && a.dim <= kMaxDim, "attention: head_dim must be 1 to 256");
    FG_REQUIRE(ctx, a.queries < (1u << 31) && a.keys < (1u << 31) && a.sequences < (1u << 24) && a.heads < (1u << 20), "attention: tensor too large");
    FG_REQUIRE(ctx, a.scale >= -0x1p127f && a.scale <= 0x1p127f, "attention: scale must be a number, 2^127 at most");      // (times log2 e it stays one)
    const uint64_t q_line = (uint64_t)a.heads * a.dim, k_line = (uint64_t)a.kv_heads * a.dim;
    if (!a.q_stride) a.q_stride = q_line;
    if (!a.k_stride) a.k_stride = k_line;
    if (!a.v_stride) a.v_stride = k_line;
    FG_REQUIRE(ctx, a.q_stride >= q_line && a.k_stride >= k_line && a.v_stride >= k_line, "attention: a stride is shorter than a token's heads");
    FG_REQUIRE(ctx, a.q_stride < (1u << 30) && a.k_stride < (1u << 30) && a.v_stride < (1u << 30), "attention: stride too large");
    a.group = a.heads / a.kv_heads;
    FG_REQUIRE(ctx, fg_attn_tiles(a.sequences, a.queries, a.heads, 2) < (1ull << 31), "attention: tensor too large");
    FG_REQUIRE(ctx, !a.queries || (a.q && a.out), "attention: NULL pointer");
    FG_REQUIRE(ctx, !a.keys || (a.k && a.v), "attention: NULL pointer");
    FG_REQUIRE(ctx, !a.sequences || (a.q_starts && a.k_starts), "attention: NULL pointer");
    const uint32_t size = fg_dtype_size(dtype);
    FG_REQUIRE(ctx, fg_at_element(a.q, size) && fg_at_element(a.k, size) && fg_at_element(a.v, size) && fg_at_element(a.out, size) && fg_at_element(a.lse, 4) &&
                        fg_at_element(a.lse_in, 4) && fg_at_element(a.dout, size) && fg_at_element(a.dq, size) && fg_at_element(a.dk, size) &&
                        fg_at_element(a.dv, size) && fg_at_element(a.q_starts, 4) && fg_at_element(a.k_starts, 4) && fg_at_element(a.k_lengths, 4),
               "attention: a tensor does not start at an element");
    return FG_OK;
}
struct Range { const void* p; uint64_t n; };
// Do two tensors of tokens share an element?  Rows of `line` bytes, `stride` apart: q, k and v of one product lie between each other's rows.
bool rows_meet(const void* p, uint64_t np, const void* q, uint64_t nq, uint64_t stride, uint64_t p_line, uint64_t q_line) {
    if (!fg_ranges_meet(p, np, q, nq)) return false;
    const int64_t d = (int64_t)(reinterpret_cast<intptr_t>(q) - reinterpret_cast<intptr_t>(p));
    int64_t r = d % (int64_t)stride;
    if (r < 0) r += stride;
    return (uint64_t)r < p_line || (uint64_t)r + q_line > stride;
}

template <typename T>
int32_t fold(fg_ctx* ctx, const FgAttnArgs& a) {
    fg_launch(ctx, attn_fold_kernel<T>, (unsigned)fg_attn_tiles(a.sequences, a.keys, 1, 8), kThreads, 0, a);
    FG_LAUNCHED(ctx);
    return FG_OK;
}

}  // namespace

int32_t fg_attn_bwd_room(fg_ctx* ctx, FgAttnArgs& a, uint32_t rows, bool with_most) {
    const uint64_t blocks = a.dk ? fg_attn_tiles(a.sequences, a.keys, 1, rows) * a.kv_heads : 0, lines = (uint64_t)a.queries * a.heads;
    a.row_shares = 1;
    if (blocks && blocks < (uint64_t)ctx->sm_count) {
        const uint64_t want = 2ull * ctx->sm_count / blocks, have = (uint64_t)a.queries * a.group / a.sequences / (4 * rows), shares = want < have ? want : have;
        if (shares >= 2) a.row_shares = (uint32_t)(shares < 64 ? shares : 64);
    }
    const uint64_t most = with_most ? (8ull * a.sequences * a.kv_heads + 255) / 256 * 256 : 0, first = most + (4 * lines + 255) / 256 * 256;
    void* w;
    const int32_t s = fg_ws_alloc(ctx, first + (a.row_shares > 1 ? 8ull * a.row_shares * a.keys * a.kv_heads * a.dim : 0), &w);
    if (s != FG_OK) return s;
    a.most = static_cast<const uint32_t*>(w);
    a.delta = reinterpret_cast<const float*>(static_cast<const char*>(w) + most);
    a.part_kv = reinterpret_cast<float*>(static_cast<char*>(w) + first);
    return FG_OK;
}
int32_t fg_attn_fold(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a) { return FG_BY_DTYPE(dtype, fold, ctx, a); }

extern "C" {

int32_t fg_attention_fwd(fg_ctx* ctx, int32_t dtype, uint32_t sequences, uint32_t queries, uint32_t keys, uint32_t heads, uint32_t kv_heads,
                         uint32_t head_dim, const uint32_t* q_starts, const uint32_t* k_starts, const uint32_t* k_lengths, const void* q,
                         uint64_t q_stride, const void* k, uint64_t k_stride, const void* v, uint64_t v_stride, float scale, int32_t causal,
                         void* out, float* lse_out) {
    FG_ENTER(ctx);
    FgAttnArgs a{};
    a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse_out;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.q_starts = q_starts; a.k_starts = k_starts; a.k_lengths = k_lengths;
    a.sequences = sequences; a.queries = queries; a.keys = keys; a.heads = heads; a.kv_heads = kv_heads; a.dim = head_dim;
    a.scale = scale; a.causal = causal != 0; a.dev_status = ctx->dev_status;
    const int32_t s = check(ctx, dtype, a);
    if (s != FG_OK) return s;
    const uint32_t size = fg_dtype_size(dtype);
    const uint64_t q_line = (uint64_t)heads * head_dim, k_line = (uint64_t)kv_heads * head_dim, out_bytes = queries * q_line * size, lse_bytes = 4ull * queries * heads;
    const Range in[] = {{q, extent(queries, a.q_stride, q_line, size)}, {k, extent(keys, a.k_stride, k_line, size)}, {v, extent(keys, a.v_stride, k_line, size)},
                        {q_starts, 4ull * sequences + 4}, {k_starts, 4ull * sequences + 4}, {k_lengths, 4ull * sequences}};
    for (const Range& r : in)
        FG_REQUIRE(ctx, !fg_ranges_meet(out, out_bytes, r.p, r.n) && !fg_ranges_meet(lse_out, lse_bytes, r.p, r.n), "fg_attention_fwd: an output overlaps another tensor");
    FG_REQUIRE(ctx, !fg_ranges_meet(out, out_bytes, lse_out, lse_bytes), "fg_attention_fwd: an output overlaps another tensor");
    if (!queries || !sequences) return FG_OK;
    return FG_BY_DTYPE(dtype, attention_fwd, ctx, a);
}

int32_t fg_attention_bwd(fg_ctx* ctx, int32_t dtype, uint32_t sequences, uint32_t queries, uint32_t keys, uint32_t heads, uint32_t kv_heads,
                         uint32_t head_dim, const uint32_t* q_starts, const uint32_t* k_starts, const uint32_t* k_lengths, const void* q,
                         uint64_t q_stride, const void* k, uint64_t k_stride, const void* v, uint64_t v_stride, float scale, int32_t causal,
                         const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv) {
    FG_ENTER(ctx);
    FgAttnArgs a{};
    a.q = q; a.k = k; a.v = v; a.out = const_cast<void*>(out); a.lse_in = lse; a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.q_starts = q_starts; a.k_starts = k_starts; a.k_lengths = k_lengths;
    a.sequences = sequences; a.queries = queries; a.keys = keys; a.heads = heads; a.kv_heads = kv_heads; a.dim = head_dim;
    a.scale = scale; a.causal = causal != 0; a.dev_status = ctx->dev_status;
    const int32_t s = check(ctx, dtype, a);
    if (s != FG_OK) return s;
    FG_REQUIRE(ctx, dq || dk || dv, "fg_attention_bwd: no output");
    FG_REQUIRE(ctx, !dk == !dv, "fg_attention_bwd: dk and dv go together");
    FG_REQUIRE(ctx, !queries || (lse && dout), "fg_attention_bwd: NULL pointer");
    const uint32_t size = fg_dtype_size(dtype);
    const uint64_t q_line = (uint64_t)heads * head_dim, k_line = (uint64_t)kv_heads * head_dim, out_bytes = queries * q_line * size;
    const uint64_t nq = extent(queries, a.q_stride, q_line, size), nk = extent(keys, a.k_stride, k_line, size), nv = extent(keys, a.v_stride, k_line, size);
    const Range in[] = {{q, nq}, {k, nk}, {v, nv}, {out, out_bytes}, {dout, out_bytes}, {lse, 4ull * queries * heads},
                        {q_starts, 4ull * sequences + 4}, {k_starts, 4ull * sequences + 4}, {k_lengths, 4ull * sequences}};
    for (const Range& r : in)
        FG_REQUIRE(ctx, !fg_ranges_meet(dq, nq, r.p, r.n) && !fg_ranges_meet(dk, nk, r.p, r.n) && !fg_ranges_meet(dv, nv, r.p, r.n),
                   "fg_attention_bwd: a gradient overlaps another tensor");
    // The gradients may be rows of one tensor, as q, k and v are: between each other's rows, not in them.
    auto apart = [&](const void* p, uint64_t np, uint64_t ps, uint64_t pl, const void* r, uint64_t nr, uint64_t rs, uint64_t rl) {
        return ps == rs ? !rows_meet(p, np, r, nr, ps * size, pl * size, rl * size) : !fg_ranges_meet(p, np, r, nr);
    };
    FG_REQUIRE(ctx, apart(dq, nq, a.q_stride, q_line, dk, nk, a.k_stride, k_line) && apart(dq, nq, a.q_stride, q_line, dv, nv, a.v_stride, k_line) &&
                        apart(dk, nk, a.k_stride, k_line, dv, nv, a.v_stride, k_line), "fg_attention_bwd: gradients overlap");
    if (!sequences) return FG_OK;
    return FG_BY_DTYPE(dtype, attention_bwd, ctx, a);
}

}  // extern "C"
