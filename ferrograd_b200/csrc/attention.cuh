// What the attention kernels share: the arguments of a call, and which rows of q and of k belong to a block of work.
#pragma once
#include "rows.cuh"

struct FgAttnArgs {
    const void *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;      // elements between tokens
    const uint32_t *q_starts, *k_starts, *k_lengths;
    uint32_t sequences, queries, keys, heads, kv_heads, group, dim;
    float scale;
    int causal;
    void* out;
    float* lse;
    // keys in shares (few queries): a share leaves sums for the rows instead of rows.  splits == 1: none
    uint32_t splits, chunk;      // a sequence has one share per chunk of keys (a multiple of 64), at most splits
    float* part_out;             // [splits][queries][heads][dim]
    float2* part_stat;           // [splits][queries][heads]: the largest score (in powers of 2) and the sum of weights
    // backward
    const void* dout;
    const float *lse_in, *delta;
    void *dq, *dk, *dv;
    // Few tiles of keys: each tile's rows in shares, which leave sums in f32 for fg_attn_fold.  row_shares == 1: none
    uint32_t row_shares;
    float* part_kv;            // [row_shares][dk, dv][keys][kv_heads][dim]
    const uint32_t* most;      // f16 on the tensor cores: the largest |dout| and |v| of each sequence's heads that share one of k and v, as bits: [sequences][kv_heads][2]
    int* dev_status;
};

// One sequence of a call.  Starts and lengths come from memory of the device, so they are held to the tensors' sizes here.
struct FgAttnSeq {
    uint32_t q0, nq, k0, nk;
    __device__ __forceinline__ FgAttnSeq(const FgAttnArgs& a, uint32_t b) {
        q0 = min(a.q_starts[b], a.queries);
        const uint32_t q1 = min(a.q_starts[b + 1], a.queries);
        k0 = min(a.k_starts[b], a.keys);
        const uint32_t k1 = min(a.k_starts[b + 1], a.keys);
        nq = q1 > q0 ? q1 - q0 : 0;
        nk = k1 > k0 ? k1 - k0 : 0;
        if (a.k_lengths) nk = min(nk, a.k_lengths[b]);
    }
    // Shares of this sequence's keys, equal ones of whole 64s; the keys of share z (false: there is none).
    __device__ __forceinline__ uint32_t shares(const FgAttnArgs& a) const { return max(1u, min(a.splits, (nk + a.chunk - 1) / a.chunk)); }
    __device__ __forceinline__ bool share(const FgAttnArgs& a, uint32_t z, uint32_t* lo, uint32_t* hi) const {
        *lo = 0;
        *hi = nk;
        if (a.splits == 1) return true;
        const uint32_t n = shares(a), each = ((nk + 63) / 64 + n - 1) / n * 64;
        *lo = (uint32_t)min((uint64_t)nk, (uint64_t)z * each);
        *hi = (uint32_t)min((uint64_t)nk, (uint64_t)*lo + each);
        return z < n;
    }
    // Keys that query i sees, from the sequence's first on.
    __device__ __forceinline__ uint32_t seen(const FgAttnArgs& a, uint32_t i) const {
        if (!a.causal) return nk;
        const int64_t n = (int64_t)i + 1 + (int64_t)nk - (int64_t)nq;
        return n < 0 ? 0 : (uint32_t)n;
    }
    // The first query that sees key j (nq: none).
    __device__ __forceinline__ uint32_t first_query(const FgAttnArgs& a, uint32_t j) const {
        if (!a.causal) return 0;
        const int64_t i = (int64_t)j - ((int64_t)nk - (int64_t)nq);
        return i <= 0 ? 0 : i >= (int64_t)nq ? nq : (uint32_t)i;
    }
};

// Work is numbered without knowing the lengths: a sequence that starts at row s of a tensor (`per` rows of work for each) has the tiles from
// s * per / rows + b on, which leaves room for all of its tiles before the next one's, and there are total * per / rows + sequences numbers.
// The sequence of tile t, by a warp that asks for 32 starts at a time; the tile within the sequence comes back in `tile`.  -1: none.
__device__ __forceinline__ int fg_attn_find(const uint32_t* starts, uint32_t sequences, uint32_t total, uint32_t per, uint32_t rows, uint64_t t,
                                            uint32_t* tile) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, n = sequences;
    uint64_t base = 0;
    for (;;) {
        const uint32_t step = (n + 31) / 32, at = lane * step;
        uint64_t mine = ~0ull;
        if (at < n) mine = (uint64_t)min(starts[lo + at], total) * per / rows + lo + at;
        const uint32_t k = __popc(__ballot_sync(0xffffffffu, mine <= t));
        if (k == 0) return -1;
        base = __shfl_sync(0xffffffffu, mine, k - 1);
        lo += (k - 1) * step;
        n = min(step, n - (k - 1) * step);
        if (n <= 1) break;
    }
    if (base > t || t - base >= 0xffffffffull) return -1;      // (starts that decrease)
    *tile = (uint32_t)(t - base);
    return (int)lo;
}
inline uint64_t fg_attn_tiles(uint32_t sequences, uint32_t total, uint32_t per, uint32_t rows) { return (uint64_t)total * per / rows + sequences; }

// A key's row of share z's sums (which = 0: dk, 1: dv), of one head.
__device__ __forceinline__ float* fg_attn_part(const FgAttnArgs& a, uint32_t z, uint32_t which, uint64_t key, uint32_t kv) {
    return a.part_kv + (((uint64_t)(z * 2 + which) * a.keys + key) * a.kv_heads + kv) * a.dim;
}
// The backward pass's room in the arena (a.delta, a.part_kv and, where it is wanted, a.most), and into how many shares of rows each tile of `rows` keys is cut: fewer tiles than SMs are
// brought to about two blocks an SM, by shares of four tiles of `rows` rows or more.
int32_t fg_attn_bwd_room(fg_ctx* ctx, FgAttnArgs& a, uint32_t rows, bool with_most);
int32_t fg_attn_fold(fg_ctx* ctx, int32_t dtype, const FgAttnArgs& a);      // adds the shares, in order

constexpr float kFgLog2e = 1.4426950408889634f, kFgLn2 = 0.6931471805599453f;
