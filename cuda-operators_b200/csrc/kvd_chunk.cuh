// kvd_chunk.cuh -- shared by the kernels of attention of packed new tokens over
// a paged cache (kvd_paged_prefill_launch): parameters, the plan of their work,
// the records of work that is split along the tokens, and the widening of codes.
#pragma once

#include <cstdint>

#include "kvd_common.cuh"

namespace kvd {

// Work of a call, in the workspace: a header, then six arrays of B + 1 entries.
struct ChunkHead {
    int32_t few_units, few_span;    // units of the kernel for few rows, and tokens of a split at most
    int32_t tile_units, tile_span;  // units of the kernel for many rows, and tokens of a split at most
    int32_t few_recs, tile_recs;    // records of split work
    int32_t ticket, pad;
};

struct ChunkParams {
    const void* Q;
    const int8_t* K;
    const int8_t* V;
    const float* ks;
    const float* vs;
    void* out;
    const int32_t* seq_lens;
    const int32_t* starts;
    const int32_t* table;
    int B, Hq, Hkv, G, D, T, bs, NB, MB, causal;
    int64_t bt_stride;
    int64_t kv_sblk, kv_sh, kv_st, sc_sblk, sc_sh, q_st, q_sh, o_st, o_sh;
    float qscale;  // softmax_scale * log2(e)
    uint32_t flags;
    FastDiv by_bs, by_g;
    int vec_q, vec_out;  // rows on 16-byte boundaries
    // plan
    ChunkHead* head;
    int32_t* few_first;   // [B + 1] units in front of request b's
    int32_t* few_rec;     // [B + 1] records in front of request b's
    int32_t* tile_first;  // the same for the requests with many rows
    int32_t* tile_rec;
    float* few_o;   // records: [slot][kFewRows][D] sums of weighted values
    float2* few_ml; // and [slot][kFewRows] (reference in base 2, sum of weights)
    float* tile_o;
    float2* tile_ml;
    int few_most;      // rows (of one KV head) up to which a request goes to the kernel for few rows
    int tile_rows;     // rows of a unit of the kernel for many rows
    int few_target, tile_target;  // units that splitting aims at
    int max_few_recs, max_tile_recs;
};

constexpr int kFewRows = 16;     // rows of a unit of the kernel for few rows
constexpr int kFewStep = 32;     // tokens of a step of that kernel
constexpr int kFewMinSpan = 256; // tokens that a split has at least
constexpr int kTileMinSpan = 512;
constexpr int kTile = 128;       // tokens of a tile of the kernel for many rows

// Rows [t0, t0 + n) of request b and its tokens.
struct ChunkRows {
    int t0, n, len;
};

__device__ __forceinline__ ChunkRows chunk_rows(const ChunkParams& p, int b) {
    ChunkRows r;
    r.t0 = min(max(0, p.starts[b]), p.T);
    r.n = min(max(r.t0, p.starts[b + 1]), p.T) - r.t0;
    r.len = static_cast<int>(min(static_cast<int64_t>(max(0, p.seq_lens[b])), static_cast<int64_t>(p.MB) * p.bs));
    return r;
}

// Tokens that row i of a request sees: the first of them, this many.
__device__ __forceinline__ int chunk_sees(const ChunkParams& p, const ChunkRows& r, int i) {
    return p.causal ? max(0, min(r.len, r.len - r.n + i + 1)) : r.len;
}

// Splits of a request's tokens, and the tokens of each (a multiple of `step`).
__device__ __forceinline__ int chunk_splits(int len, int span, int step, int& each) {
    const int n = max(1, (len + span - 1) / span);
    each = ((len + n - 1) / n + step - 1) / step * step;
    return max(1, (len + each - 1) / max(1, each));
}

// The last i in [0, n) with first[i] <= x, by a whole warp: 32 places a round.
__device__ __forceinline__ int warp_find(const int32_t* first, int n, int x) {
    const int lane = threadIdx.x & 31;
    int lo = 0;
    while (n > 1) {
        const int step = (n + 31) >> 5, at = lane * step;
        const unsigned ok = __ballot_sync(0xffffffffu, at < n && first[lo + min(at, n - 1)] <= x);
        const int k = ok ? 31 - __clz(ok) : 0;  // the places ascend
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// 2^k as a float, -126 <= k <= 127.
__device__ __forceinline__ float pow2i(int k) { return __int_as_float((k + 127) << 23); }

// Codes as fp16. A code c is the byte c + 128 once its sign bit is flipped; 0x6400 | byte is the fp16
// 1024 + byte, exactly, and 1152 from it leaves c. Even bytes of a word give one pair, odd ones the other.
__device__ __forceinline__ uint32_t half_pair(uint32_t bytes_0_2) {
    uint32_t x = (bytes_0_2 & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Two floats as a pair of fp16, and what the rounding left of them as another.
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack_half(a - f.x, b - f.y);
}

// Exponent k such that |x| 2^k < 2^top, for the largest |x| of a row or of value scales. Zero, infinities
// and NaN have none: k = 0. k stays where 2^k and 2^-k are normal.
__device__ __forceinline__ int fit_exponent(float most, int top) {
    const int e = static_cast<int>(__float_as_uint(most) >> 23);  // most >= 0
    if (most == 0.f || e == 255) return 0;
    return min(max(top - (e - 126), -126), 126);
}

cudaError_t launch_chunk_few(const ChunkParams& p, cudaStream_t st, int* launches);
cudaError_t launch_chunk_tile(const ChunkParams& p, cudaStream_t st, int* launches);

}  // namespace kvd
