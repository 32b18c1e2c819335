// kvd_chunk.cuh -- shared by the kernels of attention of packed new tokens over
// a paged cache (kvd_paged_prefill_launch).
#pragma once

#include <cstdint>

#include "kvd_common.cuh"

namespace kvd {

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
};

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

}  // namespace kvd
