// kvd_blocks.cuh -- shared by the kernels that select blocks: parameters, score
// keys and the work items of the scoring kernels.
#pragma once

#include <cstdint>

#include "kvd_common.cuh"

namespace kvd {

struct SelectParams {
    kvd_block_select_desc d;
    const void* Q;
    const int8_t* bounds;
    const float* bound_scale;
    int32_t* sel_table;
    int32_t* sel_lens;
    uint32_t* keys;  // [batch * num_kv_heads][max_blocks_per_seq]
};

// Order-preserving key of a score: larger is better; NaN counts as +inf, -0 as
// +0. Keys lie between those of -inf, 0x007fffff, and +inf, 0xff800000.
__device__ __forceinline__ uint32_t score_key(float s) {
    if (isnan(s)) s = INFINITY;
    const uint32_t u = __float_as_uint(s + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kNoBlockKey = 1;  // of a block id outside the pool
__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// Tokens and blocks of request b.
__device__ __forceinline__ int select_len(const kvd_block_select_desc& d, int b, int& n) {
    const int64_t cap = static_cast<int64_t>(d.max_blocks_per_seq) * d.block_size;
    const int len = static_cast<int>(min(static_cast<int64_t>(max(0, d.seq_lens[b])), cap));
    n = static_cast<int>((static_cast<uint32_t>(len) + d.block_size - 1) / d.block_size);
    return len;
}

// Pool id of block i of a table row, -1 for one outside the pool.
__device__ __forceinline__ int pool_id(const kvd_block_select_desc& d, const int32_t* table, int i) {
    const int id = table[i];
    if (id >= 0 && id < d.num_blocks) return id;
    record_status(KVD_STATUS_BAD_BLOCK);
    return -1;
}

// Blocks [i0, i0 + m) of row (b, h).
struct ScoreItem {
    int row, b, h, i0, m;
};

// Tensor-core scores (kvd_score_tc.cu): head_dim 64, 128 or 256, up to 64 query
// heads a KV head.
bool score_tc_ok(const SelectParams& p);
cudaError_t launch_score_tc(const SelectParams& p, cudaStream_t st);

}  // namespace kvd
