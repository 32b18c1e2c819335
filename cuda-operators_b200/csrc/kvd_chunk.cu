// kvd_chunk.cu -- attention of packed new tokens over a paged cache: entry
// points, and the kernel that takes every shape.
//
// No reference counterpart (the reference's prefill attention, attention/, is
// fp32 with no KV cache). With s_j = (q . K_j) ks_j scale over the tokens that a
// row sees, out = sum_j 2^(s_j - m) vs_j V_j / sum_j 2^(s_j - m) in base 2 (the
// scale holds log2(e)), m the running maximum: one pass over the tokens.
#include <cmath>

#include "kvd_chunk.cuh"
#include "kvd_decode.cuh"

namespace kvd {
namespace {

// ------------------------------------------------------------- any shape
// A CTA per (row, head): 64 tokens at a time, a warp per product, dims over the
// threads for the sums of values. For shapes that the tensor-core kernels do not
// take; it reads the cache once per row and head.
constexpr int kAnyThreads = 128;
constexpr int kAnyChunk = 64;
constexpr int kAnyMaxD = 512;

__global__ void __launch_bounds__(kAnyThreads) chunk_any_kernel(const ChunkParams p) {
    __shared__ float qs[kAnyMaxD];
    __shared__ float score[kAnyChunk], weight[kAnyChunk], prob[kAnyChunk], kscl[kAnyChunk], vscl[kAnyChunk];
    __shared__ int64_t row_at[kAnyChunk];
    grid_dependency_wait();
    allow_dependents();
    const int t = blockIdx.x / p.Hq, hq = blockIdx.x - t * p.Hq, hk = hq / p.G;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int lo = 0, hi = p.B;  // the last request that starts at or before row t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    const ChunkRows r = chunk_rows(p, lo);
    if (t < r.t0 || t >= r.t0 + r.n) return;
    const int n = chunk_sees(p, r, t - r.t0);
    const int64_t q0 = t * p.q_st + hq * p.q_sh, o0 = t * p.o_st + hq * p.o_sh;
    for (int d = tid; d < p.D; d += kAnyThreads) qs[d] = load_q(p.Q, q0 + d, p.flags) * p.qscale;
    constexpr int N = kAnyMaxD / kAnyThreads;
    float acc[N] = {};
    float m = -INFINITY, l = 0.f;
    for (int c0 = 0; c0 < n; c0 += kAnyChunk) {
        const int c = min(kAnyChunk, n - c0);
        if (tid < c) {
            const int j = static_cast<int>(p.by_bs.div(static_cast<uint32_t>(c0 + tid))), off = c0 + tid - j * p.bs;
            const int id = p.table[lo * p.bt_stride + j];
            const bool ok = id >= 0 && id < p.NB;
            if (!ok) record_status(KVD_STATUS_BAD_BLOCK);
            const int64_t blk = ok ? id : 0, s = blk * p.sc_sblk + hk * p.sc_sh + off;
            row_at[tid] = blk * p.kv_sblk + hk * p.kv_sh + off * p.kv_st;
            kscl[tid] = ok ? p.ks[s] : 0.f;
            vscl[tid] = ok ? p.vs[s] : 0.f;
        }
        __syncthreads();
        for (int x = warp; x < c; x += kAnyThreads / 32) {
            const int8_t* row = p.K + row_at[x];
            float dot = 0.f;
            for (int d = lane; d < p.D; d += 32) dot = fmaf(qs[d], static_cast<float>(row[d]), dot);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            if (lane == 0) score[x] = dot * kscl[x];
        }
        __syncthreads();
        float top = m;
        for (int x = 0; x < c; ++x) top = fmaxf(top, score[x]);
        const float alpha = m == -INFINITY ? 0.f : exp2f(m - top);
        if (tid < c) {  // into arrays of their own: other threads may still read the scores
            const float e = exp2f(score[tid] - top);
            prob[tid] = e;
            weight[tid] = e * vscl[tid];
        }
        __syncthreads();
        float sum = 0.f;
        for (int x = 0; x < c; ++x) sum += prob[x];
        l = l * alpha + sum;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = tid + i * kAnyThreads;
            if (d < p.D) {
                float a = acc[i] * alpha;
                for (int x = 0; x < c; ++x) a = fmaf(weight[x], static_cast<float>(p.V[row_at[x] + d]), a);
                acc[i] = a;
            }
        }
        m = top;
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int d = tid + i * kAnyThreads;
        if (d < p.D) store_out(p.out, o0 + d, n > 0 ? acc[i] / l : 0.f, p.flags);
    }
}

cudaError_t check_chunk(const kvd_paged_prefill_desc* d) {
    if (!d || d->batch < 1 || d->num_q_heads < 1 || d->num_kv_heads < 1 || d->head_dim < 1 || d->head_dim > kAnyMaxD ||
        d->num_q_heads % d->num_kv_heads != 0 || d->num_rows < 0 || d->block_size < 1 || d->num_blocks < 1 ||
        d->max_blocks_per_seq < 1 || d->block_table_stride < d->max_blocks_per_seq || !d->seq_lens || !d->row_starts ||
        !d->block_table)
        return cudaErrorInvalidValue;
    constexpr uint32_t q16 = KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16, o16 = KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16;
    if ((d->flags & ~(q16 | o16)) != 0 || (d->flags & q16) == q16 || (d->flags & o16) == o16) return cudaErrorInvalidValue;
    // tokens of a request, and rows times heads, are counted in 32 bits
    if (static_cast<int64_t>(d->max_blocks_per_seq) * d->block_size > 0x40000000LL ||
        static_cast<int64_t>(d->num_rows) * d->num_q_heads > 0x40000000LL)
        return cudaErrorInvalidValue;
    return cudaSuccess;
}

}  // namespace
}  // namespace kvd

using namespace kvd;

extern "C" size_t kvd_paged_prefill_workspace_size(const kvd_paged_prefill_desc* d) {
    if (check_chunk(d) != cudaSuccess) return 0;
    return 0;
}

extern "C" cudaError_t kvd_paged_prefill_launch(const kvd_paged_prefill_desc* d, const void* Q, const int8_t* K_pool,
                                                const int8_t* V_pool, const float* k_scale_pool,
                                                const float* v_scale_pool, void* out, void* workspace,
                                                size_t workspace_bytes, cudaStream_t stream) {
    int* launches = launch_counter();
    *launches = 0;
    cudaError_t e = check_chunk(d);
    if (e != cudaSuccess) return e;
    if (d->num_rows == 0) return cudaSuccess;
    if (!Q || !K_pool || !V_pool || !k_scale_pool || !v_scale_pool || !out) return cudaErrorInvalidValue;
    if (workspace_bytes < kvd_paged_prefill_workspace_size(d) || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
        return cudaErrorInvalidValue;
    ChunkParams p{};
    p.Q = Q; p.K = K_pool; p.V = V_pool; p.ks = k_scale_pool; p.vs = v_scale_pool; p.out = out;
    p.seq_lens = d->seq_lens; p.starts = d->row_starts; p.table = d->block_table;
    p.B = d->batch; p.Hq = d->num_q_heads; p.Hkv = d->num_kv_heads; p.G = d->num_q_heads / d->num_kv_heads;
    p.D = d->head_dim; p.T = d->num_rows; p.bs = d->block_size; p.NB = d->num_blocks; p.MB = d->max_blocks_per_seq;
    p.causal = d->causal != 0;
    p.bt_stride = d->block_table_stride;
    p.kv_sblk = d->kv_stride_block; p.kv_sh = d->kv_stride_h; p.kv_st = d->kv_stride_t;
    p.sc_sblk = d->sc_stride_block; p.sc_sh = d->sc_stride_h;
    p.q_st = d->q_stride_t; p.q_sh = d->q_stride_h; p.o_st = d->o_stride_t; p.o_sh = d->o_stride_h;
    const float scale = d->softmax_scale > 0.f ? d->softmax_scale : 1.0f / std::sqrt(static_cast<float>(d->head_dim));
    p.qscale = scale * 1.4426950408889634f;
    p.flags = d->flags;
    p.by_bs = FastDiv(static_cast<uint32_t>(p.bs));
    p.by_g = FastDiv(static_cast<uint32_t>(p.G));
    chunk_any_kernel<<<static_cast<unsigned>(p.T * p.Hq), kAnyThreads, 0, stream>>>(p);
    e = cudaGetLastError();
    if (e == cudaSuccess) ++*launches;
    return e;
}
