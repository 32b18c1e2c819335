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

// ---------------------------------------------------------------- plan
// Which kernel takes a request, and how its tokens are split: one CTA sums the
// work of all requests (tokens times units), which gives the stretch that a
// unit may have, then places every request's units and records by prefix sums.
// A stretch is at least work / target, so split units are fewer than 2 target:
// the room for their records. Bound: latency (loads, two sums, one scan).
__global__ void __launch_bounds__(1024) chunk_plan_kernel(const ChunkParams p) {
    __shared__ unsigned long long work[2];
    __shared__ int sums[4][32];
    grid_dependency_wait();
    allow_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < 2) work[tid] = 0;
    __syncthreads();
    auto shape = [&](int b, int& rows, int& units, bool& few) {
        const ChunkRows r = chunk_rows(p, b);
        rows = r.n * p.G;
        few = rows <= p.few_most;
        units = (few ? (rows + kFewRows - 1) / kFewRows : (rows + p.tile_rows - 1) / p.tile_rows) * p.Hkv;
        return r.len;
    };
    unsigned long long w[2] = {0, 0};
    for (int b = tid; b < p.B; b += blockDim.x) {
        int rows, units;
        bool few;
        const int len = shape(b, rows, units, few);
        w[few ? 0 : 1] += static_cast<unsigned long long>(units) * len;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w[i] += __shfl_xor_sync(0xffffffffu, w[i], o);
        if (lane == 0 && w[i]) atomicAdd(&work[i], w[i]);
    }
    __syncthreads();
    auto span_of = [](unsigned long long x, int target, int least) {
        const unsigned long long s = (x + target - 1) / target;
        return static_cast<int>(min(max(s, static_cast<unsigned long long>(least)), 0x40000000ull));
    };
    const int few_span = span_of(work[0], p.few_target, kFewMinSpan), tile_span = span_of(work[1], p.tile_target, kTileMinSpan);
    int carry[4] = {0, 0, 0, 0};
    for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
        const int b = b0 + tid;
        int x[4] = {0, 0, 0, 0};
        if (b < p.B) {
            int rows, units, each;
            bool few;
            const int len = shape(b, rows, units, few);
            const int n = few ? chunk_splits(len, few_span, kFewStep, each) : chunk_splits(len, tile_span, kTile, each);
            x[few ? 0 : 2] = units * n;
            x[few ? 1 : 3] = n > 1 ? units * n : 0;
        }
        int inc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            inc[i] = x[i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inc[i], o);
                if (lane >= o) inc[i] += y;
            }
        }
        __syncthreads();
        if (lane == 31)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[i][warp] = inc[i];
        __syncthreads();
        int32_t* const first[4] = {p.few_first, p.few_rec, p.tile_first, p.tile_rec};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int s = sums[i][lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += y;
            }
            const int upto = __shfl_sync(0xffffffffu, s, (warp - 1) & 31), all = __shfl_sync(0xffffffffu, s, 31);
            if (b < p.B) first[i][b] = carry[i] + (warp > 0 ? upto : 0) + inc[i] - x[i];
            carry[i] += all;
        }
    }
    if (tid == 0) {
        p.few_first[p.B] = carry[0];
        p.few_rec[p.B] = carry[1];
        p.tile_first[p.B] = carry[2];
        p.tile_rec[p.B] = carry[3];
        *p.head = ChunkHead{carry[0], few_span, carry[2], tile_span, carry[1], carry[3], 0, 0};
    }
}

// ------------------------------------------------------------- split work
// Merges the records of units that were split along the tokens: 16 rows a CTA,
// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.
template <int D>
__global__ void __launch_bounds__(128) chunk_merge_kernel(const ChunkParams p) {
    grid_dependency_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int few = p.head->few_recs, groups = p.tile_rows / kFewRows;
    const int64_t units = few + static_cast<int64_t>(p.head->tile_recs) * groups;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const bool is_few = u < few;
        const int slot = is_few ? static_cast<int>(u) : static_cast<int>((u - few) / groups);
        const int group = is_few ? 0 : static_cast<int>(u - few - static_cast<int64_t>(slot) * groups);
        const int32_t* first = is_few ? p.few_rec : p.tile_rec;
        const int b = warp_find(first, p.B, slot);
        const ChunkRows R = chunk_rows(p, b);
        const int unit_rows = is_few ? kFewRows : p.tile_rows;
        const int rows = R.n * p.G, nrb = (rows + unit_rows - 1) / unit_rows;
        int each;
        const int nsplit = is_few ? chunk_splits(R.len, p.head->few_span, kFewStep, each)
                                  : chunk_splits(R.len, p.head->tile_span, kTile, each);
        const int local = slot - first[b], item = local / nsplit;
        if (local != item * nsplit) continue;  // the first record of a unit stands for all
        const int hk = item / nrb, rb = item - hk * nrb;
        const float* o = is_few ? p.few_o : p.tile_o;
        const float2* ml = is_few ? p.few_ml : p.tile_ml;
        for (int r = group * kFewRows + warp; r < (group + 1) * kFewRows; r += 4) {
            const int row = rb * unit_rows + r;
            if (row >= rows) break;
            const int64_t at = static_cast<int64_t>(slot) * unit_rows + r;
            float M = -INFINITY;
            for (int s = lane; s < nsplit; s += 32) M = fmaxf(M, ml[at + static_cast<int64_t>(s) * unit_rows].x);
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, i));
            float L = 0.f, acc[D / 32] = {};
#pragma unroll 4
            for (int s = 0; s < nsplit; ++s) {
                const int64_t rec = at + static_cast<int64_t>(s) * unit_rows;
                const float2 v = ml[rec];
                const float f = v.x == -INFINITY ? 0.f : exp2f(v.x - M);
                L = fmaf(v.y, f, L);
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
                    const float x = o[rec * D + d * 32 + lane];
                    if (f != 0.f) acc[d] = fmaf(x, f, acc[d]);
                }
            }
            const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(row))), g = row - i * p.G;
            const int64_t o_at = static_cast<int64_t>(R.t0 + i) * p.o_st + static_cast<int64_t>(hk * p.G + g) * p.o_sh;
            const float inv = L == 0.f ? 0.f : 1.f / L;  // no token in sight
#pragma unroll
            for (int d = 0; d < D / 32; ++d) store_out(p.out, o_at + d * 32 + lane, acc[d] * inv, p.flags);
        }
    }
}

template <class... A, class... B>
cudaError_t launch_after(void (*kern)(A...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, B... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

bool tensor_shape(const kvd_paged_prefill_desc& d) {
    return (d.head_dim == 64 || d.head_dim == 128) && d.kv_stride_block >= 0 && d.kv_stride_h >= 0 && d.kv_stride_t >= 0 &&
           ((d.kv_stride_block | d.kv_stride_h | d.kv_stride_t) & 15) == 0;
}

int64_t round16(int64_t x) { return (x + 15) & ~static_cast<int64_t>(15); }

// Lays the workspace out from `base` (0: to learn its size); returns the end.
int64_t lay_out(const kvd_paged_prefill_desc& d, ChunkParams* p, uint8_t* base) {
    const int sms = device_sm_count();
    const int64_t G = d.num_q_heads / d.num_kv_heads, D = d.head_dim, entries = static_cast<int64_t>(d.batch) + 1;
    const int64_t cap = static_cast<int64_t>(d.max_blocks_per_seq) * d.block_size;
    p->few_target = 2 * sms;
    p->tile_target = sms;
    constexpr uint32_t q16 = KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16, o16 = KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16;
    p->tile_rows = (d.flags & q16) != 0 && (d.flags & o16) != 0 ? 256 : 128;
    p->few_most = 32;
    const bool tiles = static_cast<int64_t>(d.num_rows) * G > p->few_most;
    auto records = [&](int64_t target, int64_t unit_rows, int64_t least) {
        // no more units than rows give, and no more splits of each than the longest length gives
        const int64_t units = (d.num_rows * G / unit_rows + (d.batch < d.num_rows ? d.batch : d.num_rows)) * d.num_kv_heads;
        const int64_t splits = (cap + least - 1) / least;
        const int64_t most = units * splits;
        return splits <= 1 ? 0 : most < 2 * target ? most : 2 * target;
    };
    p->max_few_recs = static_cast<int>(records(p->few_target, kFewRows, kFewMinSpan));
    p->max_tile_recs = tiles ? static_cast<int>(records(p->tile_target, p->tile_rows, kTileMinSpan)) : 0;
    // the size is the same for all types of rows and output
    int64_t tile_rows = 0;
    for (int64_t r = 128; tiles && r <= 256; r += 128) {
        const int64_t x = r * records(p->tile_target, r, kTileMinSpan);
        tile_rows = x > tile_rows ? x : tile_rows;
    }
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        uint8_t* here = base + at;
        at += round16(bytes);
        return here;
    };
    p->head = reinterpret_cast<ChunkHead*>(take(sizeof(ChunkHead)));
    p->few_first = reinterpret_cast<int32_t*>(take(4 * entries));
    p->few_rec = reinterpret_cast<int32_t*>(take(4 * entries));
    p->tile_first = reinterpret_cast<int32_t*>(take(4 * entries));
    p->tile_rec = reinterpret_cast<int32_t*>(take(4 * entries));
    p->few_o = reinterpret_cast<float*>(take(4 * D * kFewRows * p->max_few_recs));
    p->few_ml = reinterpret_cast<float2*>(take(8 * kFewRows * static_cast<int64_t>(p->max_few_recs)));
    p->tile_o = reinterpret_cast<float*>(take(4 * D * tile_rows));
    p->tile_ml = reinterpret_cast<float2*>(take(8 * tile_rows));
    return at;
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
    ChunkParams p{};
    return d->head_dim == 64 || d->head_dim == 128 ? static_cast<size_t>(lay_out(*d, &p, nullptr)) : 0;
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
    const int64_t per16 = (d->flags & (KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16)) ? 8 : 4;  // elements of a row in 16 bytes
    p.vec_q = (reinterpret_cast<uintptr_t>(Q) & 15) == 0 && d->q_stride_t % per16 == 0 && d->q_stride_h % per16 == 0;
    const int64_t per16o = (d->flags & (KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16)) ? 8 : 4;
    p.vec_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && d->o_stride_t % per16o == 0 && d->o_stride_h % per16o == 0;
    const bool aligned = ((reinterpret_cast<uintptr_t>(K_pool) | reinterpret_cast<uintptr_t>(V_pool)) & 15) == 0;
    if (!tensor_shape(*d) || !aligned) {
        e = launch_after(chunk_any_kernel, static_cast<unsigned>(p.T * p.Hq), kAnyThreads, 0, stream, p);
        if (e == cudaSuccess) ++*launches;
        return e;
    }
    lay_out(*d, &p, static_cast<uint8_t*>(workspace));
    e = launch_after(chunk_plan_kernel, 1, 1024, 0, stream, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    e = launch_chunk_few(p, stream, launches);
    if (e != cudaSuccess) return e;
    if (static_cast<int64_t>(p.T) * p.G > p.few_most) {  // a request may have many rows
        e = launch_chunk_tile(p, stream, launches);
        if (e != cudaSuccess) return e;
    }
    if (p.max_few_recs + p.max_tile_recs == 0) return cudaSuccess;
    const unsigned grid = 8u * device_sm_count();
    e = p.D == 128 ? launch_after(chunk_merge_kernel<128>, grid, 128, 0, stream, p)
                   : launch_after(chunk_merge_kernel<64>, grid, 128, 0, stream, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}
