// kvd_sel_group.cu -- decode over selected blocks on CUDA cores, for the head
// dims and block sizes that the tensor-core kernel does not take: head_dim 64,
// 128 or 256, any block size, any group of query heads.
//
// No reference counterpart. Per query head and token t of the selection,
//   s_t = (q . k_t) ks_t scale log2(e),  out = sum_t 2^(s_t - m) vs_t v_t / sum_t 2^(s_t - m),
// with the running maximum m and sum of a softmax in one pass. A CTA takes one
// part of a group (up to 8 heads) over a split of the row's tokens, 64 at a
// time, so that every code is read once for all its heads and converted once:
//  * scores: two threads a token, neighbouring 16-byte pieces of its K row each,
//    queries from shared memory, packed fp32 FMAs;
//  * values: a thread per (4 dims, share of the 64 tokens), weights from shared
//    memory, a float4 of accumulators per head; the shares are added at the end.
// Bound: HBM up to 2 heads, above that the packed FMAs (2 D a head and token)
// and the shared-memory reads that feed them. 64 x 8 rows of 2,048 tokens in
// blocks of 16, groups of 1, 2, 4, 8, 16: head_dim 64 (151 MB) 51, 63, 84, 141,
// 244 us; head_dim 256 (554 MB) 187 us for 1, 491 for 8; head_dim 128 in blocks
// of 24 112 and 259. Where both run, the tensor-core kernel takes 47 and 64 us
// (group 1 and 8, blocks of 16) against 65 and 237 here; little work is done
// sooner here (sel_group_first).
#include "kvd_common.cuh"
#include "kvd_decode.cuh"

namespace kvd {
namespace {

constexpr int kSgThreads = 128;
constexpr int kSgTok = 64;

struct SgParams {
    const void* Q;
    const int8_t* K;
    const int8_t* V;
    const float* ks;
    const float* vs;
    void* out;
    float* partials;  // [B*Hq][splits] records of D+4 floats when splits > 1
    const int32_t* lens;   // [B*Hkv]
    const int32_t* table;  // [B*Hkv][bt_stride]
    int Hq, Hkv, S, splits, span;
    int sub, per, group;  // parts of a group, heads of a part, heads of the group
    int nblk;
    FastDiv by_bs;
    int bs;
    int64_t bt_stride, kv_sblk, kv_sh, kv_st, sc_sblk, sc_sh, q_sb, q_sh, o_sb, o_sh;
    float qscale;
    uint32_t flags;
};

__device__ __forceinline__ float redux_max(float x) {  // NaN is left out
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

template <int D, int HP>
__global__ void __launch_bounds__(kSgThreads) sel_group_kernel(const SgParams p) {
    constexpr int QUADS = D / 4, SHARES = kSgThreads / QUADS, PER = kSgTok / SHARES;  // tokens of a share
    static_assert(SHARES * QUADS == kSgThreads, "head_dim 64, 128 or 256");
    __shared__ __align__(16) float q_s[HP][D];
    __shared__ __align__(16) float w_s[kSgTok][HP];
    __shared__ __align__(16) float o_s[SHARES > 1 ? (SHARES - 1) * QUADS * 4 : 4];
    __shared__ const int8_t* vrow[kSgTok];
    __shared__ float red[4][HP];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int heads = gridDim.x / p.sub;  // B * Hkv
    const int part = blockIdx.x / heads, row = blockIdx.x - part * heads;
    const int b = row / p.Hkv, kvh = row - b * p.Hkv, split = blockIdx.y;
    const int h0 = kvh * p.group + part * p.per, nh = min(p.per, p.group - part * p.per);
    grid_dependency_wait();
    allow_dependents();
    const int len = min(max(0, p.lens[row]), p.S);
    const int t_lo = min(len, split * p.span), t_hi = min(len, t_lo + p.span);
    for (int x = tid; x < HP * D; x += kSgThreads) {
        const int h = x / D, d = x - h * D;
        q_s[h][d] = h < nh ? load_q(p.Q, b * p.q_sb + static_cast<int64_t>(h0 + h) * p.q_sh + d, p.flags) * p.qscale : 0.f;
    }
    float m[HP], l[HP];
    float4 acc[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h) { m[h] = -INFINITY; l[h] = 0.f; acc[h] = make_float4(0.f, 0.f, 0.f, 0.f); }
    const int tok = tid >> 1, half = tid & 1;
    const int quad = tid % QUADS, share = tid / QUADS;
    const int64_t v_at = p.V - p.K;
    const int32_t* table = p.table + row * p.bt_stride;
    // A chunk's loads depend on one another (block id, then scales and codes), so they run ahead of
    // their use: block ids two chunks, scales and K codes one, V codes across the scores.
    auto block_at = [&](int c0) {
        const int t = c0 + tok;
        return t < t_hi ? table[p.by_bs.div(t)] : 0;
    };
    const int8_t* kr = p.K;
    float ks = 0.f, vs = 0.f;
    uint4 code[D / 32];
    auto fetch = [&](int c0, int blk) {  // this thread's token of the chunk at c0
        const int t = c0 + tok;
        kr = p.K;
        ks = vs = 0.f;
        if (t >= t_hi) return;
        const int off = t - static_cast<int>(p.by_bs.div(t)) * p.bs;
        if (blk >= 0 && blk < p.nblk) {
            kr = p.K + blk * p.kv_sblk + kvh * p.kv_sh + off * p.kv_st;
            const int64_t sc = blk * p.sc_sblk + kvh * p.sc_sh + off;
            ks = p.ks[sc];
            vs = p.vs[sc];
        } else {  // score 0 and value 0, as in the other kernels
            record_status(KVD_STATUS_BAD_BLOCK);
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) code[i] = *reinterpret_cast<const uint4*>(kr + 32 * i + 16 * half);
    };
    int blk_next = 0;
    if (t_lo < t_hi) {
        fetch(t_lo, block_at(t_lo));
        blk_next = block_at(t_lo + kSgTok);
    }
    for (int c0 = t_lo; c0 < t_hi; c0 += kSgTok) {
        const int n = min(kSgTok, t_hi - c0);
        const bool in = tok < n;
        const float ks_now = ks, vs_now = vs;
        float2 dot[HP];
#pragma unroll
        for (int h = 0; h < HP; ++h) dot[h] = make_float2(0.f, 0.f);
        __syncthreads();  // queries are there; the chunk before is done with w_s and the rows
        if (half == 0) vrow[tok] = kr + v_at;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int piece = 2 * i + half;
            const uint32_t w[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float2 k0, k1;
                dequant4(w[x], k0, k1);
#pragma unroll
                for (int h = 0; h < HP; ++h) {
                    const float4 q = *reinterpret_cast<const float4*>(&q_s[h][16 * piece + 4 * x]);
                    dot[h] = __ffma2_rn(make_float2(q.x, q.y), k0, dot[h]);
                    dot[h] = __ffma2_rn(make_float2(q.z, q.w), k1, dot[h]);
                }
            }
        }
        fetch(c0 + kSgTok, blk_next);
        blk_next = block_at(c0 + 2 * kSgTok);
        float s[HP];
#pragma unroll
        for (int h = 0; h < HP; ++h) {
            float x = dot[h].x + dot[h].y;
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            s[h] = in ? x * ks_now : -INFINITY;
            const float mx = redux_max(s[h]);
            if (lane == 0) red[warp][h] = mx;
        }
        __syncthreads();
        constexpr int AHEAD = PER < 16 ? PER : 16;
        uint32_t vcode[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int tt = share * PER + i;
            vcode[i] = tt < n ? *reinterpret_cast<const uint32_t*>(vrow[tt] + 4 * quad) : 0u;
        }
#pragma unroll
        for (int h = 0; h < HP; ++h) {
            const float mx = fmaxf(fmaxf(red[0][h], red[1][h]), fmaxf(red[2][h], red[3][h]));
            const float m_new = fmaxf(m[h], mx);  // finite: the chunk has a token
            const float alpha = exp2f(m[h] - m_new);
            const float pr = in ? exp2f(s[h] - m_new) : 0.f;
            m[h] = m_new;
            l[h] = l[h] * alpha + (half == 0 ? pr : 0.f);
            acc[h].x *= alpha; acc[h].y *= alpha; acc[h].z *= alpha; acc[h].w *= alpha;
            if (half == 0) w_s[tok][h] = in ? pr * vs_now : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int i0 = 0; i0 < PER; i0 += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {  // a token past the chunk: weight and code 0
                const int tt = share * PER + i0 + i;
                float2 v0, v1;
                dequant4(vcode[i], v0, v1);
                if (i0 + AHEAD < PER) {
                    const int later = tt + AHEAD;
                    vcode[i] = later < n ? *reinterpret_cast<const uint32_t*>(vrow[later] + 4 * quad) : 0u;
                }
#pragma unroll
                for (int h = 0; h < HP; ++h) {
                    const float2 w = make_float2(w_s[tt][h], w_s[tt][h]);
                    const float2 a = __ffma2_rn(w, v0, make_float2(acc[h].x, acc[h].y));
                    const float2 c = __ffma2_rn(w, v1, make_float2(acc[h].z, acc[h].w));
                    acc[h] = make_float4(a.x, a.y, c.x, c.y);
                }
            }
        }
    }
    // one head at a time: sums of weights over the CTA, accumulators over the shares
    const bool records = p.splits > 1 || (p.flags & KVD_FLAG_PARTIAL_OUT);
#pragma unroll
    for (int h = 0; h < HP; ++h) {
        if (h >= nh) break;
        float sum = l[h];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        __syncthreads();
        if (lane == 0) red[warp][0] = sum;
        if (share > 0) *reinterpret_cast<float4*>(&o_s[((share - 1) * QUADS + quad) * 4]) = acc[h];
        __syncthreads();
        if (share > 0) continue;
        sum = red[0][0] + red[1][0] + red[2][0] + red[3][0];
        float4 a = acc[h];
#pragma unroll
        for (int x = 0; x + 1 < SHARES; ++x) {
            const float4 y = *reinterpret_cast<const float4*>(&o_s[(x * QUADS + quad) * 4]);
            a.x += y.x; a.y += y.y; a.z += y.z; a.w += y.w;
        }
        const int hq = h0 + h;
        if (!records) {
            const int64_t at = b * p.o_sb + static_cast<int64_t>(hq) * p.o_sh + 4 * quad;
            const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) store_out(p.out, at + x, sum > 0.f ? v[x] / sum : 0.f, p.flags);
        } else {
            float* rec = p.splits > 1 ? p.partials + ((static_cast<int64_t>(b) * p.Hq + hq) * p.splits + split) * (D + 4)
                                      : static_cast<float*>(p.out) + b * p.o_sb + static_cast<int64_t>(hq) * p.o_sh;
            if (quad == 0) { rec[0] = m[h]; rec[1] = sum; }
            float* o = rec + 4 + 4 * quad;
            o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
        }
    }
}

void group_parts(const kvd_decode_desc& d, int* sub, int* per) {
    const int group = d.num_q_heads / d.num_kv_heads;
    *sub = (group + 7) / 8;
    *per = (group + *sub - 1) / *sub;
}

int sel_group_splits(const kvd_decode_desc& d) {
    int sub, per;
    group_parts(d, &sub, &per);
    const int64_t rows = static_cast<int64_t>(d.batch) * d.num_kv_heads * sub;
    const int chunks = (d.max_seq_len + kSgTok - 1) / kSgTok;
    int64_t want = (8LL * device_sm_count() + rows - 1) / rows;  // two rounds of four CTAs an SM
    if (want > chunks) want = chunks;
    return static_cast<int>(want < 1 ? 1 : want > 65535 ? 65535 : want);
}

template <int D>
cudaError_t launch_d(const SgParams& p, unsigned rows, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows, p.splits, 1);
    cfg.blockDim = dim3(kSgThreads, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (p.per > 4) return cudaLaunchKernelEx(&cfg, sel_group_kernel<D, 8>, p);
    if (p.per > 2) return cudaLaunchKernelEx(&cfg, sel_group_kernel<D, 4>, p);
    if (p.per > 1) return cudaLaunchKernelEx(&cfg, sel_group_kernel<D, 2>, p);
    return cudaLaunchKernelEx(&cfg, sel_group_kernel<D, 1>, p);
}

}  // namespace

bool sel_group_ok(const kvd_decode_desc& d, const PagedView& pv, const int8_t* K, const int8_t* V) {
    if (d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 256) return false;
    if (((reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V)) & 15) != 0) return false;
    if (((pv.kv_sblk | d.kv_stride_h | pv.kv_st) & 15) != 0) return false;
    return static_cast<int64_t>(d.batch) * d.num_q_heads <= 0x7fffffff;
}

// Little work is a matter of latency, and this kernel's splits of 64 tokens and
// short set-up end sooner than the tensor-core kernel's tiles of 128: head_dim
// 128, 8 KV heads, blocks of 16, us here | there, for requests x tokens:
//            1 x 512      1 x 2,048    1 x 4,096    4 x 512     8 x 512     8 x 1,024
//   1 head   5.3 | 8.2    7.4 | 9.4    11 | 11      5.9 | 8.9   6.9 | 10    11 | 11
//   2        6.0 | 8.7    8.4 | 9.8    12 | 12      6.6 | 9.4   8.1 | 10    13 | 12
//   4        7.2 | 9.5    10 | 11      17 | 13      8.4 | 10    13 | 11     20 | 13
//   8        10 | 9.6     13 | 11      23 | 14      12 | 10     20 | 12     35 | 14
bool sel_group_first(const kvd_decode_desc& d) {
    int sub, per;
    group_parts(d, &sub, &per);
    const int64_t tokens = static_cast<int64_t>(d.batch) * d.num_kv_heads * sub * d.max_seq_len;
    return per <= 4 && tokens <= (per <= 2 ? 32768 : 16384);
}

size_t sel_group_workspace_size(const kvd_decode_desc& d) {
    const int splits = sel_group_splits(d);
    return splits > 1 ? static_cast<size_t>(d.batch) * d.num_q_heads * splits * (d.head_dim + 4) * sizeof(float) : 0;
}

cudaError_t launch_sel_group(const kvd_decode_desc& d, const void* Q, const int8_t* K, const int8_t* V,
                             const float* ks, const float* vs, void* out, void* ws, size_t ws_bytes, cudaStream_t st,
                             int* launches, const PagedView& pv) {
    SgParams p{};
    p.Q = Q; p.K = K; p.V = V; p.ks = ks; p.vs = vs; p.out = out;
    p.lens = d.seq_lens; p.table = pv.table;
    p.Hq = d.num_q_heads; p.Hkv = d.num_kv_heads; p.S = d.max_seq_len;
    p.group = d.num_q_heads / d.num_kv_heads;
    group_parts(d, &p.sub, &p.per);
    p.splits = sel_group_splits(d);
    const size_t per_split = static_cast<size_t>(d.batch) * d.num_q_heads * (d.head_dim + 4) * sizeof(float);
    if (!ws || ws_bytes < 2 * per_split) p.splits = 1;
    else if (ws_bytes < p.splits * per_split) p.splits = static_cast<int>(ws_bytes / per_split);
    const int chunks = (d.max_seq_len + kSgTok - 1) / kSgTok;
    p.span = (chunks + p.splits - 1) / p.splits * kSgTok;
    p.partials = static_cast<float*>(ws);
    p.nblk = pv.num_blocks; p.bs = pv.block_size; p.by_bs = FastDiv(pv.block_size);
    p.bt_stride = pv.bt_stride; p.kv_sblk = pv.kv_sblk; p.kv_sh = d.kv_stride_h; p.kv_st = pv.kv_st;
    p.sc_sblk = pv.sc_sblk; p.sc_sh = d.sc_stride_h;
    p.q_sb = d.q_stride_b; p.q_sh = d.q_stride_h; p.o_sb = d.o_stride_b; p.o_sh = d.o_stride_h;
    const float scale = d.softmax_scale > 0.f ? d.softmax_scale : 1.0f / sqrtf(static_cast<float>(d.head_dim));
    p.qscale = scale * 1.4426950408889634f;
    p.flags = d.flags;
    const unsigned rows = static_cast<unsigned>(d.batch) * d.num_kv_heads * p.sub;
    cudaError_t e = d.head_dim == 64 ? launch_d<64>(p, rows, st) : d.head_dim == 128 ? launch_d<128>(p, rows, st)
                                                                                      : launch_d<256>(p, rows, st);
    if (e != cudaSuccess) return e;
    ++*launches;
    if (p.splits > 1) {
        const int64_t rs = d.head_dim + 4;
        e = launch_combine_records(p.partials, p.splits, rs, rs * p.splits,
                                   static_cast<int64_t>(d.batch) * d.num_q_heads, d.num_q_heads, d.head_dim, out,
                                   d.o_stride_b, d.o_stride_h, d.flags, st, launches);
    }
    return e;
}

}  // namespace kvd
