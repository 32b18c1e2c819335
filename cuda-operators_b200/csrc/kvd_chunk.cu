// kvd_chunk.cu -- attention of packed new tokens over a paged cache: entry
// points, and the kernel that takes every shape.
//
// No reference counterpart (the reference's prefill attention, attention/, is
// fp32 with no KV cache). With s_j = (q . K_j) ks_j scale over the tokens that a
// row sees, out = sum_j 2^(s_j - m) vs_j V_j / sum_j 2^(s_j - m) in base 2 (the
// scale holds log2(e)), m the running maximum: one pass over the tokens.
#include <atomic>
#include <chrono>
#include <cmath>
#include <random>

#include "kvd_chunk.cuh"
#include "kvd_decode.cuh"

namespace kvd {
namespace {

// ------------------------------------------------------------- any shape
// A CTA per (row, head): 64 tokens at a time, a warp per product, dims over the
// threads for the sums of values. For shapes that the tensor-core kernels do not
// take; it reads the cache once per row and head, which bounds it (16 single tokens
// of up to 8,192, 64 heads, 96 dims: 3.5 ms).
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
            prob[tid] = fabsf(vscl[tid]) < INFINITY ? e : NAN;
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
// Which kernel takes a request, and how its tokens are split: one CTA looks at
// all requests and, for each kernel, at six stretches that a unit may have at
// most: no limit, and the work (tokens times units) over a half to four times
// the CTAs that run at once (twice for many rows). It takes the one whose estimate is least,
//   max(longest stretch, rounds of CTAs x mean stretch)
// for many rows (for few: the mean work of a CTA and half of the longest
// stretch), each stretch with what a unit costs beside its tokens, then places every
// request's units and records by prefix sums. Split units are fewer than twice
// the work over the stretch: the room for their records. Bound: latency (loads,
// two rounds of sums, one scan): 5 us of a call.
constexpr int kSpans = 6;
// Units that stretch k aims at, in quarters of the CTAs that run at once (0: no limit). The records of many rows are
// large: those are split into twice the CTAs' units at most.
__host__ __device__ constexpr int span_quarters(int cls, int k) {
    return k == 0 ? 0 : k == 1 ? 2 : k == 2 ? 3 : k == 3 ? 4 : cls == kMany ? 8 : k == 4 ? 8 : 16;
}

struct ChunkShape {
    int rows, units, len, cls;
};

__device__ __forceinline__ ChunkShape chunk_shape(const ChunkParams& p, int b) {
    const ChunkRows r = chunk_rows(p, b);
    ChunkShape s;
    s.len = r.len;
    s.rows = r.n * p.G;
    s.cls = chunk_class(p, s.rows);
    const int per = s.cls == 0 ? p.unit_rows[0] : s.cls == 1 ? p.unit_rows[1] : p.unit_rows[kMany];
    s.units = (s.rows + per - 1) / per * p.Hkv;
    return s;
}

__device__ __forceinline__ int chunk_step(int cls) { return cls == kMany ? kTile : kFewStep; }

constexpr int kPlanShapes = 1024;  // requests whose shapes the plan keeps in shared memory

__global__ void __launch_bounds__(1024) chunk_plan_kernel(const ChunkParams p) {
    __shared__ ChunkShape shapes[kPlanShapes];
    __shared__ unsigned long long work[kClasses], claimed;
    __shared__ int units_at[kClasses * kSpans], longest_at[kClasses * kSpans], span[kClasses];
    __shared__ int sums[2 * kClasses][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    if (tid < kClasses) work[tid] = 0;
    if (tid == 0) claimed = 0;
    if (tid < kClasses * kSpans) units_at[tid] = longest_at[tid] = 0;
    grid_dependency_wait();
    allow_dependents();
    __syncthreads();
    const bool kept = p.B <= kPlanShapes;
    unsigned long long mine[kClasses + 1] = {};  // work of each class, units of all
    for (int b = tid; b < p.B; b += blockDim.x) {
        const ChunkShape s = chunk_shape(p, b);
        if (kept) shapes[b] = s;
#pragma unroll
        for (int c = 0; c < kClasses; ++c)
            if (c == s.cls) mine[c] += static_cast<unsigned long long>(s.units) * s.len;
        mine[kClasses] += s.units;
    }
#pragma unroll
    for (int c = 0; c <= kClasses; ++c) {  // (64-bit adds to shared memory are slow: one a warp)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine[c] += __shfl_xor_sync(0xffffffffu, mine[c], o);
        if (lane == 0 && mine[c]) atomicAdd(c < kClasses ? &work[c] : &claimed, mine[c]);
    }
    __syncthreads();
    // Rows times heads are at most 2^30, so starts that ascend give fewer units than this; others may give nothing.
    const bool sane = claimed < 0x50000000ull;
    auto shape_of = [&](int b) { return kept ? shapes[b] : chunk_shape(p, b); };
    auto span_of = [&](int cls, int k) {
        if (k == 0) return 0x40000000;
        const unsigned long long parts = static_cast<unsigned long long>(span_quarters(cls, k)) * (cls == 0 ? p.ctas[0] : cls == 1 ? p.ctas[1] : p.ctas[kMany]);
        const unsigned long long s = (4 * work[cls] + parts - 1) / parts, least = cls == kMany ? kTileMinSpan : kFewMinSpan;
        return static_cast<int>(min(max(s, least), 0x40000000ull));
    };
    for (int64_t i = tid; i < static_cast<int64_t>(p.B) * kSpans; i += blockDim.x) {  // a thread per request and stretch
        const int b = static_cast<int>(i / kSpans), k = static_cast<int>(i - static_cast<int64_t>(b) * kSpans);
        const ChunkShape s = shape_of(b);
        if (s.units == 0 || !sane) continue;
        int each;
        const int n = chunk_splits(s.len, span_of(s.cls, k), chunk_step(s.cls), each);
        atomicAdd(&units_at[s.cls * kSpans + k], s.units * n);
        atomicMax(&longest_at[s.cls * kSpans + k], min(each, s.len));
    }
    __syncthreads();
    if (tid < kClasses) {
        const float extra = tid == kMany ? kTileExtra : kFewExtra;
        const int ctas = tid == 0 ? p.ctas[0] : tid == 1 ? p.ctas[1] : p.ctas[kMany];
        int best = 0;
        float least = INFINITY;
        for (int k = 0; k < kSpans; ++k) {
            const int units = max(1, units_at[tid * kSpans + k]);
            const float mean = static_cast<float>(work[tid]) / static_cast<float>(units);
            const float longest = longest_at[tid * kSpans + k] + extra;
            // one CTA of many rows an SM works in rounds; several of few rows share their SM's rate
            const float all = tid == kMany ? static_cast<float>((units + ctas - 1) / ctas) * (mean + extra)
                                           : static_cast<float>(units) / ctas * (mean + extra) + 0.5f * longest;
            const float cost = fmaxf(longest, all);
            if (cost < least) {
                least = cost;
                best = k;
            }
        }
        span[tid] = span_of(tid, best);
    }
    __syncthreads();
    // Starts that do not ascend may give more rows than the call has, and more records than there is room for: no
    // stretch has a limit then.
    int carry[2 * kClasses];
    bool fits = false;
    for (int attempt = 0; attempt < 2 && !fits; ++attempt) {
#pragma unroll
        for (int i = 0; i < 2 * kClasses; ++i) carry[i] = 0;
        for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
            const int b = b0 + tid;
            int x[2 * kClasses] = {}, inc[2 * kClasses];
            if (b < p.B && sane) {
                const ChunkShape s = shape_of(b);
                int each;
                const int n = chunk_splits(s.len, span[s.cls], chunk_step(s.cls), each);
#pragma unroll
                for (int c = 0; c < kClasses; ++c) {
                    x[2 * c] = c == s.cls ? s.units * n : 0;
                    x[2 * c + 1] = c == s.cls && n > 1 ? s.units * n : 0;
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * kClasses; ++i) {
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
                for (int i = 0; i < 2 * kClasses; ++i) sums[i][warp] = inc[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2 * kClasses; ++i) {
                int s = lane < nw ? sums[i][lane] : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, s, o);
                    if (lane >= o) s += y;
                }
                const int upto = __shfl_sync(0xffffffffu, s, (warp - 1) & 31), all = __shfl_sync(0xffffffffu, s, 31);
                int32_t* to = i & 1 ? p.rec[i >> 1] : p.first[i >> 1];
                if (b < p.B) to[b] = carry[i] + (warp > 0 ? upto : 0) + inc[i] - x[i];
                carry[i] += all;
            }
        }
        fits = carry[1] <= p.max_recs[0] && carry[3] <= p.max_recs[1] && carry[5] <= p.max_recs[kMany];
        if (!fits) {
            __syncthreads();
            if (tid < kClasses) span[tid] = 0x40000000;
            __syncthreads();
        }
    }
#pragma unroll
    for (int c = 0; c < kMany; ++c)  // nobody has arrived yet
        for (int i = tid; i < carry[2 * c + 1]; i += blockDim.x) p.arrived[c][i] = 0;
    if (tid == 0) {
        ChunkHead h{};
#pragma unroll
        for (int c = 0; c < kClasses; ++c) {
            p.first[c][p.B] = h.units[c] = carry[2 * c];
            p.rec[c][p.B] = h.recs[c] = carry[2 * c + 1];
            h.span[c] = span[c];
        }
        *p.head = h;
    }
    __syncthreads();  // all of the plan, then the stamp
    if (tid == 0) asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(&p.head->ready), "l"(p.stamp) : "memory");
}

// ------------------------------------------------------------- split work
// Merges the records of units of many rows that were split along the tokens:
// eight rows a CTA, out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s. (Units of
// few rows are merged by the CTA that is last to write one.)
constexpr int kMergeRows = 8;

template <int D>
__global__ void __launch_bounds__(128) chunk_merge_kernel(const ChunkParams p) {
    grid_dependency_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int unit_rows = p.unit_rows[kMany], groups = unit_rows / kMergeRows, span = p.head->span[kMany];
    const int64_t units = static_cast<int64_t>(p.head->recs[kMany]) * groups;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int slot = static_cast<int>(u / groups), group = static_cast<int>(u - static_cast<int64_t>(slot) * groups);
        const int b = warp_find(p.rec[kMany], p.B, slot);
        const ChunkRows R = chunk_rows(p, b);
        const int rows = R.n * p.G, nrb = (rows + unit_rows - 1) / unit_rows;
        int each;
        const int nsplit = chunk_splits(R.len, span, kTile, each);
        const int local = slot - p.rec[kMany][b], item = local / nsplit;
        if (local != item * nsplit) continue;  // the first record of a unit stands for all
        const int hk = item / nrb, rb = item - hk * nrb, r0 = group * kMergeRows + warp * 2;
        merge_records<D, 2>(p, R, p.part_o[kMany], p.part_ml[kMany], slot, nsplit, unit_rows, hk, rb * unit_rows, r0, rows, lane);
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

int64_t group_rows(const kvd_paged_prefill_desc& d) { return static_cast<int64_t>(d.num_rows) * (d.num_q_heads / d.num_kv_heads); }

// Rows of a KV head up to which a request has few: 48. Units of 16 rows re-read and re-widen what a tile shares: 16
// requests of 4,096 to 8,192 bf16 tokens x 8 KV heads, 128 dims, take 89, 138, 181 and 252 us with 16, 32, 48 and 64
// rows each by the kernel for few, 177, 187, 187 and 191 by the one for many (fp32 118, 186, 233, 311 and 229 to 244; 64
// dims 63, 94, 121, 166 and 145 to 153). A call whose requests have up to 32 rows on average and 256 in all takes them all for
// few, which saves two launches.
int few_most(const kvd_paged_prefill_desc& d) {
    const int64_t rows = group_rows(d);
    return rows <= 256 && rows <= 32LL * d.batch ? 256 : 48;
}

// Rows up to which a request goes to the kernel for units of 8: 8, unless there are too few requests to fill the GPU
// and others beside them; one launch less then counts more.
int tiny_most(const kvd_paged_prefill_desc& d) {
    const bool alone = d.num_rows <= d.batch;  // single tokens
    return alone || static_cast<int64_t>(d.batch) * d.num_kv_heads >= 2LL * device_sm_count() ? 8 : 0;
}

// Whether a request of the call may be of a class, by what the host knows.
bool has_class(const kvd_paged_prefill_desc& d, int cls) {
    const int64_t G = d.num_q_heads / d.num_kv_heads, most = group_rows(d);
    return cls == 0 ? G <= tiny_most(d) : cls == 1 ? most > tiny_most(d) && G <= few_most(d) : most > few_most(d);
}

// Rows that requests of a class have at most in any call like this one with as many rows or fewer. Room for records goes
// by this, not by has_class, so that scratch for a loop's largest step serves the smaller ones, which may be of other
// classes: single tokens are tiny in a step by themselves (tiny_most), and 256 rows of a KV head few (few_most).
int64_t class_rows(const kvd_paged_prefill_desc& d, int cls) {
    const int64_t T = d.num_rows, B = d.batch, G = d.num_q_heads / d.num_kv_heads;
    const int64_t alone = T < B ? T : B, few = (B < 8 ? 32 * B : 256) / G;
    if (cls == 0) return G > 8 ? 0 : B * d.num_kv_heads >= 2LL * device_sm_count() ? T : alone;
    if (cls == 1) return G <= 48 ? T : T < few ? T : few;
    return has_class(d, kMany) ? T : 0;  // never in a call of fewer rows than one that has it not
}

int64_t round16(int64_t x) { return (x + 15) & ~static_cast<int64_t>(15); }

// Lays the workspace out from `base` (nullptr: to learn its size, which is the same for all types of rows and
// output and does not fall as rows are added); returns its bytes.
int64_t lay_out(const kvd_paged_prefill_desc& d, ChunkParams* p, uint8_t* base, bool& split) {
    split = false;  // whether units of many rows may be
    const int sms = device_sm_count();
    const int64_t G = d.num_q_heads / d.num_kv_heads, D = d.head_dim, entries = static_cast<int64_t>(d.batch) + 1;
    const int64_t cap = static_cast<int64_t>(d.max_blocks_per_seq) * d.block_size;
    constexpr uint32_t q16 = KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16, o16 = KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16;
    p->unit_rows[0] = 8;
    p->unit_rows[1] = 16;
    p->unit_rows[kMany] = (d.flags & q16) != 0 && (d.flags & o16) != 0 ? 256 : 128;
    for (int c = 0; c < kMany; ++c) p->ctas[c] = sms * chunk_few_ctas(d.head_dim, c, (d.flags & q16) != 0);
    p->ctas[kMany] = sms;
    p->tiny_most = tiny_most(d);
    p->few_most = few_most(d);
    // no more units than rows give, and no more splits of each than the longest length gives
    auto records = [&](int cls, int64_t unit_rows) -> int64_t {
        const int64_t least = cls == kMany ? kTileMinSpan : kFewMinSpan;
        const int64_t rows = class_rows(d, cls), units = (rows * G / unit_rows + (d.batch < rows ? d.batch : rows)) * d.num_kv_heads;
        const int64_t splits = (cap + least - 1) / least, most = units * splits;
        const int64_t ctas = cls == kMany ? sms : sms * chunk_few_ctas(d.head_dim, cls, true), room = 2 * span_quarters(cls, kSpans - 1) * ctas / 4;
        return splits <= 1 ? 0 : most < room ? most : room;
    };
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        uint8_t* here = base + at;
        at += round16(bytes);
        return here;
    };
    p->head = reinterpret_cast<ChunkHead*>(take(sizeof(ChunkHead)));
    for (int c = 0; c < kClasses; ++c) {
        p->first[c] = reinterpret_cast<int32_t*>(take(4 * entries));
        p->rec[c] = reinterpret_cast<int32_t*>(take(4 * entries));
        int64_t rows = records(c, p->unit_rows[c]) * p->unit_rows[c];
        p->max_recs[c] = static_cast<int>(rows / p->unit_rows[c]);
        if (c == kMany) {
            const int64_t x = 128 * records(c, 128), y = 256 * records(c, 256);
            rows = x > y ? x : y;
        }
        p->part_o[c] = reinterpret_cast<float*>(take(4 * D * rows));
        p->part_ml[c] = reinterpret_cast<float2*>(take(8 * rows));
        if (c < kMany) p->arrived[c] = reinterpret_cast<int32_t*>(take(4 * rows / p->unit_rows[c]));
        else split |= rows > 0;
    }
    p->aside = reinterpret_cast<float4*>(take(has_class(d, kMany) && cap > kAsideTiles * kTile ? 4LL * sms * 2 * 128 * D : 0));
    p->aside_tiles = (d.flags & o16) != 0 ? kAsideTiles16 : kAsideTiles;
    return at;
}

// A number that no other call has. Scratch may hold anything, so the numbers start where chance says.
uint64_t next_stamp() {
    static std::atomic<uint64_t> stamp{[]() -> uint64_t {
        try {
            std::random_device chance;
            return static_cast<uint64_t>(chance()) << 32 | chance();
        } catch (...) {  // no source of chance: the time
            return static_cast<uint64_t>(std::chrono::system_clock::now().time_since_epoch().count()) * 0x9e3779b97f4a7c15ull;
        }
    }()};
    uint64_t s = 0;
    while (s == 0) s = stamp.fetch_add(1, std::memory_order_relaxed);  // 0: none
    return s;
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
    bool split;
    return d->head_dim == 64 || d->head_dim == 128 ? static_cast<size_t>(lay_out(*d, &p, nullptr, split)) : 0;
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
    bool split;
    lay_out(*d, &p, static_cast<uint8_t*>(workspace), split);
    p.stamp = next_stamp();
    e = launch_after(chunk_plan_kernel, 1, p.B <= 256 ? 256 : 1024, 0, stream, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    for (int c = 0; c < kClasses; ++c) {
        if (!has_class(*d, c)) continue;
        p.last = c == kMany || !(has_class(*d, kMany) || (c == 0 && has_class(*d, 1)));
        e = c == kMany ? launch_chunk_tile(p, stream, launches) : launch_chunk_few(p, c, stream, launches);
        if (e != cudaSuccess) return e;
        p.follows = 1;
    }
    if (!split) return cudaSuccess;
    const unsigned grid = 8u * device_sm_count();
    e = p.D == 128 ? launch_after(chunk_merge_kernel<128>, grid, 128, 0, stream, p)
                   : launch_after(chunk_merge_kernel<64>, grid, 128, 0, stream, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}
