// kvd_pages.cu -- sharing, copying, freeing and moving the blocks of a paged
// cache: rows of the block table become copies of other rows (fork), and the
// blocks in use move to the lowest ids (compact).
//
// No reference counterpart (the reference's caches are dense and complete,
// kv_cache/new_kvint8.cu:83-84).
//
// Which blocks are held follows from the table alone: every call marks, in a
// bitmap over the pool, the blocks that the rows name, so no count of holders
// has to be kept, and a block that several rows name is one bit. Both calls are
// two launches. The first marks; its CTA that ends last turns the bitmaps into
// lists (a prefix sum of bit counts) and clears them. The second rewrites the
// table rows and copies blocks, a warp per (block, K or V, head).
//
// Bound: latency of the two launches and of the last CTA's sums, then HBM. Fork:
// 32 rows 11 us, 256 rows that become copies of 32 with their partly filled
// blocks 15 us (0.03 GB), 2,048 rows 29 us. Compact: 2,048 blocks of 16 tokens 21 us;
// 4,096 of 8,192 blocks of 64 tokens x 8 heads x 128 dims in use, half of them
// moved, 103 us: 5.4 TB/s. Marks by 1,024 threads a CTA were slower.
#include "kvd_common.cuh"
#include "kvd_decode.cuh"

namespace kvd {
namespace {

constexpr int kPagesMaxBatch = 8192;  // rows: four bytes each in the shared memory of a CTA, twice
constexpr int kMarkThreads = 512;
constexpr int kWords = 4;  // words of a bitmap that a thread holds at a time
constexpr int kApplyThreads = 256;
constexpr int kEntries = 256;  // table entries a warp takes at a time, eight loads a lane
constexpr int kNoHeir = 0x7fffffff;
constexpr int kNoBlock = INT32_MIN;  // no fresh block is needed

struct Pools {
    int8_t* K;
    int8_t* V;
    float* ks;
    float* vs;
    int8_t* bounds;  // or nullptr
    float* bound_scale;
    int64_t sblk, sh, st, sc_blk, sc_h;
    int H, D;
    FastDiv by_vecs;  // D / bytes a lane copies at a time
    bool bounds16;    // a head's bounds lie on 16-byte boundaries
};

struct PagesParams {
    int B, bs, NB, MB, chunks;  // chunks: stretches of kEntries in a row
    int64_t stride, stride_out;
    const int32_t* lens;
    const int32_t* table;
    int32_t* table_out;
    int32_t* free_in;
    int32_t* free_out;
    const int32_t* count_in;
    int32_t* count_out;
    unsigned int* ticket;
    uint32_t* bits_a;  // fork: blocks of rows that go on; compact: blocks in use
    uint32_t* bits_b;  // fork: blocks of rows that end; compact: free blocks
    int64_t words;
    FastDiv by_bs;
    // fork
    const int32_t* parents;
    int32_t* lens_out;
    int32_t* fresh;   // [B] block of a row's copied tail, or kNoBlock
    int32_t* staged;  // [B][MB] new rows when the table is rewritten in place, or nullptr
    // compact
    int32_t* used;
    uint32_t* movers;  // [words] blocks that move
    int32_t* before;   // [words] blocks that move in front of the word
    // copies: source, destination, tokens
    int32_t* n_copies;
    int32_t* src;
    int32_t* dst;
    int32_t* tokens;  // nullptr: whole blocks
};

__device__ __forceinline__ int row_len(const PagesParams& p, int b) {
    const int64_t cap = static_cast<int64_t>(p.MB) * p.bs;
    return static_cast<int>(min(static_cast<int64_t>(max(0, p.lens[b])), cap));
}

__device__ __forceinline__ int blocks_of(const PagesParams& p, int len) {
    const int whole = static_cast<int>(p.by_bs.div(static_cast<uint32_t>(len)));
    return whole + (whole * p.bs != len);
}

__device__ __forceinline__ bool in_pool(const PagesParams& p, int id) { return id >= 0 && id < p.NB; }

// Marks the blocks id[i] with 32 i < n; returns whether one lies outside the pool. Many rows may name a block: the bits
// are read first, all of them at once, so that most rows write nothing. (A bit that looks unset may be set by now.)
template <int N>
__device__ __forceinline__ bool mark(const PagesParams& p, uint32_t* bits, const int (&id)[N], int n) {
    uint32_t word[N];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool there = 32 * i < n, good = there && in_pool(p, id[i]);
        word[i] = good ? __ldcg(bits + (id[i] >> 5)) : 0xffffffffu;
        bad |= there && !good;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t bit = 1u << (id[i] & 31);
        if (!(word[i] & bit)) atomicOr(bits + (id[i] >> 5), bit);
    }
    return bad;
}

// Exclusive prefix sums of N values a thread over the CTA; total: the sums of all.
template <int N>
__device__ __forceinline__ void cta_scan(int (&x)[N], int (&total)[N], int (*sums)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int inc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        inc[i] = x[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc[i], o);
            if (lane >= o) inc[i] += y;
        }
    }
    __syncthreads();  // the sums of the scan before are no longer read
    if (lane == 31)
#pragma unroll
        for (int i = 0; i < N; ++i) sums[i][warp] = inc[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        int s = lane < nw ? sums[i][lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        const int upto = __shfl_sync(0xffffffffu, s, (warp - 1) & 31);
        total[i] = __shfl_sync(0xffffffffu, s, 31);
        x[i] = inc[i] - x[i] + (warp > 0 ? upto : 0);
    }
}

// True in every thread of the CTA that is the last to get here; what the others wrote before is then visible.
__device__ __forceinline__ bool last_cta(unsigned int* ticket) {
    __shared__ int s_last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        s_last = atomicInc(ticket, gridDim.x - 1) == gridDim.x - 1;
        __threadfence();
    }
    __syncthreads();
    return s_last != 0;
}

// Words [first, last) of a bitmap that this thread turns into lists.
__device__ __forceinline__ void my_words(const PagesParams& p, int64_t& first, int64_t& last) {
    const int64_t n = (p.words + blockDim.x - 1) / blockDim.x;
    first = min(p.words, n * threadIdx.x);
    last = min(p.words, first + n);
}

// kWords words of a bitmap from w on, zeros behind its end; written by other CTAs.
__device__ __forceinline__ void load_words(const PagesParams& p, const uint32_t* bits, int64_t w, uint32_t (&x)[kWords]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) x[i] = w + i < p.words ? __ldcg(bits + w + i) : 0u;
}

// A row's entries from e0 on that a warp marks: its unit u of all rows' stretches.
__device__ __forceinline__ int unit_row(const PagesParams& p, int64_t u, int& e0) {
    if (p.chunks == 1) {
        e0 = 0;
        return static_cast<int>(u);
    }
    const int b = static_cast<int>(u / p.chunks);
    e0 = static_cast<int>(u - static_cast<int64_t>(b) * p.chunks) * kEntries;
    return b;
}

// ------------------------------------------------------------------------ fork
// heir[p]: the row that takes over row p's partly filled last block, -1 for row
// p itself, else the lowest of the rows that copy it; kNoHeir: row p ends.
__global__ void __launch_bounds__(kMarkThreads) fork_mark_kernel(const PagesParams p) {
    extern __shared__ int32_t pages_smem[];
    __shared__ int sums[1][32];
    int32_t* heir = pages_smem;
    int32_t* len = heir + p.B;
    grid_dependency_wait();
    allow_dependents();
    for (int b = threadIdx.x; b < p.B; b += blockDim.x) heir[b] = kNoHeir;
    __syncthreads();
    constexpr int R = 4;  // rows a thread has under way
    for (int b0 = threadIdx.x; b0 < p.B; b0 += R * blockDim.x) {
        int from[R], tokens[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int b = b0 + i * blockDim.x;
            from[i] = b < p.B ? p.parents[b] : -1;
            tokens[i] = b < p.B ? row_len(p, b) : 0;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int b = b0 + i * blockDim.x;
            if (b < p.B) len[b] = tokens[i];
            if (from[i] >= 0 && from[i] < p.B) atomicMin(&heir[from[i]], from[i] == b ? -1 : b);
        }
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x >> 5);
    int status = 0;
    const int64_t units = static_cast<int64_t>(p.B) * p.chunks;
    for (int64_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        int e0;
        const int b = unit_row(p, u, e0);
        const int n = blocks_of(p, len[b]);
        uint32_t* bits = heir[b] == kNoHeir ? p.bits_b : p.bits_a;
        const int32_t* row = p.table + b * p.stride;
        if (e0 < n) {
            int id[kEntries / 32];
#pragma unroll
            for (int i = 0; i < kEntries / 32; ++i) id[i] = 32 * i < n - e0 - lane ? row[e0 + 32 * i + lane] : -1;
            if (mark(p, bits, id, n - e0 - lane)) status |= KVD_STATUS_BAD_BLOCK;
        }
        const int from = p.staged ? p.parents[b] : b;
        if (from != b && from >= 0 && from < p.B) {
            const int m = blocks_of(p, len[from]);
            for (int e = e0 + lane; e < min(m, e0 + kEntries); e += 32)
                p.staged[static_cast<int64_t>(b) * p.MB + e] = p.table[from * p.stride + e];
        }
    }
    if (status) record_status(status);
    if (!last_cta(p.ticket)) return;
    status = 0;
    // blocks that only ended rows held go on the stack, in the order of their ids
    const int fc = min(max(0, *p.count_in), p.NB);
    int pushed = 0;
    for (int64_t base = 0; base < p.words; base += static_cast<int64_t>(blockDim.x) * kWords) {
        const int64_t w = base + static_cast<int64_t>(threadIdx.x) * kWords;
        uint32_t bits[kWords], on[kWords];
        load_words(p, p.bits_b, w, bits);
        load_words(p, p.bits_a, w, on);
        int freed[1] = {0}, total[1];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if (bits[i]) p.bits_b[w + i] = 0;
            if (on[i]) p.bits_a[w + i] = 0;
            bits[i] &= ~on[i];
            freed[0] += __popc(bits[i]);
        }
        cta_scan<1>(freed, total, sums);
        int at = fc + pushed + freed[0];
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            for (; bits[i]; bits[i] &= bits[i] - 1, ++at) {
                if (at < p.NB) p.free_out[at] = static_cast<int32_t>((w + i) * 32) + __ffs(bits[i]) - 1;
                else status |= KVD_STATUS_BAD_BLOCK;  // the list held blocks that rows held too
            }
        pushed += total[0];
    }
    const int height = min(p.NB, fc + pushed);
    __syncthreads();
    // a fresh block, from the top of the stack, for every row that needs a copy of a partly filled block
    constexpr int N = 4;  // neighbouring rows a thread
    int carry = 0;
    for (int base = 0; base < p.B; base += blockDim.x * N) {
        int from[N], tail[N], tail_id[N];
        int copies[1] = {0}, all[1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int b = base + threadIdx.x * N + i;
            from[i] = -1;
            tail[i] = 0;
            tail_id[i] = -1;  // no copy; a bad id is passed on as it is
            if (b >= p.B) continue;
            const int f = p.parents[b];
            if (f < 0 || f >= p.B) continue;
            from[i] = f;
            const int whole = static_cast<int>(p.by_bs.div(static_cast<uint32_t>(len[f])));
            tail[i] = len[f] - whole * p.bs;
            const bool takes_over = heir[f] == -1 ? f == b : heir[f] == b;
            if (tail[i] > 0 && !takes_over) {
                const int id = p.table[f * p.stride + whole];
                if (in_pool(p, id)) tail_id[i] = id;
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) copies[0] += tail_id[i] >= 0;
        cta_scan<1>(copies, all, sums);
        int k = carry + copies[0];
        carry += all[0];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int b = base + threadIdx.x * N + i;
            if (b >= p.B) continue;
            const bool wants = tail_id[i] >= 0, refused = wants && k >= height;
            int id = kNoBlock;
            if (wants && !refused) {
                id = p.free_out[height - 1 - k];
                const bool good = in_pool(p, id);
                if (!good) status |= KVD_STATUS_BAD_BLOCK;
                p.src[k] = tail_id[i];
                p.dst[k] = id;
                p.tokens[k] = good ? tail[i] : 0;
            }
            k += wants;
            if (refused) status |= KVD_STATUS_NO_BLOCKS;
            p.fresh[b] = id;
            p.lens_out[b] = from[i] >= 0 && !refused ? len[from[i]] : 0;
        }
    }
    if (threadIdx.x == 0) {
        const int served = min(carry, height);
        *p.n_copies = served;
        *p.count_out = height - served;
    }
    if (status) record_status(status);
}

// ---------------------------------------------------------------------- copies
// A warp copies the first n tokens of one head of one block, K or V, with their
// scales, and with K the head's bounds. Vec: the widest type on which pools,
// strides and head_dim lie. Bound: HBM; eight loads a lane are under way before the
// first store.
template <class Vec>
__device__ __forceinline__ void copy_head(const Pools& q, int from, int to, int n, bool v_side, int h, int lane) {
    const int8_t* pool = v_side ? q.V : q.K;
    const Vec* src = reinterpret_cast<const Vec*>(pool + from * q.sblk + h * q.sh);
    Vec* dst = reinterpret_cast<Vec*>(const_cast<int8_t*>(pool) + to * q.sblk + h * q.sh);
    const int per = q.D / static_cast<int>(sizeof(Vec));
    const int64_t st = q.st / static_cast<int64_t>(sizeof(Vec));
    const uint32_t all = static_cast<uint32_t>(n) * per;
    constexpr int U = 8;
    for (uint32_t i0 = lane; i0 < all; i0 += 32 * U) {
        Vec x[U];
        int64_t at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = i0 + 32 * u;
            const uint32_t t = q.by_vecs.div(i);
            at[u] = t * st + (i - t * per);
            if (i < all) x[u] = src[at[u]];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 32 * u < all) dst[at[u]] = x[u];
    }
    float* scale = v_side ? q.vs : q.ks;
    const float* s = scale + from * q.sc_blk + h * q.sc_h;
    float* d = scale + to * q.sc_blk + h * q.sc_h;
    for (int t = lane; t < n; t += 32) d[t] = s[t];
    if (!v_side && q.bounds) {
        const int64_t a = (static_cast<int64_t>(from) * q.H + h) * 2 * q.D, b = (static_cast<int64_t>(to) * q.H + h) * 2 * q.D;
        const int pieces = q.bounds16 ? 2 * q.D / 16 : 0;
        for (int i = lane; i < pieces; i += 32)
            reinterpret_cast<uint4*>(q.bounds + b)[i] = reinterpret_cast<const uint4*>(q.bounds + a)[i];
        for (int i = pieces * 16 + lane; i < 2 * q.D; i += 32) q.bounds[b + i] = q.bounds[a + i];
        if (lane == 0) q.bound_scale[static_cast<int64_t>(to) * q.H + h] = q.bound_scale[static_cast<int64_t>(from) * q.H + h];
    }
}

template <class Vec>
__device__ __forceinline__ void copy_blocks(const PagesParams& p, const Pools& q) {
    const int lane = threadIdx.x & 31, per = 2 * q.H;
    const int64_t units = static_cast<int64_t>(*p.n_copies) * per, warps = gridDim.x * (blockDim.x >> 5);
    for (int64_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        const int k = units < 0x7fffffff ? static_cast<int>(static_cast<uint32_t>(u) / static_cast<uint32_t>(per)) : static_cast<int>(u / per);
        const int rest = static_cast<int>(u - static_cast<int64_t>(k) * per);
        const int n = p.tokens ? p.tokens[k] : p.bs;
        const int from = p.src[k], to = p.dst[k];
        if (n > 0) copy_head<Vec>(q, from, to, n, rest >= q.H, rest >= q.H ? rest - q.H : rest, lane);
    }
}

// The new table rows, and the copies of partly filled blocks.
template <class Vec>
__global__ void __launch_bounds__(kApplyThreads) fork_apply_kernel(const PagesParams p, const Pools q) {
    grid_dependency_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x >> 5);
    const int64_t units = static_cast<int64_t>(p.B) * p.chunks;
    for (int64_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        int e0;
        const int b = unit_row(p, u, e0);
        const int from = p.parents[b];
        if (from < 0 || from >= p.B || (p.staged && from == b)) continue;
        const int n = blocks_of(p, p.lens_out[b]), fresh = p.fresh[b];
        const int32_t* row = p.staged ? p.staged + static_cast<int64_t>(b) * p.MB : p.table + from * p.stride;
        for (int e = e0 + lane; e < min(n, e0 + kEntries); e += 32)
            p.table_out[b * p.stride_out + e] = e == n - 1 && fresh != kNoBlock ? fresh : row[e];
    }
    copy_blocks<Vec>(p, q);
}

// --------------------------------------------------------------------- compact
// U blocks in use and F free ones of these requests: the |U| lowest ids of both
// together are where the blocks in use belong. The free ones among them (holes)
// take the blocks in use above them (movers), in order; there are as many of one
// as of the other.
__global__ void __launch_bounds__(kMarkThreads) compact_mark_kernel(const PagesParams p) {
    __shared__ int sums[3][32];
    __shared__ int s_used;
    grid_dependency_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x >> 5);
    const int me = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    int status = 0;
    const int64_t units = static_cast<int64_t>(p.B) * p.chunks;
    for (int64_t u = me; u < units; u += warps) {
        int e0;
        const int b = unit_row(p, u, e0);
        const int n = blocks_of(p, row_len(p, b));
        if (e0 >= n) continue;
        const int32_t* row = p.table + b * p.stride;
        int id[kEntries / 32];
#pragma unroll
        for (int i = 0; i < kEntries / 32; ++i) id[i] = 32 * i < n - e0 - lane ? row[e0 + 32 * i + lane] : -1;
        if (mark(p, p.bits_a, id, n - e0 - lane)) status |= KVD_STATUS_BAD_BLOCK;
    }
    const int fc = min(max(0, *p.count_in), p.NB);
    for (int64_t i = static_cast<int64_t>(me) * 32 + lane; i < fc; i += static_cast<int64_t>(warps) * 32) {
        const int id[1] = {p.free_in[i]};
        if (mark(p, p.bits_b, id, 1)) status |= KVD_STATUS_BAD_BLOCK;
    }
    if (status) record_status(status);
    if (!last_cta(p.ticket)) return;
    if (threadIdx.x == 0) s_used = 0;
    int64_t w0, w1;
    my_words(p, w0, w1);
    int sum[2] = {0, 0}, all[2];
    for (int64_t w = w0; w < w1; ++w) {
        const uint32_t U = __ldcg(p.bits_a + w), F = __ldcg(p.bits_b + w);
        sum[0] += __popc(U);
        sum[1] += __popc(U | F);
    }
    cta_scan<2>(sum, all, sums);
    const int n = all[0];
    // The ids of a word that belong to the n lowest; `owned`: how many ids lie in front of it.
    auto low = [&](uint32_t O, int owned) -> uint32_t {
        const int c = __popc(O);
        if (owned + c <= n) return O;
        if (owned >= n) return 0u;
        uint32_t keep = 0u;
        for (int i = owned; i < n; ++i) {
            const uint32_t bit = O & (0u - O);
            keep |= bit;
            O ^= bit;
        }
        return keep;
    };
    int count[3] = {0, 0, 0}, totals[3];  // holes, movers, blocks that are free afterwards
    int owned = sum[1], top = 0;
    for (int64_t w = w0; w < w1; ++w) {
        const uint32_t U = __ldcg(p.bits_a + w), F = __ldcg(p.bits_b + w), O = U | F, L = low(O, owned);
        count[0] += __popc(L & ~U);
        count[1] += __popc(U & ~L);
        count[2] += __popc(O & ~L);
        if (L) top = static_cast<int>(w * 32) + 32 - __clz(L);
        owned += __popc(O);
    }
    cta_scan<3>(count, totals, sums);
    owned = sum[1];
    for (int64_t w = w0; w < w1; ++w) {
        const uint32_t U = __ldcg(p.bits_a + w), F = __ldcg(p.bits_b + w), O = U | F, L = low(O, owned);
        const int base = static_cast<int>(w * 32);
        owned += __popc(O);
        p.bits_a[w] = p.bits_b[w] = 0;
        p.movers[w] = U & ~L;
        p.before[w] = count[1];
        for (uint32_t x = L & ~U; x; x &= x - 1) p.dst[count[0]++] = base + __ffs(x) - 1;
        for (uint32_t x = U & ~L; x; x &= x - 1) p.src[count[1]++] = base + __ffs(x) - 1;
        // the lowest id ends on top of the stack
        for (uint32_t x = O & ~L; x; x &= x - 1) p.free_out[totals[2] - 1 - count[2]++] = base + __ffs(x) - 1;
    }
    if (top) atomicMax(&s_used, top);
    __syncthreads();
    if (threadIdx.x == 0) {
        *p.n_copies = totals[1];
        *p.count_out = totals[2];
        *p.used = s_used;
    }
}

template <class Vec>
__global__ void __launch_bounds__(kApplyThreads) compact_apply_kernel(const PagesParams p, const Pools q) {
    grid_dependency_wait();
    allow_dependents();
    const int lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x >> 5);
    const int64_t units = static_cast<int64_t>(p.B) * p.chunks;
    const bool moved_only = p.table_out == p.table;
    for (int64_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        int e0;
        const int b = unit_row(p, u, e0);
        const int n = blocks_of(p, row_len(p, b));
        for (int e = e0 + lane; e < min(n, e0 + kEntries); e += 32) {
            const int id = p.table[b * p.stride + e];
            int to = id;
            if (in_pool(p, id)) {
                const uint32_t bits = p.movers[id >> 5], bit = 1u << (id & 31);
                if (bits & bit) to = p.dst[p.before[id >> 5] + __popc(bits & (bit - 1))];
            }
            if (!moved_only || to != id) p.table_out[b * p.stride_out + e] = to;
        }
    }
    copy_blocks<Vec>(p, q);
}

// ------------------------------------------------------------------------ host
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

cudaError_t check_pages(const kvd_pages_desc* d) {
    if (!d || d->batch < 1 || d->batch > kPagesMaxBatch || d->num_kv_heads < 1 || d->head_dim < 1 || d->block_size < 1 ||
        d->num_blocks < 1 || d->max_blocks_per_seq < 1 || d->block_table_stride < d->max_blocks_per_seq ||
        d->block_table_out_stride < d->max_blocks_per_seq)
        return cudaErrorInvalidValue;
    // sums of blocks, a row's entries and tokens, and a copy's bytes are counted in 32 bits
    if (d->num_blocks > 0x40000000 || d->max_blocks_per_seq > 0x40000000 || static_cast<int64_t>(d->block_size) * d->head_dim > 0x3fffffffLL ||
        static_cast<int64_t>(d->max_blocks_per_seq) * d->block_size > 0x7fffffffLL)
        return cudaErrorInvalidValue;
    return cudaSuccess;
}

int64_t bitmap_words(const kvd_pages_desc& d) { return (static_cast<int64_t>(d.num_blocks) + 31) / 32; }

// Four counters, then two bitmaps (all zero between calls), then lists.
PagesParams make_params(const kvd_pages_desc& d, const int32_t* lens, const int32_t* table, int32_t* table_out, void* ws) {
    PagesParams p{};
    p.B = d.batch; p.bs = d.block_size; p.NB = d.num_blocks; p.MB = d.max_blocks_per_seq;
    p.chunks = (d.max_blocks_per_seq + kEntries - 1) / kEntries;
    p.stride = d.block_table_stride; p.stride_out = d.block_table_out_stride;
    p.lens = lens; p.table = table; p.table_out = table_out;
    p.words = bitmap_words(d);
    uint32_t* w = static_cast<uint32_t*>(ws);
    p.ticket = w;
    p.n_copies = reinterpret_cast<int32_t*>(w + 1);
    p.bits_a = w + 4;
    p.bits_b = p.bits_a + p.words;
    p.by_bs = FastDiv(static_cast<uint32_t>(d.block_size));
    return p;
}

// Bytes of the widest type on which the pools, their strides and head_dim lie.
int vec_bytes(const kvd_pages_desc& d, const void* K, const void* V) {
    const uint64_t a = reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) | static_cast<uint64_t>(d.kv_stride_block) |
                       static_cast<uint64_t>(d.kv_stride_h) | static_cast<uint64_t>(d.kv_stride_t) |
                       static_cast<uint64_t>(d.head_dim);
    return (a & 15) == 0 ? 16 : (a & 3) == 0 ? 4 : 1;
}

Pools make_pools(const kvd_pages_desc& d, int8_t* K, int8_t* V, float* ks, float* vs, int8_t* bounds, float* bound_scale,
                 int vec) {
    return Pools{K, V, ks, vs, bounds, bound_scale, d.kv_stride_block, d.kv_stride_h, d.kv_stride_t, d.sc_stride_block,
                 d.sc_stride_h, d.num_kv_heads, d.head_dim, FastDiv(static_cast<uint32_t>(d.head_dim / vec)),
                 (reinterpret_cast<uintptr_t>(bounds) & 15) == 0 && d.head_dim % 8 == 0};
}

unsigned mark_grid(const PagesParams& p) {
    const int64_t want = (static_cast<int64_t>(p.B) * p.chunks + kMarkThreads / 32 - 1) / (kMarkThreads / 32);
    const int64_t most = 2LL * device_sm_count();
    return static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
}

// As many CTAs as fit on the GPU, or fewer where no more can have work.
unsigned apply_grid(const PagesParams& p, const Pools& q, int64_t most_copies) {
    const int64_t rows = static_cast<int64_t>(p.B) * p.chunks, copies = most_copies * 2 * q.H;
    const int64_t want = ((rows > copies ? rows : copies) + kApplyThreads / 32 - 1) / (kApplyThreads / 32);
    const int64_t most = 8LL * device_sm_count();
    return static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
}

bool pools_ok(const void* K, const void* V, const void* ks, const void* vs, const void* bounds, const void* bound_scale) {
    return K && V && ks && vs && (bounds == nullptr) == (bound_scale == nullptr);
}

}  // namespace
}  // namespace kvd

using namespace kvd;

extern "C" size_t kvd_paged_fork_workspace_size(const kvd_pages_desc* d) {
    if (check_pages(d) != cudaSuccess) return 0;
    return 4 * (4 + 2 * static_cast<size_t>(bitmap_words(*d)) + 4 * static_cast<size_t>(d->batch) +
                static_cast<size_t>(d->batch) * d->max_blocks_per_seq);
}

extern "C" cudaError_t kvd_paged_fork_launch(const kvd_pages_desc* d, const int32_t* parents, const int32_t* seq_lens,
                                             const int32_t* block_table, int32_t* free_blocks, const int32_t* free_count,
                                             int8_t* K_pool, int8_t* V_pool, float* k_scale_pool, float* v_scale_pool,
                                             int8_t* bounds, float* bound_scale, int32_t* seq_lens_out,
                                             int32_t* block_table_out, int32_t* free_count_out, void* workspace,
                                             size_t workspace_bytes, cudaStream_t stream) {
    int* launches = launch_counter();
    *launches = 0;
    const cudaError_t bad = check_pages(d);
    if (bad != cudaSuccess) return bad;
    if (!parents || !seq_lens || !block_table || !free_blocks || !free_count || !seq_lens_out || !block_table_out ||
        !free_count_out || !workspace || !pools_ok(K_pool, V_pool, k_scale_pool, v_scale_pool, bounds, bound_scale))
        return cudaErrorInvalidValue;
    if (workspace_bytes < kvd_paged_fork_workspace_size(d) || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0)
        return cudaErrorInvalidValue;
    if (block_table_out == block_table && d->block_table_out_stride != d->block_table_stride) return cudaErrorInvalidValue;
    if (parents == seq_lens_out) return cudaErrorInvalidValue;  // the second launch reads the parents
    PagesParams p = make_params(*d, seq_lens, block_table, block_table_out, workspace);
    p.parents = parents;
    p.lens_out = seq_lens_out;
    p.free_in = p.free_out = free_blocks;
    p.count_in = free_count;
    p.count_out = free_count_out;
    p.fresh = reinterpret_cast<int32_t*>(p.bits_b + p.words);
    p.src = p.fresh + p.B;
    p.dst = p.src + p.B;
    p.tokens = p.dst + p.B;
    p.staged = block_table_out == block_table ? p.tokens + p.B : nullptr;
    const int vec = vec_bytes(*d, K_pool, V_pool);
    const Pools q = make_pools(*d, K_pool, V_pool, k_scale_pool, v_scale_pool, bounds, bound_scale, vec);
    const size_t smem = 8 * static_cast<size_t>(p.B);
    static PerDeviceOnce once;
    cudaError_t e = once.run([] {
        return cudaFuncSetAttribute(fork_mark_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * kPagesMaxBatch);
    });
    if (e != cudaSuccess) return e;
    e = launch_after(fork_mark_kernel, mark_grid(p), kMarkThreads, smem, stream, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    const unsigned grid = apply_grid(p, q, p.B);
    e = vec == 16  ? launch_after(fork_apply_kernel<uint4>, grid, kApplyThreads, 0, stream, p, q)
        : vec == 4 ? launch_after(fork_apply_kernel<uint32_t>, grid, kApplyThreads, 0, stream, p, q)
                   : launch_after(fork_apply_kernel<uint8_t>, grid, kApplyThreads, 0, stream, p, q);
    if (e == cudaSuccess) ++*launches;
    return e;
}

extern "C" size_t kvd_paged_compact_workspace_size(const kvd_pages_desc* d) {
    if (check_pages(d) != cudaSuccess) return 0;
    return 4 * (4 + 4 * static_cast<size_t>(bitmap_words(*d)) + 2 * static_cast<size_t>(d->num_blocks));
}

extern "C" cudaError_t kvd_paged_compact_launch(const kvd_pages_desc* d, const int32_t* seq_lens, const int32_t* block_table,
                                                const int32_t* free_blocks, int32_t* free_count, int8_t* K_pool,
                                                int8_t* V_pool, float* k_scale_pool, float* v_scale_pool, int8_t* bounds,
                                                float* bound_scale, int32_t* block_table_out, int32_t* free_blocks_out,
                                                int32_t* used, void* workspace, size_t workspace_bytes,
                                                cudaStream_t stream) {
    int* launches = launch_counter();
    *launches = 0;
    const cudaError_t bad = check_pages(d);
    if (bad != cudaSuccess) return bad;
    if (!seq_lens || !block_table || !free_blocks || !free_count || !block_table_out || !free_blocks_out || !used ||
        !workspace || !pools_ok(K_pool, V_pool, k_scale_pool, v_scale_pool, bounds, bound_scale))
        return cudaErrorInvalidValue;
    if (workspace_bytes < kvd_paged_compact_workspace_size(d) || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0)
        return cudaErrorInvalidValue;
    if (block_table_out == block_table && d->block_table_out_stride != d->block_table_stride) return cudaErrorInvalidValue;
    PagesParams p = make_params(*d, seq_lens, block_table, block_table_out, workspace);
    p.free_in = const_cast<int32_t*>(free_blocks);
    p.free_out = free_blocks_out;
    p.count_in = free_count;
    p.count_out = free_count;
    p.used = used;
    p.movers = p.bits_b + p.words;
    p.before = reinterpret_cast<int32_t*>(p.movers + p.words);
    p.src = p.before + p.words;
    p.dst = p.src + p.NB;
    const int vec = vec_bytes(*d, K_pool, V_pool);
    const Pools q = make_pools(*d, K_pool, V_pool, k_scale_pool, v_scale_pool, bounds, bound_scale, vec);
    cudaError_t e = launch_after(compact_mark_kernel, mark_grid(p), kMarkThreads, 0, stream, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    const unsigned grid = apply_grid(p, q, p.NB / 2 + 1);
    e = vec == 16  ? launch_after(compact_apply_kernel<uint4>, grid, kApplyThreads, 0, stream, p, q)
        : vec == 4 ? launch_after(compact_apply_kernel<uint32_t>, grid, kApplyThreads, 0, stream, p, q)
                   : launch_after(compact_apply_kernel<uint8_t>, grid, kApplyThreads, 0, stream, p, q);
    if (e == cudaSuccess) ++*launches;
    return e;
}
