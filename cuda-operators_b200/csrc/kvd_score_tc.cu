// kvd_score_tc.cu -- block scores on the 5th-generation tensor cores (tcgen05,
// sm_100a), for the selection of blocks that a decode attends to.
//
// No reference counterpart. A block's bound codes are one row [hi | lo] of 2D
// int8 values and a query head's one row [max(c, 0) | min(c, 0)], so the bound
// of q . k is a plain dot product of 2D integers:
//   sum_d max(c hi, c lo) = sum_d c+ hi + sum_d c- lo,
// exact in int32. A tile is 128 blocks (M) by the heads of a group padded to
// NQ (N) by 2D (K). Its rows lie anywhere in the pool: asynchronous 16-byte
// copies, neighbouring lanes on neighbouring pieces of a row, put them into the
// swizzled operand layout; a thread per block then turns its NQ sums into a
// score. Bound: HBM, 2D + 4 bytes a block and head: 64 requests x 8 heads x up
// to 4,096 blocks of 128 dims, 410 MB in rows of 256 bytes, take 78 us, 5.2 TB/s
// (rows so scattered are read at 6.2 to 6.4 TB/s by a kernel that does nothing
// else). Warp-level int8 products, m16n8k32, took 350 instructions per 16 blocks
// and 101 us, TMA gathers of four rows 164 us; four loading warps instead of
// eight 3 us more.
//
// Roles: warps 0-3 quantise a row's query heads, then score tile by tile;
// warps 4-11 load; warp 12 issues the products and owns the tensor memory. Every
// wait is bounded; on expiry the kernel records KVD_STATUS_WAIT_TIMEOUT and
// unwinds.
#include <type_traits>

#include "kvd_blocks.cuh"
#include "kvd_common.cuh"
#include "kvd_decode.cuh"
#include "kvd_tc.cuh"

namespace kvd {
namespace {

template <int SL, int NQ_>
struct ScoreCfg {
    static constexpr int D = 64 * SL;                  // 2D = 128 bytes a slab
    static constexpr int NQ = NQ_;                     // heads, padded
    static constexpr int E = D / 32;                   // query values a lane quantises
    static constexpr int STAGES = SL == 4 && NQ > 16 ? 2 : 12 / SL;
    static constexpr int LW = 8;                       // loading warps
    static constexpr int LAG = STAGES > 5 ? STAGES - 5 : 1;  // tiles between a tile's issue and the wait for it
    static constexpr int STEPS = 16;                   // tiles whose steps are kept: more than are under way (STAGES + 2)
    static constexpr int SLAB = 128 * 128;             // 128 blocks x 128 bytes
    static constexpr int Q_SLAB = NQ * 128;
    static constexpr int TMEM_COLS = 2 * NQ <= 32 ? 32 : 128;
    static constexpr int THREADS = 32 * (4 + LW + 1);
    static constexpr int OFF_Q = STAGES * SL * SLAB;
    static constexpr int OFF_SQ = OFF_Q + SL * Q_SLAB;  // [2][NQ] scales
    static constexpr int OFF_STEP = OFF_SQ + 2 * NQ * 4;       // [STEPS][128] steps
    static constexpr int OFF_BAR = OFF_STEP + STEPS * 512;
    static constexpr int B_FULL = 0, B_EMPTY = STAGES, B_ACC = 2 * STAGES, B_FREE = B_ACC + 2, B_Q = B_FREE + 2,
                         B_DONE = B_Q + 1, B_DRAIN = B_DONE + 1, B_STEP = B_DRAIN + 1, NBAR = B_STEP + STEPS;
    static constexpr int OFF_TMEM = OFF_BAR + NBAR * 8;
    static constexpr int SMEM_BYTES = OFF_TMEM + 8 + 1024;  // slack to align the base to 1024
    static_assert(2 * NQ <= 128 && NQ % 16 == 0, "tensor memory columns");
    static_assert(SMEM_BYTES <= 227 * 1024 && STEPS >= STAGES + 3, "shared memory");
};

// The tiles of all rows that have any, in order of (request, KV head, tile), are
// dealt to the CTAs in equal stretches: a stretch is a walk over parts of rows.
struct Walk {
    int b, h, tile, left;
};

// Tiles of a row of request b; n: its blocks.
__device__ __forceinline__ int row_tiles(const SelectParams& p, int b, int& n) {
    select_len(p.d, b, n);
    return n > p.d.budget ? (n + 127) / 128 : 0;
}

// This CTA's stretch, found by all threads together: thread i sums the tiles of
// its share of the requests, and the one whose share holds the stretch's first
// tile walks to it.
template <int THREADS>
__device__ __forceinline__ Walk first_part(const SelectParams& p, Walk* found, int* warp_sums) {
    constexpr int WARPS = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, H = p.d.num_kv_heads;
    const int each = (p.d.batch + THREADS - 1) / THREADS;
    const int b0 = min(p.d.batch, tid * each), b1 = min(p.d.batch, b0 + each);
    int mine = 0, n;
    for (int b = b0; b < b1; ++b) mine += row_tiles(p, b, n) * H;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) warp_sums[warp] = upto;
    if (tid == 0) found->left = 0;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w == warp) upto += total;
        total += warp_sums[w];
    }
    const int first = static_cast<int>(static_cast<int64_t>(total) * blockIdx.x / gridDim.x);
    const int last = static_cast<int>(static_cast<int64_t>(total) * (blockIdx.x + 1) / gridDim.x);
    int at = upto - mine;
    if (first < last && first >= at && first < upto) {
        int b = b0, tiles = row_tiles(p, b, n);
        while (first >= at + tiles * H) {
            at += tiles * H;
            tiles = row_tiles(p, ++b, n);
        }
        found->b = b;
        found->h = (first - at) / tiles;
        found->tile = (first - at) % tiles;
        found->left = last - first;
    }
    __syncthreads();
    return *found;
}

// The next part of a row of the walk; false at its end.
__device__ __forceinline__ bool next_part(const SelectParams& p, Walk& w, ScoreItem& I) {
    if (w.left <= 0) return false;
    int n, tiles;
    while ((tiles = row_tiles(p, w.b, n)) == 0) ++w.b;
    const int take = min(w.left, tiles - w.tile);
    I.b = w.b;
    I.h = w.h;
    I.row = w.b * p.d.num_kv_heads + w.h;
    I.i0 = w.tile * 128;
    I.m = min(n - I.i0, take * 128);
    w.left -= take;
    w.tile += take;
    if (w.tile == tiles) {
        w.tile = 0;
        if (++w.h == p.d.num_kv_heads) {
            w.h = 0;
            ++w.b;
        }
    }
    return true;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// fn(N - 1), ..., fn(0), as compile-time constants.
template <int N, class F>
__device__ __forceinline__ void each_down(F& fn) {
    if constexpr (N > 0) {
        fn(std::integral_constant<int, N - 1>{});
        each_down<N - 1>(fn);
    }
}

// A place in the ring of stages and how often it was passed.
template <int STAGES>
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++s == STAGES) {
            s = 0;
            phase ^= 1u;
        }
    }
};

// One of LW loading warps: its share of every tile's rows, a row of 2D bytes by
// SL * 8 neighbouring lanes, 16 bytes each, to their swizzled places. A tile
// counts as full once its copies are done and fenced for the tensor cores'
// reads. The wait for that comes LAG tiles after the issue, LAG below the
// number of stages: the stage that the next tile goes to is then free before it
// is asked for, and the warps wait for memory only (with 6 stages, selecting for
// 64 requests takes 89.5 us with a LAG of 1, 90.1, 91.4 and 93.3 of 2, 3 and 4;
// four accumulators instead of two change nothing). The blocks' steps
// come along, into a ring of their own that the scoring warps read.
template <int SL, int NQ>
__device__ __forceinline__ void score_loader(const SelectParams& p, uint8_t* smem, Walk walk, int w) {
    using C = ScoreCfg<SL, NQ>;
    constexpr int LAG = C::LAG, ROWS = 128 / C::LW;
    constexpr int PIECES = SL * 8;    // 16-byte pieces of a row
    constexpr int RPI = 32 / PIECES;  // rows an instruction covers
    static_assert(ROWS <= 32, "a lane per row");
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    const int lane = threadIdx.x & 31, H = p.d.num_kv_heads;
    const int sub = lane / PIECES, piece = lane % PIECES;
    Ring<C::STAGES> in, out;  // issued, arrived
    Ring<C::STEPS> step_in, step_out;
    int issued = 0;  // up to LAG, then constant
    auto arrive = [&] {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&bars[C::B_FULL + out.s]);
            mbar_arrive(&bars[C::B_STEP + step_out.s]);
        }
        out.next();
        step_out.next();
    };
    const uint32_t stride = static_cast<uint32_t>(H) * (2 * C::D);
    // place of this lane's piece of row j + sub: row * 128 + ((piece ^ row) & 7) * 16, whose swizzle
    // depends on j through a few values only
    uint32_t swz[8 / RPI];
#pragma unroll
    for (int x = 0; x < 8 / RPI; ++x) swz[x] = sub * 128 + (((piece ^ (x * RPI + sub)) & 7) << 4);
    const uint32_t mine = smem_u32(smem) + (piece >> 3) * C::SLAB + w * ROWS * 128;
    bool ok = true, wrapped = false;
    ScoreItem I;
    while (ok && next_part(p, walk, I)) {
        const int32_t* table = p.d.block_table + I.b * p.d.block_table_stride + I.i0 + ROWS * w + lane;
        const int8_t* bounds = p.bounds + static_cast<int64_t>(I.h) * (2 * C::D) + piece * 16;
        // ids are loaded a tile ahead and looked at only then: a test would wait for the load
        int left = I.m - ROWS * w;  // rows from this warp's first one of the tile to the part's end
        int loaded = lane < left ? table[0] : 0;
        for (int i = 0; i < I.m; i += 128, left -= 128) {
            int id = loaded;
            const bool good = id >= 0 && id < p.d.num_blocks;
            if (!good) {  // row 0 is read in its place
                record_status(KVD_STATUS_BAD_BLOCK);
                id = 0;
            }
            table += 128;
            loaded = lane < left - 128 ? table[0] : 0;
            if (wrapped && !mbar_wait(&bars[C::B_EMPTY + in.s], in.phase ^ 1u)) {
                ok = false;
                break;
            }
            const uint32_t tile = mine + in.s * (SL * C::SLAB);
            uint32_t dst[8 / RPI];
#pragma unroll
            for (int x = 0; x < 8 / RPI; ++x) dst[x] = tile + swz[x];
            uint32_t rid[ROWS / RPI];  // all shuffles first: one before each copy would wait for it
#pragma unroll
            for (int j = 0; j < ROWS / RPI; ++j) rid[j] = __shfl_sync(0xffffffffu, id, j * RPI + sub);
            auto copy = [&](int j) {
                cp_async16(dst[(j & 7) / RPI] + j * 128, bounds + static_cast<uint64_t>(rid[j / RPI]) * stride);
            };
            if (left >= ROWS) {
#pragma unroll
                for (int j = 0; j < ROWS; j += RPI) copy(j);
            } else {
#pragma unroll
                for (int j = 0; j < ROWS; j += RPI)
                    if (j < left) copy(j);  // the same for the whole warp
            }
            float* step = reinterpret_cast<float*>(smem + C::OFF_STEP) + step_in.s * 128 + w * ROWS + lane;
            if (good && lane < ROWS) cp_async4(smem_u32(step), p.bound_scale + static_cast<int64_t>(id) * H + I.h);
            else if (lane < ROWS) *step = -1.f;  // no block: below every score
            cp_async_commit();
            step_in.next();
            in.next();
            if (in.s == 0) wrapped = true;
            if (issued == LAG) {
                cp_async_wait<LAG>();
                arrive();
            } else {
                ++issued;
            }
        }
    }
    // the last tiles, each as soon as it is there
    auto rest = [&](auto left) {
        constexpr int X = decltype(left)::value;
        if (issued > X) {
            cp_async_wait<X>();
            arrive();
        }
    };
    each_down<LAG>(rest);
}

// The whole warp walks along and one elected lane issues, so that operands stay
// in uniform registers: issued by a single thread a tile's eight products took
// about 1,000 cycles and bounded the kernel.
template <int SL, int NQ>
__device__ __forceinline__ void score_mma(const SelectParams& p, uint8_t* smem, uint32_t tmem, Walk walk) {
    using C = ScoreCfg<SL, NQ>;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    constexpr uint32_t idesc = idesc_i8(true, true, false, false, NQ, 128);
    Ring<C::STAGES> in;
    Ring<2> acc;
    bool second = false;  // both accumulators were used
    uint32_t q_phase = 0;
    ScoreItem I;
    while (next_part(p, walk, I)) {
        if (!mbar_wait(&bars[C::B_Q], q_phase)) return;
        q_phase ^= 1u;
        for (int i = 0; i < I.m; i += 128) {
            if (!mbar_wait(&bars[C::B_FULL + in.s], in.phase)) return;
            if (second && !mbar_wait(&bars[C::B_FREE + acc.s], acc.phase ^ 1u)) return;
            tc_fence_after();
            const uint32_t abase = smem_u32(smem + in.s * SL * C::SLAB), qbase = smem_u32(smem + C::OFF_Q);
#pragma unroll
            for (int x = 0; x < 4 * SL; ++x) {
                const uint64_t ad = smem_desc(abase + (x >> 2) * C::SLAB + 32u * (x & 3), 16u, 1024u, kLayoutSw128);
                const uint64_t bd = smem_desc(qbase + (x >> 2) * C::Q_SLAB + 32u * (x & 3), 16u, 1024u, kLayoutSw128);
                mma_i8_warp(tmem + acc.s * NQ, ad, bd, idesc, x > 0);
            }
            mma_commit_warp(&bars[C::B_EMPTY + in.s]);
            mma_commit_warp(&bars[C::B_ACC + acc.s]);
            in.next();
            acc.next();
            if (acc.s == 0) second = true;
        }
    }
}

// Codes of the part's query heads by the cache's quantiser rule (kvd_quant.cuh)
// into the K-major, 128-byte-swizzled operand: head w + 4 j is warp w's.
template <int SL, int NQ>
__device__ __forceinline__ void score_query(const SelectParams& p, uint8_t* smem, const ScoreItem& I, float* scales) {
    using C = ScoreCfg<SL, NQ>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.d.num_q_heads / p.d.num_kv_heads;
    constexpr int ROUND = SL <= 2 ? 4 : 2;  // heads whose loads are in flight together
    for (int n0 = warp; n0 < G; n0 += 4 * ROUND) {
        float x[ROUND][C::E], a[ROUND];
#pragma unroll
        for (int y = 0; y < ROUND; ++y) {
            const int n = n0 + 4 * y;
            const int64_t q0 = I.b * p.d.q_stride_b + static_cast<int64_t>(I.h * G + n) * p.d.q_stride_h + lane * C::E;
#pragma unroll
            for (int j = 0; j < C::E; ++j) x[y][j] = n < G ? load_q(p.Q, q0 + j, p.d.flags) : 0.f;
        }
#pragma unroll
        for (int y = 0; y < ROUND; ++y) {
            a[y] = 0.f;
#pragma unroll
            for (int j = 0; j < C::E; ++j) a[y] = fmaxf(a[y], fabsf(x[y][j]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int y = 0; y < ROUND; ++y) a[y] = fmaxf(a[y], __shfl_xor_sync(0xffffffffu, a[y], o));
#pragma unroll
        for (int y = 0; y < ROUND; ++y) {
            const int n = n0 + 4 * y;
            if (n >= G) break;
            const float s = a[y] == 0.f ? 0.f : a[y] / 127.0f;
#pragma unroll
            for (int j = 0; j < C::E; j += 2) {  // two neighbouring dims: their bytes never straddle a 16-byte piece
                uint32_t pos = 0, neg = 0;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const int c = a[y] == 0.f ? 0 : static_cast<int>(fminf(fmaxf(rintf(x[y][j + z] / s), -127.0f), 127.0f));
                    pos |= (static_cast<uint32_t>(max(c, 0)) & 0xffu) << (8 * z);
                    neg |= (static_cast<uint32_t>(min(c, 0)) & 0xffu) << (8 * z);
                }
                auto place = [&](int k) {
                    const int kk = k & 127;
                    return smem + C::OFF_Q + (k >> 7) * C::Q_SLAB + (n >> 3) * 1024 + (n & 7) * 128 +
                           ((((kk >> 4) ^ (n & 7)) << 4) | (kk & 15));
                };
                *reinterpret_cast<uint16_t*>(place(lane * C::E + j)) = static_cast<uint16_t>(pos);
                *reinterpret_cast<uint16_t*>(place(C::D + lane * C::E + j)) = static_cast<uint16_t>(neg);
            }
            if (lane == 0) scales[n] = s;
        }
    }
}

template <int SL, int NQ>
__device__ __forceinline__ void score_epilogue(const SelectParams& p, uint8_t* smem, uint32_t tmem, Walk walk) {
    using C = ScoreCfg<SL, NQ>;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    const int r = threadIdx.x, warp = r >> 5, lane = r & 31;
    const int G = p.d.num_q_heads / p.d.num_kv_heads;
    for (int x = r; x < SL * C::Q_SLAB / 16; x += 128)  // heads past the group stay zero
        reinterpret_cast<uint4*>(smem + C::OFF_Q)[x] = make_uint4(0u, 0u, 0u, 0u);
    named_bar_sync(1, 128);
    Ring<2> acc;
    Ring<C::STEPS> steps;
    int parity = 0;
    ScoreItem I;
    while (next_part(p, walk, I)) {
        uint32_t* keys = p.keys + static_cast<int64_t>(I.row) * p.d.max_blocks_per_seq + I.i0;
        // The products of the part before have ended (this warp has read their sums). Scales alternate
        // between two places: a warp may still read those of the part before.
        float* scales = reinterpret_cast<float*>(smem + C::OFF_SQ) + parity * NQ;
        parity ^= 1;
        score_query<SL, NQ>(p, smem, I, scales);
        fence_async_smem();
        named_bar_sync(1, 128);
        if (lane == 0) mbar_arrive(&bars[C::B_Q]);
        float scale[8];
        bool finite = G <= 8;  // up to 8 heads with finite scales: no NaN can arise
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            scale[g] = g < G ? scales[g] : NAN;
            finite &= g >= G || isfinite(scale[g]);
        }
        for (int i = 0; i < I.m; i += 128) {
            if (!mbar_wait(&bars[C::B_STEP + steps.s], steps.phase)) return;
            const float step = reinterpret_cast<const float*>(smem + C::OFF_STEP)[steps.s * 128 + r];
            steps.next();
            if (!mbar_wait(&bars[C::B_ACC + acc.s], acc.phase)) return;
            tc_fence_after();
            float best = -INFINITY;
            const uint32_t sums_at = tmem + (static_cast<uint32_t>(warp * 32) << 16) + acc.s * NQ;
            if (finite) {  // a missing head's NaN scale leaves the maximum as it is
                uint32_t sums[8];
                tmem_ld8(sums_at, sums);
                tmem_wait_ld();
#pragma unroll
                for (int g = 0; g < 8; ++g) best = fmaxf(best, __int2float_rn(static_cast<int>(sums[g])) * scale[g]);
            } else {
                for (int g0 = 0; g0 < G; g0 += 8) {
                    uint32_t sums[8];
                    tmem_ld8(sums_at + g0, sums);
                    tmem_wait_ld();
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        const float v = __int2float_rn(static_cast<int>(sums[g])) * scales[min(g0 + g, NQ - 1)];
                        if (g0 + g < G) best = fmaxf(best, isnan(v) ? INFINITY : v);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[C::B_FREE + acc.s]);
            acc.next();
            if (i + r < I.m) keys[i + r] = step < 0.f ? kNoBlockKey : score_key(best * step);
        }
    }
}

template <int SL, int NQ>
__global__ void __launch_bounds__(ScoreCfg<SL, NQ>::THREADS, 1)
    score_tc_kernel(const SelectParams p) {
    using C = ScoreCfg<SL, NQ>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Walk s_walk;
    __shared__ int s_sums[C::THREADS / 32];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&bars[C::B_FULL + s], C::LW);  // loading warps
            mbar_init(&bars[C::B_EMPTY + s], 1);  // commit
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&bars[C::B_ACC + a], 1);
            mbar_init(&bars[C::B_FREE + a], 4);
        }
        for (int s = 0; s < C::STEPS; ++s) mbar_init(&bars[C::B_STEP + s], C::LW);
        mbar_init(&bars[C::B_Q], 4);
        mbar_init(&bars[C::B_DONE], 4);
        mbar_init(&bars[C::B_DRAIN], 1);
        fence_mbar_init();
    }
    if (warp == 4 + C::LW) tmem_alloc(reinterpret_cast<uint32_t*>(smem + C::OFF_TMEM), C::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + C::OFF_TMEM);
    // a programmatic dependent of the kernel before it: no global access before this
    grid_dependency_wait();
    allow_dependents();
    const Walk walk = first_part<C::THREADS>(p, &s_walk, s_sums);
    if (warp >= 4 && warp < 4 + C::LW) {
        score_loader<SL, NQ>(p, smem, walk, warp - 4);
    } else if (warp == 4 + C::LW) {
        score_mma<SL, NQ>(p, smem, tmem, walk);
        mma_commit_warp(&bars[C::B_DRAIN]);  // arrives once every product issued above has ended
        mbar_wait(&bars[C::B_DRAIN], 0);
        mbar_wait(&bars[C::B_DONE], 0);  // the other warps have read their sums
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    } else {
        score_epilogue<SL, NQ>(p, smem, tmem, walk);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[C::B_DONE]);
    }
}

template <int SL, int NQ>
cudaError_t launch_score(const SelectParams& p, cudaStream_t st) {
    using C = ScoreCfg<SL, NQ>;
    const kvd_block_select_desc& d = p.d;
    const int64_t rows = static_cast<int64_t>(d.batch) * d.num_kv_heads;
    const int64_t most = device_sm_count();
    const int64_t tiles = (d.max_blocks_per_seq + 127) / 128;
    if (rows * tiles > 0x7fff0000LL) return cudaErrorInvalidValue;
    auto kern = score_tc_kernel<SL, NQ>;
    static PerDeviceOnce once;
    const cudaError_t e = once.run(
        [kern] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES); });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * tiles < most ? rows * tiles : most), 1, 1);
    cfg.blockDim = dim3(C::THREADS, 1, 1);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int SL>
cudaError_t launch_score_g(const SelectParams& p, cudaStream_t st) {
    if (p.d.num_q_heads / p.d.num_kv_heads <= 16) return launch_score<SL, 16>(p, st);
    return launch_score<SL, 64>(p, st);
}

}  // namespace

bool score_tc_ok(const SelectParams& p) {
    const kvd_block_select_desc& d = p.d;
    if (d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 256) return false;
    if (d.num_q_heads / d.num_kv_heads > 64 || (reinterpret_cast<uintptr_t>(p.bounds) & 15) != 0) return false;
    return true;
}

cudaError_t launch_score_tc(const SelectParams& p, cudaStream_t st) {
    const kvd_block_select_desc& d = p.d;
    switch (d.head_dim) {
        case 64: return launch_score_g<1>(p, st);
        case 128: return launch_score_g<2>(p, st);
        default: return launch_score_g<4>(p, st);
    }
}

}  // namespace kvd
