// kvd_chunk_tile.cu -- attention of packed new tokens over a paged cache for
// requests with many rows a KV head, on the tcgen05 tensor cores.
//
// A unit is (request, KV head, block of rows, stretch of tokens); rows are the
// request's tokens times the group's heads, so a tile of the cache is read and
// widened once for all of them. With u_j = q . K_j (fp32 accumulators of fp16
// products; q times a power of two per row, codes exact), s_j = u_j ks_j rf in
// base 2 and p_j = 2^(s_j - m):
//   l = sum p_j,   O = sum fp16(p_j vs_j 2^e) V_j,   out = O 2^-e / l,
// with m a running maximum that may trail by 8 and 2^e a power of two that keeps
// the weights in fp16's range (it falls when larger value scales come).
//
// Outputs of 16 bits (TERMS 1): one fp16 term of the queries (exact for 16-bit
// ones) and of the weights; 256 rows, 128 to each of two softmax warpgroups,
// share a tile. Outputs of 32 bits or fp32 queries (TERMS 2): two terms of both
// (22 bits), 128 rows, the warpgroups take tiles in turn with their own m, l
// and O and are merged at the end. Blocks of at most 128 rows go that way too
// with one term. So there are always two score tiles in flight: while one
// warpgroup turns its scores into weights the tensor cores work for the other.
//
// One CTA an SM, 20 warps:
//   0-7   softmax, a row a thread (= TMEM lane): S from tensor memory, weights
//         back into the columns that S had, from where they are an MMA operand;
//   8-15  widen INT8 rows, straight from global memory (a tile ahead in
//         registers), into fp16 tiles in shared memory: 128-byte swizzled rows of
//         tokens, the K-major operand of q K^T and the MN-major one of P V; and
//         the unit's queries;
//   16    issues the MMAs;
//   17    takes units from a ticket that all CTAs share, for the whole CTA, and
//         looks its tiles' blocks up ahead: row offsets, scales.
// Outputs in bf16 (FOLD) have the value scales in the values, one multiplication
// where codes are widened instead of one for every row's weight: 4.33 ms instead
// of 5.36 for 4,096 new tokens of 32,768 (64 heads, 8 KV heads, 128 dims) when it
// was tried; fp16 outputs keep 3 more bits than those products would have. Tiles
// in which hidden tokens have the largest value scales are without it: there
// each row has an exponent of its own, from the tokens that it sees.
//
// Bound: latency. A step of 128 x 128 takes a warpgroup about 4,300 cycles, 2,600 to
// 3,000 of them in the softmax's chain (scores out of tensor memory, scales, the
// largest, exponentials, weights back; 3,900 where value scales multiply the
// weights, 6,500 with two terms), against 1,024 of products. No pipe is full, tensor
// 43 %, exponentials 43 %, issue slots 52 %: two softmax warps a scheduler do
// not cover each other's waits. Measured: those 4,096 tokens in 4.2 to 4.3 ms, 970
// TFLOP/s (4.7 in long runs, power cap); 512 of 8,192 in fp16 229 us; 7,003 tokens
// of five fp32 prompts (32 heads) 571 to 600 us, about 55 of them for sums put
// aside. When the 4,096 tokens took 5.4 ms: tiles of 64 tokens with two
// score buffers 8.0, votes per 32 columns 5.6, a row's pieces over lanes 5.6.
//
// Every wait is bounded; on expiry the kernel records KVD_STATUS_WAIT_TIMEOUT
// and unwinds.
#include "kvd_chunk.cuh"
#include "kvd_decode.cuh"
#include "kvd_tc.cuh"

namespace kvd {
namespace {

constexpr int kThreads = 640;
constexpr int kConvWarps = 8, kConvThreads = 32 * kConvWarps;
// Registers a thread has after the split, of 96 at launch: 256 x 136 + 256 x 72 + 128 x 64 = 640 x 96.
constexpr int kSoftmaxRegs = 136, kConvRegs = 72, kOtherRegs = 64;
static_assert(256 * kSoftmaxRegs + kConvThreads * kConvRegs + 128 * kOtherRegs <= kThreads * 96, "registers of the launch");
constexpr int kMetaStages = 4;
constexpr int kUnitStages = 4;

// What is known of a tile before it is read.
struct TileMeta {
    float ks[kTile];
    float vs[kTile];     // times 2^ve, or as they are where `vary`; 0 where it is not finite
    int64_t row[kTile];  // offset of the token's row in the pools; where there is none 0, and its scales are 0
    uint32_t odd[kTile / 32];  // tokens whose value scale is not finite
    int ve;
    int vary;  // tokens that some rows do not see have the largest scales: each row has an exponent of its own
    int pad[10];
};

template <int D>
struct TileSmem {
    static constexpr int kRows = 128 * D * 2;  // fp16 tile: 128 rows, D/64 columns of 128 bytes
    static constexpr int kQ = 0;               // [2]
    static constexpr int kK = 2 * kRows;       // [2]
    static constexpr int kV = 4 * kRows;       // [2]
    static constexpr int kMeta = 6 * kRows;
    static constexpr int kRf = kMeta + kMetaStages * static_cast<int>(sizeof(TileMeta));  // [2][256]
    static constexpr int kMl = kRf + 2 * 256 * 4;                                         // [2][128] m, l, ve
    static constexpr int kUnits = kMl + 2 * 128 * 16;  // [kUnitStages]
    static constexpr int kBar = kUnits + kUnitStages * 4;
    static constexpr int kBars = 2 * kMetaStages + 8 + 4 + 2 + 2 + 3 + 2 * kUnitStages;
    static constexpr int kTmem = kBar + kBars * 8;
    static constexpr int kBytes = kTmem + 16 + 1024;  // slack to align the base
};
static_assert(sizeof(TileMeta) % 16 == 0, "alignment");
static_assert(TileSmem<128>::kBytes <= 232448, "shared memory");

enum Bars {
    kMetaFull = 0,
    kMetaEmpty = kMetaFull + kMetaStages,
    kKFull = kMetaEmpty + kMetaStages,
    kKEmpty = kKFull + 2,
    kVFull = kKEmpty + 2,
    kVEmpty = kVFull + 2,
    kSFull = kVEmpty + 2,
    kPFull = kSFull + 2,
    kQFull = kPFull + 2,
    kQEmpty = kQFull + 1,
    kOFull = kQEmpty + 1,
    kMerge = kOFull + 2,
    kDone = kMerge + 1,
    kDrain = kDone + 1,
    kUnitFull = kDrain + 1,
    kUnitEmpty = kUnitFull + kUnitStages,
};

constexpr uint32_t kColO = 256;  // S and P: columns 0 and 128; O: 256 and 384

__host__ __device__ constexpr uint32_t idesc_fp16(int N, int M, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void mma_f16_ss_warp(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}

__device__ __forceinline__ bool mbar_wait_all(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int N>
__device__ __forceinline__ void regs_more() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_less() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

struct TileUnit {
    int b, hk, rb, split, nsplit, nrb;
    ChunkRows R;
    int rows;            // of the request and KV head
    int begin, end, nt;  // tokens, tiles
    int least;           // tokens in front of this one are seen by every row
    bool alt;            // the warpgroups take tiles in turn
};

// Later blocks of rows see more tokens and come first, so that the last units to be taken are short ones.
template <int TERMS>
__device__ __forceinline__ TileUnit tile_unit(const ChunkParams& p, int unit) {
    constexpr int ROWS = TERMS == 1 ? 256 : 128;
    TileUnit u;
    u.b = warp_find(p.first[kMany], p.B, unit);
    u.R = chunk_rows(p, u.b);
    u.rows = u.R.n * p.G;
    u.nrb = (u.rows + ROWS - 1) / ROWS;
    int each;
    u.nsplit = chunk_splits(u.R.len, p.head->span[kMany], kTile, each);
    int rest = unit - p.first[kMany][u.b];
    u.hk = rest % p.Hkv;
    rest /= p.Hkv;
    u.split = rest % u.nsplit;
    u.rb = u.nrb - 1 - rest / u.nsplit;
    const int last = min(u.rows, (u.rb + 1) * ROWS) - 1;
    const int most = chunk_sees(p, u.R, static_cast<int>(p.by_g.div(static_cast<uint32_t>(last))));
    u.begin = u.split * each;
    u.end = min(min(u.begin + each, u.R.len), most);
    u.least = min(u.end, chunk_sees(p, u.R, static_cast<int>(p.by_g.div(static_cast<uint32_t>(u.rb * ROWS)))));
    u.nt = u.end > u.begin ? (u.end - u.begin + kTile - 1) / kTile : 0;
    u.alt = TERMS == 2 || u.rows - u.rb * ROWS <= 128;
    return u;
}

// The CTA's n-th unit, -1 behind the last one, for a warp; every role's warps ask for all of them.
template <int D>
__device__ __forceinline__ int next_unit(uint8_t* smem, uint64_t* bars, int& n) {
    const int st = n & (kUnitStages - 1);
    if (!mbar_wait_all(&bars[kUnitFull + st], (n / kUnitStages) & 1)) return -1;
    const int unit = reinterpret_cast<const int*>(smem + TileSmem<D>::kUnits)[st];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&bars[kUnitEmpty + st]);
    ++n;
    return unit;
}

// ------------------------------------------------------------------ look-ahead
__device__ __forceinline__ void tile_scout(const ChunkParams& p, const TileUnit& u, TileMeta* meta, uint64_t* bars, int& j, bool& ok) {
    const int lane = threadIdx.x & 31;
    const int32_t* table = p.table + u.b * p.bt_stride;
    constexpr int N = kTile / 32;
    int id[N], off[N];
    auto look_up = [&](int i) {
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int t = u.begin + i * kTile + 32 * x + lane;
            id[x] = -1;
            off[x] = 0;
            if (t < u.end) {
                const int k = static_cast<int>(p.by_bs.div(static_cast<uint32_t>(t)));
                off[x] = t - k * p.bs;
                id[x] = table[k];
            }
        }
    };
    // Exponents for the scales of tokens that every row sees, and of all. Where the second is smaller, rows choose for
    // themselves, so that no hidden token costs a row bits. From then on it stays smaller: every later token is hidden
    // from some row.
    int ve = 126, ve_all = 126;
    look_up(0);
    for (int i = 0; i < u.nt && ok; ++i, ++j) {
        TileMeta* m = meta + (j & (kMetaStages - 1));
        float ks[N], vs[N];
        int64_t row[N];
        bool bad = false;
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const bool there = id[x] >= 0 && id[x] < p.NB;
            bad |= !there && u.begin + i * kTile + 32 * x + lane < u.end;
            const int64_t s = there ? id[x] * p.sc_sblk + u.hk * p.sc_sh + off[x] : 0;
            row[x] = there ? id[x] * p.kv_sblk + u.hk * p.kv_sh + off[x] * p.kv_st : 0;
            ks[x] = there ? p.ks[s] : 0.f;
            vs[x] = there ? p.vs[s] : 0.f;
        }
        if (bad) record_status(KVD_STATUS_BAD_BLOCK);
        if (i + 1 < u.nt) look_up(i + 1);  // on its way while this tile's scales come
        float top = 0.f, top_all = 0.f;
        uint32_t odd[N];
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const bool fine = fabsf(vs[x]) < INFINITY;
            odd[x] = __ballot_sync(0xffffffffu, !fine);
            if (!fine) vs[x] = 0.f;
            if (u.begin + i * kTile + 32 * x + lane < u.least) top = fmaxf(top, fabsf(vs[x]));
            top_all = fmaxf(top_all, fabsf(vs[x]));
        }
        const int bits = __reduce_max_sync(0xffffffffu, __float_as_int(top));
        const int bits_all = __reduce_max_sync(0xffffffffu, __float_as_int(top_all));
        if (bits != 0) ve = min(ve, fit_exponent(__int_as_float(bits), 7));
        if (bits_all != 0) ve_all = min(ve_all, fit_exponent(__int_as_float(bits_all), 7));
        const bool vary = ve_all < ve;
        const float f = vary ? 1.f : pow2i(ve);
        ok = j < kMetaStages || mbar_wait_all(&bars[kMetaEmpty + (j & (kMetaStages - 1))], ((j / kMetaStages) - 1) & 1);
        if (!ok) break;
#pragma unroll
        for (int x = 0; x < N; ++x) {
            m->ks[32 * x + lane] = ks[x];
            m->vs[32 * x + lane] = vs[x] * f;
            m->row[32 * x + lane] = row[x];
            if (lane == 0) m->odd[x] = odd[x];
        }
        if (lane == 0) {
            m->ve = ve;
            m->vary = vary;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kMetaFull + (j & (kMetaStages - 1))]);
    }
}

// ------------------------------------------------------------------ converters
// Place of 16-byte piece ch (of 8) of column col of row r in an fp16 tile.
__device__ __forceinline__ int piece_at(int r, int col, int ch) {
    return col * 16384 + (r >> 3) * 1024 + (r & 7) * 128 + ((ch ^ (r & 7)) << 4);
}

// Sixteen codes of row r, dims 16 c16 .., as two pieces; FOLD: times the row's scale, rounded.
template <bool FOLD>
__device__ __forceinline__ void store_codes(uint8_t* tile, int r, int c16, uint4 w, float scale) {
    uint4 a, b;
    const __half2 f = __float2half2_rn(scale);
    // words hold dims 4i..4i+3: pairs (0,1) and (2,3) in the order of the dims
    auto two = [f](uint32_t x, uint32_t& lo, uint32_t& hi) {
        const uint32_t y = x ^ 0x80808080u;
        uint32_t l = __byte_perm(y, 0x64646464u, 0x4140), h = __byte_perm(y, 0x64646464u, 0x4342);
        const __half2 k = __half2half2(__ushort_as_half(0x6480));
        __half2 hl = __hsub2(*reinterpret_cast<const __half2*>(&l), k), hh = __hsub2(*reinterpret_cast<const __half2*>(&h), k);
        if (FOLD) {
            hl = __hmul2(hl, f);
            hh = __hmul2(hh, f);
        }
        lo = *reinterpret_cast<const uint32_t*>(&hl);
        hi = *reinterpret_cast<const uint32_t*>(&hh);
    };
    two(w.x, a.x, a.y);
    two(w.y, a.z, a.w);
    two(w.z, b.x, b.y);
    two(w.w, b.z, b.w);
    const int col = c16 >> 2, ch = (c16 & 3) * 2;
    *reinterpret_cast<uint4*>(tile + piece_at(r, col, ch)) = a;
    *reinterpret_cast<uint4*>(tile + piece_at(r, col, ch + 1)) = b;
}

// The pieces of 16 codes that a thread takes of a tile. Eight lanes that store together take four pieces of a row
// of even number and the other four of the next one (all four of both at 64 dims), which are eight different places
// of the swizzle; a warp's loads cover whole rows.
template <int D>
struct Codes {
    static constexpr int PER = D / 16;                  // pieces of a row
    static constexpr int N = 128 * PER / kConvThreads;  // pieces a thread
    static constexpr int STEP = kConvThreads / PER;     // rows of all threads together
    uint4 w[N];
    static __device__ __forceinline__ void place(int ct, int& r, int& c16) {
        if constexpr (D == 128) {
            const int odd = (ct >> 2) & 1;
            r = 2 * (ct >> 4) + odd;
            c16 = (ct & 3) + 4 * (odd ^ ((ct >> 3) & 1));
        } else {
            r = ct >> 2;
            c16 = ct & 3;
        }
    }
    __device__ __forceinline__ void load(const int8_t* pool, const TileMeta* m, int ct) {
        int r, c16;
        place(ct, r, c16);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint4*>(pool + m->row[r + i * STEP] + c16 * 16);
    }
    template <bool FOLD>
    __device__ __forceinline__ void store(uint8_t* tile, int ct, const float* scale) const {
        int r, c16;
        place(ct, r, c16);
#pragma unroll
        for (int i = 0; i < N; ++i) store_codes<FOLD>(tile, r + i * STEP, c16, w[i], FOLD ? scale[r + i * STEP] : 0.f);
    }
};

// The unit's rows as fp16, each times its power of two, and what the scores are multiplied with instead.
template <int D, int TERMS>
__device__ __forceinline__ void load_queries(const ChunkParams& p, const TileUnit& u, uint8_t* q, float* rf, int ct) {
    constexpr int ROWS = TERMS == 1 ? 256 : 128;
    constexpr int PER = D / 16;
    const int there = min(ROWS, u.rows - u.rb * ROWS), most = TERMS == 1 && there > 128 ? 256 : 128;
    const int c16 = ct % PER;
#pragma unroll 1
    for (int r = ct / PER; r < most; r += kConvThreads / PER) {
        float x[16];
#pragma unroll
        for (int d = 0; d < 16; ++d) x[d] = 0.f;
        if (r < there) {
            const int row = u.rb * ROWS + r;
            const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(row))), g = row - i * p.G;
            const int64_t at = static_cast<int64_t>(u.R.t0 + i) * p.q_st + static_cast<int64_t>(u.hk * p.G + g) * p.q_sh + c16 * 16;
            if (!p.vec_q) {
#pragma unroll
                for (int d = 0; d < 16; ++d) x[d] = load_q(p.Q, at + d, p.flags);
            } else if (p.flags & (KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16)) {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.Q) + at);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint4 v = src[k];
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        float2 f;
                        if (p.flags & KVD_FLAG_Q_BF16)
                            f = make_float2(__uint_as_float(w[y] << 16), __uint_as_float(w[y] & 0xffff0000u));
                        else
                            f = __half22float2(*reinterpret_cast<const __half2*>(&w[y]));
                        x[8 * k + 2 * y] = f.x;
                        x[8 * k + 2 * y + 1] = f.y;
                    }
                }
            } else {
                const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.Q) + at);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float4 v = src[k];
                    x[4 * k] = v.x; x[4 * k + 1] = v.y; x[4 * k + 2] = v.z; x[4 * k + 3] = v.w;
                }
            }
        }
        float top = 0.f;
#pragma unroll
        for (int d = 0; d < 16; ++d) top = fmaxf(top, fabsf(x[d]));
#pragma unroll
        for (int o = 1; o < PER; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // Two terms (32-bit rows): whole numbers up to 2^11 and what is left. A product's sum is cut off, not rounded,
        // behind every step, by a unit of its size, which whole numbers alone would not feel below 2^24.
        const bool whole = TERMS == 2 && (p.flags & (KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16)) == 0;
        const int k = fit_exponent(top, whole ? 11 : 15);
        const float f = pow2i(k);
        if (c16 == 0) rf[r] = fmaxf(p.qscale * pow2i(-k), 0x1p-126f);  // never 0, which would make -inf times it NaN
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const float a = x[2 * d] * f, b = x[2 * d + 1] * f;
            hi[d] = whole ? pack_half(rintf(a), rintf(b)) : pack_half(a, b);
            if (TERMS == 2) lo[d] = pack_rest(a, b, hi[d]);
        }
        uint8_t* tile = q + (r >> 7) * TileSmem<D>::kRows;
        const int col = c16 >> 2, ch = (c16 & 3) * 2, rr = r & 127;
        *reinterpret_cast<uint4*>(tile + piece_at(rr, col, ch)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(tile + piece_at(rr, col, ch + 1)) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
        if constexpr (TERMS == 2) {
            uint8_t* rest = q + TileSmem<D>::kRows;
            *reinterpret_cast<uint4*>(rest + piece_at(rr, col, ch)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            *reinterpret_cast<uint4*>(rest + piece_at(rr, col, ch + 1)) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
        }
    }
}

// Tiles in the order in which the MMAs want them: K of the first two, then V of a tile and K of the second next.
template <int D, int TERMS, bool FOLD>
__device__ __forceinline__ bool tile_convert(const ChunkParams& p, const TileUnit& u, uint8_t* smem, uint64_t* bars, int j0, int nu) {
    using S = TileSmem<D>;
    const int ct = threadIdx.x - 256, lane = ct & 31;
    const TileMeta* meta = reinterpret_cast<const TileMeta*>(smem + S::kMeta);
    const int jobs = 2 * u.nt;
    auto job = [&](int q, int& tile, bool& v) {
        v = q == jobs - 1 || (q >= 2 && (q & 1) == 0);
        tile = v ? (q == jobs - 1 ? u.nt - 1 : (q - 2) >> 1) : (q == 0 ? 0 : (q + 1) >> 1);
    };
    auto load = [&](int q, Codes<D>& c) -> bool {
        if (q >= jobs) return true;
        int tile;
        bool v;
        job(q, tile, v);
        const int j = j0 + tile, st = j & (kMetaStages - 1);
        if (!v && !mbar_wait(&bars[kMetaFull + st], (j / kMetaStages) & 1)) return false;
        c.load(v ? p.V : p.K, meta + st, ct);
        if (v && !FOLD) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[kMetaEmpty + st]);
        }
        return true;
    };
    auto store = [&](int q, const Codes<D>& c) -> bool {
        int tile;
        bool v;
        job(q, tile, v);
        const int j = j0 + tile, st = j & 1;
        if (j >= 2 && !mbar_wait(&bars[(v ? kVEmpty : kKEmpty) + st], ((j >> 1) - 1) & 1)) return false;
        uint8_t* to = smem + (v ? S::kV : S::kK) + st * S::kRows;
        // (where exponents vary the value scales are the weights')
        if (FOLD && v && !(u.begin + (tile + 1) * kTile > u.least && meta[j & (kMetaStages - 1)].vary))
            c.template store<true>(to, ct, meta[j & (kMetaStages - 1)].vs);
        else c.template store<false>(to, ct, nullptr);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&bars[(v ? kVFull : kKFull) + st]);
            if (FOLD && v) mbar_arrive(&bars[kMetaEmpty + (j & (kMetaStages - 1))]);
        }
        return true;
    };
    Codes<D> a, b;
    if (!load(0, a)) return false;
    if (nu > 0 && !mbar_wait(&bars[kQEmpty], (nu - 1) & 1)) return false;
    load_queries<D, TERMS>(p, u, smem + S::kQ, reinterpret_cast<float*>(smem + S::kRf) + (nu & 1) * 256, ct);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[kQFull]);
#pragma unroll 1
    for (int q = 0; q < jobs; q += 2) {  // an even number of jobs
        if (!load(q + 1, b) || !store(q, a) || !load(q + 2, a) || !store(q + 1, b)) return false;
    }
    return true;
}

// ------------------------------------------------------------------ MMA issuer
// Step i works for warpgroup i & 1: on tile i when the warpgroups take tiles in turn, else on tile i / 2. The
// scores of step i + 2 are issued behind the weights' product of step i, which reads the columns they overwrite.
template <int D, int TERMS>
__device__ __forceinline__ bool tile_mma(const TileUnit& u, uint8_t* smem, uint32_t tmem, uint64_t* bars, int j0, int nu, int (&np)[2], int nq) {
    using S = TileSmem<D>;
    constexpr uint32_t id_s = idesc_fp16(kTile, 128, false), id_o = idesc_fp16(D, 128, true);
    const int steps = u.alt ? u.nt : 2 * u.nt;
    if (!mbar_wait_all(&bars[kQFull], nu & 1)) return false;
    auto scores = [&](int i) -> bool {
        const int w = i & 1, j = j0 + (u.alt ? i : i >> 1), st = j & 1;
        if ((u.alt || w == 0) && !mbar_wait_all(&bars[kKFull + st], (j >> 1) & 1)) return false;
        tc_fence_after();
        const uint64_t kd = smem_desc(smem_u32(smem + S::kK + st * S::kRows), 16u, 1024u, kLayoutSw128);
        // The smaller term first: errors of 9.7e-7 against 3.3e-6 for scores of hundreds, of 6.0e-7 against 8.5e-7 for
        // ordinary ones (128 dims; fp32 matrix products 2.9e-6 and 5.1e-7).
#pragma unroll
        for (int t = TERMS - 1; t >= 0; --t) {
            if (t < nq) {
                const int tile = TERMS == 2 ? t : (u.alt ? 0 : w);
                const uint64_t qd = smem_desc(smem_u32(smem + S::kQ + tile * S::kRows), 16u, 1024u, kLayoutSw128);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint64_t step = ((k >> 2) * 16384u + (k & 3) * 32u) >> 4;
                    mma_f16_ss_warp(tmem + w * 128u, qd + step, kd + step, id_s, t < nq - 1 || k > 0);
                }
            }
        }
        mma_commit_warp(&bars[kSFull + w]);
        if (u.alt || w == 1) mma_commit_warp(&bars[kKEmpty + st]);
        return true;
    };
    if (!scores(0)) return false;
    if (steps > 1 && !scores(1)) return false;
    bool loaded = true;  // the unit's queries are still needed
    for (int i = 0; i < steps; ++i) {
        const int w = i & 1, j = j0 + (u.alt ? i : i >> 1), st = j & 1;
        if (!mbar_wait_all(&bars[kPFull + w], np[w] & 1)) return false;
        ++np[w];
        if ((u.alt || w == 0) && !mbar_wait_all(&bars[kVFull + st], (j >> 1) & 1)) return false;
        tc_fence_after();
        // 16 tokens: two groups of 8 rows (1,024 bytes each); dims 64.. one column on
        const uint64_t vd = smem_desc(smem_u32(smem + S::kV + st * S::kRows), 16384u, 1024u, kLayoutSw128);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
                mma_f16_ts_warp(tmem + kColO + w * 128u, tmem + w * 128u + 64u * t + 8u * k, vd + (2048u * k >> 4), id_o,
                                i >= 2 || t > 0 || k > 0);
        if (u.alt || w == 1) mma_commit_warp(&bars[kVEmpty + st]);
        if (i + 2 < steps) {
            if (!scores(i + 2)) return false;
        } else {
            mma_commit_warp(&bars[kOFull + w]);
        }
        // Behind the last scores, and behind weights of every warpgroup that has any: these have then waited for
        // this unit's queries, whose barrier may not complete twice before they do.
        if (loaded && i + 3 >= steps && (i >= 1 || steps == 1)) {
            mma_commit_warp(&bars[kQEmpty]);
            loaded = false;
        }
    }
    return true;
}

// ------------------------------------------------------------------ softmax
// Columns d0 .. d0 + 31 of a row.
__device__ __forceinline__ void store_row32(const ChunkParams& p, int64_t at, const float (&x)[32]) {
    const bool o16 = (p.flags & (KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16)) != 0;
    if (!p.vec_out) {
#pragma unroll
        for (int d = 0; d < 32; ++d) store_out(p.out, at + d, x[d], p.flags);
    } else if (!o16) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
#pragma unroll
        for (int d = 0; d < 8; ++d) dst[d] = make_float4(x[4 * d], x[4 * d + 1], x[4 * d + 2], x[4 * d + 3]);
    } else {
        uint32_t w[16];
#pragma unroll
        for (int d = 0; d < 16; ++d) {
            if (p.flags & KVD_FLAG_OUT_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * d], x[2 * d + 1]);
                w[d] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                w[d] = pack_half(x[2 * d], x[2 * d + 1]);
            }
        }
        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at);
#pragma unroll
        for (int d = 0; d < 4; ++d) dst[d] = make_uint4(w[4 * d], w[4 * d + 1], w[4 * d + 2], w[4 * d + 3]);
    }
}

// Scores of 32 tokens of this thread's row: the largest u ks (raw products times the tokens' scales) of the first
// `lim` ones.
template <bool MASK>
__device__ __forceinline__ float top32(uint32_t col, const float4* ks4, int lim) {
    uint32_t s[32];
    tmem_ld32(col, s);
    tmem_wait_ld();
    float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float4 kq = ks4[k];
        const float2 a = __fmul2_rn(make_float2(__uint_as_float(s[4 * k]), __uint_as_float(s[4 * k + 1])), make_float2(kq.x, kq.y));
        const float2 b = __fmul2_rn(make_float2(__uint_as_float(s[4 * k + 2]), __uint_as_float(s[4 * k + 3])), make_float2(kq.z, kq.w));
        const float v0 = !MASK || 4 * k < lim ? a.x : -INFINITY, v1 = !MASK || 4 * k + 1 < lim ? a.y : -INFINITY;
        const float v2 = !MASK || 4 * k + 2 < lim ? b.x : -INFINITY, v3 = !MASK || 4 * k + 3 < lim ? b.y : -INFINITY;
        tm[k & 1] = max3(max3(tm[k & 1], v0, v1), v2, v3);
    }
    return fmaxf(tm[0], tm[1]);
}

// Weights of 32 tokens with reference m: their sum onto `sum`, p vs 2^ve as fp16 pairs (and their rests). Returns
// the largest u ks. MASK: the first `lim` tokens only; vf is 2^ve where the exponent is the row's own (`vary`), else 1.
template <bool MASK, bool FOLD>
__device__ __forceinline__ float weights32(uint32_t col, const float4* ks4, const float4* vs4, int lim, float vf, bool vary, float rf,
                                           float m, float2 (&sum)[2], uint32_t (&hi)[16], uint32_t* lo) {
    uint32_t s[32];
    tmem_ld32(col, s);
    tmem_wait_ld();
    const float2 nm = make_float2(-m, -m), rf2 = make_float2(rf, rf);
    float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float4 kq = ks4[k];
        float4 vq = make_float4(1.f, 1.f, 1.f, 1.f);
        if (!FOLD || (MASK && vary)) vq = vs4[k];
        if (MASK)  // a hidden token's scale may be too large for 2^ve
            vq = make_float4(4 * k < lim ? vq.x * vf : 0.f, 4 * k + 1 < lim ? vq.y * vf : 0.f, 4 * k + 2 < lim ? vq.z * vf : 0.f,
                             4 * k + 3 < lim ? vq.w * vf : 0.f);
        float2 a = __fmul2_rn(make_float2(__uint_as_float(s[4 * k]), __uint_as_float(s[4 * k + 1])), make_float2(kq.x, kq.y));
        float2 b = __fmul2_rn(make_float2(__uint_as_float(s[4 * k + 2]), __uint_as_float(s[4 * k + 3])), make_float2(kq.z, kq.w));
        if (MASK) {
            a = make_float2(4 * k < lim ? a.x : -INFINITY, 4 * k + 1 < lim ? a.y : -INFINITY);
            b = make_float2(4 * k + 2 < lim ? b.x : -INFINITY, 4 * k + 3 < lim ? b.y : -INFINITY);
        }
        tm[k & 1] = max3(max3(tm[k & 1], a.x, a.y), b.x, b.y);
        a = __ffma2_rn(a, rf2, nm);
        b = __ffma2_rn(b, rf2, nm);
        const float2 pa = make_float2(ex2_fast(a.x), ex2_fast(a.y)), pb = make_float2(ex2_fast(b.x), ex2_fast(b.y));
        sum[0] = __fadd2_rn(sum[0], pa);
        sum[1] = __fadd2_rn(sum[1], pb);
        const bool plain = FOLD && !MASK;
        const float2 x = plain ? pa : __fmul2_rn(pa, make_float2(vq.x, vq.y)), y = plain ? pb : __fmul2_rn(pb, make_float2(vq.z, vq.w));
        hi[2 * k] = pack_half(x.x, x.y);
        hi[2 * k + 1] = pack_half(y.x, y.y);
        if (lo) {
            lo[2 * k] = pack_rest(x.x, x.y, hi[2 * k]);
            lo[2 * k + 1] = pack_rest(y.x, y.y, hi[2 * k + 1]);
        }
    }
    return fmaxf(tm[0], tm[1]);
}

// 32 columns of a warp's 32 rows in pieces: lane l has rows l/4, +8, +16, +24 and, of every eight columns, 2 (l % 4)
// and the next one.
__device__ __forceinline__ void tmem_ld_rows(uint32_t col, uint32_t (&r)[32]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[16 * h]), "=r"(r[16 * h + 1]), "=r"(r[16 * h + 2]), "=r"(r[16 * h + 3]), "=r"(r[16 * h + 4]),
              "=r"(r[16 * h + 5]), "=r"(r[16 * h + 6]), "=r"(r[16 * h + 7]), "=r"(r[16 * h + 8]), "=r"(r[16 * h + 9]),
              "=r"(r[16 * h + 10]), "=r"(r[16 * h + 11]), "=r"(r[16 * h + 12]), "=r"(r[16 * h + 13]),
              "=r"(r[16 * h + 14]), "=r"(r[16 * h + 15])
            : "r"(col + (static_cast<uint32_t>(16 * h) << 16)));
}

// The two softmax warpgroups meet (a bounded wait).
__device__ __forceinline__ bool both_here(uint64_t* bars, int& count) {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&bars[kMerge]);
    const bool ok = mbar_wait(&bars[kMerge], count & 1);
    ++count;
    tc_fence_after();
    return ok;
}

// What sums that were put aside with the reference and the exponent `of` (x, z) are worth with these.
__device__ __forceinline__ float aside_factor(const float4& of, float m, int ve) {
    const int fall = __float_as_int(of.z) - ve;
    return of.x == -INFINITY || fall > 126 ? 0.f : ex2_fast(of.x - m) * pow2i(-fall);
}

// Adds this thread's row of O to the sums that it has put aside, and starts O again from zero. The sums keep the
// reference and exponent of the first time (`of`), which O is raised to on its way, so that nothing waits for
// them; once that is too far, they are read and lowered instead.
template <int D>
__device__ __forceinline__ void put_aside(float4* aside, float4* of, uint32_t col_o, bool first, float m, int ve) {
    float f = 0.f;  // times the old sums, or times O
    bool read = false;
    if (!first) {
        const float4 was = *of;
        const float up = m - was.x;
        const int fall = __float_as_int(was.z) - ve;
        read = __any_sync(0xffffffffu, m != -INFINITY && !(up + static_cast<float>(fall) <= 60.f));
        f = read ? aside_factor(was, m, ve) : m == -INFINITY ? 0.f : ex2_fast(up) * pow2i(fall);
    }
    if (first || read) *of = make_float4(m, 0.f, __int_as_float(ve), 0.f);
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
        uint32_t o[32];
        tmem_ld32(col_o + d, o);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
            float4* at = aside + (d + x) / 4 * 128;
            float4 y = make_float4(__uint_as_float(o[x]), __uint_as_float(o[x + 1]), __uint_as_float(o[x + 2]), __uint_as_float(o[x + 3]));
            if (first || read) {
                if (f != 0.f) {
                    const float4 z = __ldcg(at);
                    y = make_float4(fmaf(z.x, f, y.x), fmaf(z.y, f, y.y), fmaf(z.z, f, y.z), fmaf(z.w, f, y.w));
                }
                __stcg(at, y);
            } else {
                asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(y.x * f), "f"(y.y * f),
                             "f"(y.z * f), "f"(y.w * f) : "memory");
            }
            o[x] = o[x + 1] = o[x + 2] = o[x + 3] = 0u;
        }
        tmem_st32(col_o + d, o);
    }
    tmem_wait_st();  // O may be read again in the same tile, and only this wait puts a load behind the stores
}

template <int D, int TERMS, bool FOLD>
__device__ __forceinline__ bool tile_softmax(const ChunkParams& p, const TileUnit& u, uint8_t* smem, uint32_t tmem, uint64_t* bars, int j0,
                                             int nu, int& ns, int& no, int& nm_sync) {
    using S = TileSmem<D>;
    constexpr int ROWS = TERMS == 1 ? 256 : 128;
    // Weights up to 2^8 times value scales below 2^7 fit fp16. Weights without the scales have the room of these, so the
    // reference lies 2^7 below the largest score: small ones stay normal numbers for as long as the others do.
    constexpr int kBelow = FOLD ? 7 : 0;
    const int w = threadIdx.x >> 7, r = threadIdx.x & 127, lane = r & 31;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(r & ~31) << 16);
    const uint32_t col_s = lanes + w * 128u, col_o = lanes + kColO + w * 128u;
    const TileMeta* meta = reinterpret_cast<const TileMeta*>(smem + S::kMeta);
    const int in_unit = u.alt ? r : w * 128 + r, row = u.rb * ROWS + in_unit;
    const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(row))), g = row - i * p.G;
    const bool there = row < u.rows;
    const int64_t o_at = static_cast<int64_t>(u.R.t0 + i) * p.o_st + static_cast<int64_t>(u.hk * p.G + g) * p.o_sh;
    const int slot = u.nsplit > 1 ? p.rec[kMany][u.b] + (u.hk * u.nrb + u.rb) * u.nsplit + u.split : -1;
    const int64_t rec = static_cast<int64_t>(slot) * ROWS + in_unit;
    if (u.nt == 0) {  // nothing in sight
        if (there && (!u.alt || w == 0)) {
            if (slot >= 0) {
                p.part_ml[kMany][rec] = make_float2(-INFINITY, 0.f);
            } else {
                const float none[32] = {};
#pragma unroll 1
                for (int d = 0; d < D; d += 32) store_row32(p, o_at + d, none);
            }
        }
        return true;
    }
    // (a warpgroup without tiles does not wait: nothing holds the barrier up for it)
    if ((!u.alt || w < u.nt) && !mbar_wait(&bars[kQFull], nu & 1)) return false;
    const float rf = reinterpret_cast<const float*>(smem + S::kRf)[(nu & 1) * 256 + in_unit];
    const int sees = chunk_sees(p, u.R, min(i, u.R.n - 1));  // rows that are not there see what the last one does
    float m = -INFINITY;
    // One term: sums of a thread's four tokens in turn (few tiles add to them one token at a time). Two: one sum.
    float2 lp[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    float l = 0.f;
    int ve = 126;
    bool any = false;  // O holds sums of this unit
    for (int tile = u.alt ? w : 0; tile < u.nt; tile += u.alt ? 2 : 1) {
        const int j = j0 + tile, st = j & (kMetaStages - 1), t0 = u.begin + tile * kTile;
        if (!mbar_wait(&bars[kMetaFull + st], (j / kMetaStages) & 1)) return false;
        const float4* ks4 = reinterpret_cast<const float4*>(meta[st].ks);
        const float4* vs4 = reinterpret_cast<const float4*>(meta[st].vs);
        const int lim = min(sees, u.end) - t0;  // tokens of the tile that the row sees
        const bool masked = t0 + kTile > u.least;
        if (!mbar_wait(&bars[kSFull + w], ns & 1)) return false;
        ++ns;
        tc_fence_after();
        const int own_tile = u.alt ? tile >> 1 : tile;
        const bool full = own_tile != 0 && (own_tile & (p.aside_tiles - 1)) == 0;  // O holds as many as it should
        bool done = false;
        if constexpr (TERMS == 1) {
            // With the reference of the tiles before: one pass. It stands unless a score is above it by more than 8.
            if (!masked && !full && __all_sync(0xffffffffu, m != -INFINITY) && meta[st].ve == ve) {
                uint32_t pk[kTile / 2];
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                float top = -INFINITY;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    top = fmaxf(top, weights32<false, FOLD>(col_s + 32u * q, ks4 + 8 * q, vs4 + 8 * q, 0, 1.f, false, rf, m, sum,
                                                      *reinterpret_cast<uint32_t(*)[16]>(&pk[16 * q]), nullptr));
                done = !__any_sync(0xffffffffu, top * rf > m + (8.f + kBelow));
                if (done) {
                    lp[0] = __fadd2_rn(lp[0], sum[0]);
                    lp[1] = __fadd2_rn(lp[1], sum[1]);
                    tmem_st32(col_s, *reinterpret_cast<uint32_t(*)[32]>(&pk[0]));
                    tmem_st32(col_s + 32u, *reinterpret_cast<uint32_t(*)[32]>(&pk[32]));
                }
            }
        }
        if (!done) {
            int ve_now = meta[st].ve;
            const bool vary = masked && meta[st].vary;
            if (vary) {
                float seen = 0.f;
#pragma unroll 4
                for (int x = 0; x < kTile / 4; ++x) {
                    const float4 v = vs4[x];
                    if (4 * x < lim) seen = fmaxf(seen, fabsf(v.x));
                    if (4 * x + 1 < lim) seen = fmaxf(seen, fabsf(v.y));
                    if (4 * x + 2 < lim) seen = fmaxf(seen, fabsf(v.z));
                    if (4 * x + 3 < lim) seen = fmaxf(seen, fabsf(v.w));
                }
                ve_now = seen == 0.f ? ve : min(ve, fit_exponent(seen, 7 - kBelow));
            }
            const float vf = vary ? pow2i(ve_now) : 1.f;
            float top = -INFINITY;
            if (masked) {
#pragma unroll 1
                for (int q = 0; q < 4; ++q) top = fmaxf(top, top32<true>(col_s + 32u * q, ks4 + 8 * q, lim - 32 * q));
            } else {
#pragma unroll 1
                for (int q = 0; q < 4; ++q) top = fmaxf(top, top32<false>(col_s + 32u * q, ks4 + 8 * q, 0));
            }
            top *= rf;  // rf > 0: -inf stays
            if (full)  // this warpgroup's products before this tile's scores are complete: O may change
                put_aside<D>(p.aside + (blockIdx.x * 2 + w) * (D / 4) * 128 + r, reinterpret_cast<float4*>(smem + S::kMl) + w * 128 + r,
                             col_o, own_tile == p.aside_tiles, m, ve);
            const bool move = top > m + (m == -INFINITY ? 0.f : 8.f + kBelow);
            const float to = top - kBelow;
            if (any && __any_sync(0xffffffffu, (move && m != -INFINITY) || ve_now != ve)) {
                // this warpgroup's products before this tile's scores are complete: O may change
                const float f = move && m != -INFINITY ? ex2_fast(m - to) : 1.f;
                const float fo = f * (ve - ve_now > 126 ? 0.f : pow2i(ve_now - ve));
#pragma unroll 1
                for (int d = 0; d < D; d += 32) {
                    uint32_t o[32];
                    tmem_ld32(col_o + d, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * fo);
                    tmem_st32(col_o + d, o);
                }
                if constexpr (TERMS == 1) {
                    lp[0] = __fmul2_rn(lp[0], make_float2(f, f));
                    lp[1] = __fmul2_rn(lp[1], make_float2(f, f));
                } else {
                    l *= f;
                }
            }
            ve = ve_now;
            if (move) m = to;
            const float me = m == -INFINITY ? 0.f : m;
            // two terms: small weights of a tile are added to each other before they meet a sum that may be far larger
            float2 two[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            float2(&tp)[2] = TERMS == 1 ? lp : two;
            // hidden tokens (weight 0) and their value scales, which are finite here, leave no trace
            uint32_t hi[16], rest[TERMS == 2 ? 3 : 1][16];
            // (one copy of this rare path where it can be: unrolled, its registers cost the path above 500 us of 4,790)
#pragma unroll (TERMS == 2 ? 4 : 1)
            for (int q = 0; q < 4; ++q) {
                uint32_t* lo = TERMS == 2 ? rest[q < 3 ? q : 2] : nullptr;
                if (TERMS == 2 && q == 3) {  // the columns that these terms go to have been read by now
                    tmem_st16(col_s + 64u, rest[0]);
                    tmem_st16(col_s + 80u, rest[1]);
                    uint32_t last[16];
                    if (masked) weights32<true, FOLD>(col_s + 96u, ks4 + 24, vs4 + 24, lim - 96, vf, vary, rf, me, tp, hi, last);
                    else weights32<false, FOLD>(col_s + 96u, ks4 + 24, vs4 + 24, 0, 1.f, false, rf, me, tp, hi, last);
                    tmem_st16(col_s + 96u, rest[2]);
                    tmem_st16(col_s + 112u, last);
                } else if (masked) {
                    weights32<true, FOLD>(col_s + 32u * q, ks4 + 8 * q, vs4 + 8 * q, lim - 32 * q, vf, vary, rf, me, tp, hi, lo);
                } else {
                    weights32<false, FOLD>(col_s + 32u * q, ks4 + 8 * q, vs4 + 8 * q, 0, 1.f, false, rf, me, tp, hi, lo);
                }
                tmem_st16(col_s + 16u * q, hi);
            }
            if (TERMS == 2) l += (tp[0].x + tp[0].y) + (tp[1].x + tp[1].y);
        }
        any = true;
        if (meta[st].odd[0] | meta[st].odd[1] | meta[st].odd[2] | meta[st].odd[3]) {
#pragma unroll
            for (int x = 0; x < kTile / 32; ++x) {
                const int n = lim - 32 * x;
                if (meta[st].odd[x] & (n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u)) (TERMS == 1 ? lp[0].x : l) = NAN;
            }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&bars[kPFull + w]);
            mbar_arrive_n(&bars[kMetaEmpty + st], u.alt ? 2u : 1u);
        }
    }
    // ---- the rows
    if (any) {
        if (!mbar_wait(&bars[kOFull + w], no & 1)) return false;
        ++no;
    }
    tc_fence_after();
    if ((u.alt ? (u.nt - w + 1) / 2 : u.nt) > p.aside_tiles) {  // sums were put aside: they come back
        const float4* aside = p.aside + (blockIdx.x * 2 + w) * (D / 4) * 128 + r;
        const float f = aside_factor(reinterpret_cast<const float4*>(smem + S::kMl)[w * 128 + r], m, ve);
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
            uint32_t o[32];
            tmem_ld32(col_o + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; x += 4) {
                const float4 y = __ldcg(aside + (d + x) / 4 * 128);
                if (f != 0.f) {
                    o[x] = __float_as_uint(fmaf(y.x, f, __uint_as_float(o[x])));
                    o[x + 1] = __float_as_uint(fmaf(y.y, f, __uint_as_float(o[x + 1])));
                    o[x + 2] = __float_as_uint(fmaf(y.z, f, __uint_as_float(o[x + 2])));
                    o[x + 3] = __float_as_uint(fmaf(y.w, f, __uint_as_float(o[x + 3])));
                }
            }
            tmem_st32(col_o + d, o);
        }
        tmem_wait_st();
    }
    if (TERMS == 1) l = (lp[0].x + lp[0].y) + (lp[1].x + lp[1].y);
    float back = pow2i(-ve), other_back = 0.f;
    int d0 = 0, d1 = D;
    if (u.alt) {  // the two warpgroups' sums, half of the dims each
        float4* ml = reinterpret_cast<float4*>(smem + S::kMl);
        ml[w * 128 + r] = make_float4(m, l, __int_as_float(ve), 0.f);
        if (!both_here(bars, nm_sync)) return false;
        const float4 other = ml[(w ^ 1) * 128 + r];
        const int other_ve = __float_as_int(other.z);
        const float M = fmaxf(m, other.x);
        const float f0 = m == -INFINITY ? 0.f : ex2_fast(m - M), f1 = other.x == -INFINITY ? 0.f : ex2_fast(other.x - M);
        l = l * f0 + other.y * f1;
        m = M;
        back *= f0;
        other_back = u.nt > 1 ? pow2i(-other_ve) * f1 : 0.f;
        if (!any) back = 0.f;
        if (any && u.nt == 1) other_back = 0.f;
        if (!any) other_back = pow2i(-other_ve) * f1;
        d0 = w * (D / 2);
        d1 = d0 + D / 2;
    }
    const float inv = slot >= 0 ? 1.f : (l == 0.f ? 0.f : 1.f / l);  // no token in sight: 0; NaN stays
    const bool both = u.alt && u.nt > 1;
    const uint32_t own = lanes + kColO + (u.alt && !any ? (w ^ 1) : w) * 128u, second = lanes + kColO + (w ^ 1) * 128u;
    const float own_back = u.alt && !any ? other_back : back;
    if constexpr (TERMS == 2)
    if ((slot >= 0 || (p.vec_out && (p.flags & (KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16)) == 0))) {
        // 32-bit rows: four lanes write 32 bytes of a row together, where a row a lane would write half sectors
        // (one term has no registers left for this)
        float* row_to = !there ? nullptr : slot >= 0 ? p.part_o[kMany] + rec * D : static_cast<float*>(p.out) + o_at;
        float fa[4], fb[4];
        float* to[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int from = 8 * i + (lane >> 2);
            fa[i] = __shfl_sync(0xffffffffu, own_back * inv, from);
            fb[i] = __shfl_sync(0xffffffffu, other_back * inv, from);
            to[i] = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row_to), from));
        }
#pragma unroll 1
        for (int d = d0; d < d1; d += 32) {
            uint32_t o[32], o2[32];
            tmem_ld_rows(own + d, o);
            if (both) tmem_ld_rows(second + d, o2);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; y += 2) {
                const int i = 2 * (y >> 4) + ((y >> 1) & 1), k = (y >> 2) & 3;
                float2 x = fa[i] == 0.f ? make_float2(0.f, 0.f) : make_float2(__uint_as_float(o[y]) * fa[i], __uint_as_float(o[y + 1]) * fa[i]);
                if (both && fb[i] != 0.f)
                    x = make_float2(fmaf(__uint_as_float(o2[y]), fb[i], x.x), fmaf(__uint_as_float(o2[y + 1]), fb[i], x.y));
                if (to[i]) *reinterpret_cast<float2*>(to[i] + d + 8 * k + 2 * (lane & 3)) = x;
            }
        }
        d1 = d0;  // done
    }
#pragma unroll 1
    for (int d = d0; d < d1; d += 32) {
        float x[32];
        {
            uint32_t o[32];
            tmem_ld32(own + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; ++y) x[y] = own_back == 0.f ? 0.f : __uint_as_float(o[y]) * own_back;
        }
        if (both) {
            uint32_t o[32];
            tmem_ld32(second + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; ++y) x[y] = other_back == 0.f ? x[y] : fmaf(__uint_as_float(o[y]), other_back, x[y]);
        }
        if (there) {
            if (slot >= 0) {
                float4* dst = reinterpret_cast<float4*>(p.part_o[kMany] + rec * D + d);
#pragma unroll
                for (int y = 0; y < 8; ++y) dst[y] = make_float4(x[4 * y], x[4 * y + 1], x[4 * y + 2], x[4 * y + 3]);
            } else {
#pragma unroll
                for (int y = 0; y < 32; ++y) x[y] *= inv;
                store_row32(p, o_at + d, x);
            }
        }
    }
    if (slot >= 0 && there && (!u.alt || w == 0)) p.part_ml[kMany][rec] = make_float2(m, l);
    tc_fence_before();
    return !u.alt || both_here(bars, nm_sync);  // both have read both
}

template <int D, int TERMS, bool FOLD>
__global__ void __launch_bounds__(kThreads, 1) chunk_tile_kernel(const __grid_constant__ ChunkParams p) {
    using S = TileSmem<D>;
    extern __shared__ uint8_t tile_smem[];
    uint8_t* smem = tile_smem + ((1024u - (smem_u32(tile_smem) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMetaStages; ++s) {
            mbar_init(&bars[kMetaFull + s], 1);
            mbar_init(&bars[kMetaEmpty + s], kConvWarps + 8);  // converter and softmax warps
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bars[kKFull + s], kConvWarps);
            mbar_init(&bars[kKEmpty + s], 1);
            mbar_init(&bars[kVFull + s], kConvWarps);
            mbar_init(&bars[kVEmpty + s], 1);
            mbar_init(&bars[kSFull + s], 1);
            mbar_init(&bars[kPFull + s], 4);
            mbar_init(&bars[kOFull + s], 1);
        }
        mbar_init(&bars[kQFull], kConvWarps);
        mbar_init(&bars[kQEmpty], 1);
        mbar_init(&bars[kMerge], 8);
        mbar_init(&bars[kDone], 8);
        mbar_init(&bars[kDrain], 1);
        for (int s = 0; s < kUnitStages; ++s) {
            mbar_init(&bars[kUnitFull + s], 1);
            mbar_init(&bars[kUnitEmpty + s], 8 + kConvWarps + 1);  // softmax, converters, MMA issuer
        }
        fence_mbar_init();
    }
    if (warp == 16) tmem_alloc(reinterpret_cast<uint32_t*>(smem + S::kTmem), 512);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + S::kTmem);
    class_begins(p);
    const int units = p.head->units[kMany];
    if (warp < 8) {
        regs_more<kSoftmaxRegs>();
        int j = 0, nu = 0, ns = 0, no = 0, nm = 0;
        for (int n = 0, unit = next_unit<D>(smem, bars, n); unit >= 0; unit = next_unit<D>(smem, bars, n)) {
            const TileUnit u = tile_unit<TERMS>(p, unit);
            if (!tile_softmax<D, TERMS, FOLD>(p, u, smem, tmem, bars, j, nu, ns, no, nm)) break;
            j += u.nt;
            nu += u.nt > 0;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kDone]);
    } else if (warp < 8 + kConvWarps) {
        regs_less<kConvRegs>();
        int j = 0, nu = 0;
        for (int n = 0, unit = next_unit<D>(smem, bars, n); unit >= 0; unit = next_unit<D>(smem, bars, n)) {
            const TileUnit u = tile_unit<TERMS>(p, unit);
            if (u.nt == 0) continue;
            if (!tile_convert<D, TERMS, FOLD>(p, u, smem, bars, j, nu)) break;
            j += u.nt;
            ++nu;
        }
    } else {
        regs_less<kOtherRegs>();
        if (warp == 16) {
            const int nq = p.flags & (KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16) ? 1 : 2;
            int j = 0, nu = 0, np[2] = {0, 0};
            for (int n = 0, unit = next_unit<D>(smem, bars, n); unit >= 0; unit = next_unit<D>(smem, bars, n)) {
                const TileUnit u = tile_unit<TERMS>(p, unit);
                if (u.nt == 0) continue;
                if (!tile_mma<D, TERMS>(u, smem, tmem, bars, j, nu, np, nq)) break;
                j += u.nt;
                ++nu;
            }
            mma_commit_warp(&bars[kDrain]);  // arrives once every MMA issued above has completed
            mbar_wait(&bars[kDrain], 0);
            mbar_wait(&bars[kDone], 0);  // the softmax warps have finished with tensor memory
            __syncwarp();
            tc_fence_after();
            tmem_dealloc(tmem, 512);
        } else if (warp == 17) {
            int j = 0;
            bool ok = true;
            for (int n = 0; ok; ++n) {
                int unit = 0;
                if (lane == 0) unit = atomicAdd(&p.head->ticket, 1);
                unit = __shfl_sync(0xffffffffu, unit, 0);
                const int st = n & (kUnitStages - 1);
                ok = n < kUnitStages || mbar_wait_all(&bars[kUnitEmpty + st], ((n / kUnitStages) - 1) & 1);
                if (!ok) break;
                if (lane == 0) {
                    reinterpret_cast<int*>(smem + S::kUnits)[st] = unit < units ? unit : -1;
                    mbar_arrive(&bars[kUnitFull + st]);
                }
                if (unit >= units) break;
                const TileUnit u = tile_unit<TERMS>(p, unit);
                tile_scout(p, u, reinterpret_cast<TileMeta*>(smem + S::kMeta), bars, j, ok);
            }
        }
    }
    class_ends(p);
}

template <int D, int TERMS, bool FOLD>
cudaError_t launch_tile(const ChunkParams& p, cudaStream_t st) {
    auto kern = chunk_tile_kernel<D, TERMS, FOLD>;
    static PerDeviceOnce once;
    cudaError_t e = once.run([kern] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TileSmem<D>::kBytes);
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(device_sm_count(), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = TileSmem<D>::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

cudaError_t take_chunk_tile_status(int32_t* status) {
    int32_t v = 0;
    const int32_t zero = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
    if (e != cudaSuccess) return e;
    *status |= v;
    return v ? cudaMemcpyToSymbol(g_status, &zero, sizeof(zero)) : cudaSuccess;
}

cudaError_t launch_chunk_tile(const ChunkParams& p, cudaStream_t st, int* launches) {
    const bool two = p.unit_rows[kMany] == 128, fold = !two && (p.flags & KVD_FLAG_OUT_BF16) != 0;
    const cudaError_t e = p.D == 128 ? (two ? launch_tile<128, 2, false>(p, st) : fold ? launch_tile<128, 1, true>(p, st) : launch_tile<128, 1, false>(p, st))
                                     : (two ? launch_tile<64, 2, false>(p, st) : fold ? launch_tile<64, 1, true>(p, st) : launch_tile<64, 1, false>(p, st));
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace kvd
