// kvd_chunk_few.cu -- attention of packed new tokens over a paged cache for
// requests with few rows a KV head (single tokens, drafted tokens, short
// chunks): bound by the cache's bytes.
//
// A unit is (request, 8 or 16 rows of a KV head, stretch of tokens); its rows
// are the request's tokens times the group's heads, so a token's codes are read
// once for all of them. Each of the CTA's warps walks every fourth step of 32
// tokens with its own running maximum, sum and output: with s_j = (q . K_j)
// ks_j scale in base 2, p_j = 2^(s_j - m),
//   l = sum p_j,  o = sum (p_j vs_j) V_j,
// and the four are merged at the end. Codes come through a ring in shared memory
// that only this warp uses (16-byte cp.async, a step or two ahead), are widened
// to fp16 exactly and multiplied with mma.m16n8k16, tokens and then dims as its
// 16 rows and the queries' rows as its 8 columns: S^T = K q^T, O^T = V^T P^T (the
// smallest tile of tcgen05 has 64). The order of dims within a product is
// whatever makes a lane's operands neighbours in memory, and movmatrix turns the
// weights into the second product's operand. Requests of up to 8 rows have
// a kernel of their own, which holds half the output in registers, so more warps
// fit beside each other.
//
// Bound: HBM where rows fill a unit, and behind it the widening of codes (64
// single tokens of up to 8,192, 8 heads a KV head, 128 dims: DRAM 52 %, ALU 61 %;
// 256 of them 664 us, 502 at the copy rate); short units by their chain of loads
// (8 requests of 23 drafted tokens in all: 44 us with the plan, 8.4). 32-bit outputs:
// a product cuts the sum that it adds to off, so each makes a sum of its own (98 us
// instead of 89 for 16 single fp32 tokens of up to 8,192 when it was tried, 93 now).
#include "kvd_chunk.cuh"
#include "kvd_decode.cuh"
#include "kvd_tc.cuh"

namespace kvd {
namespace {

constexpr int kFewWarps = 4;
constexpr int kStep = kFewStep;
constexpr int kInfBits = 0x7f800000;
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Copies BYTES (4 or 16) to shared memory, or zeros when !there.
template <int BYTES>
__device__ __forceinline__ void async_copy(void* dst, const void* src, bool there) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// NR: 8-row groups of a unit. Stages of a warp's ring, and CTAs of an SM, are what 227 KB of shared memory and 64 K
// registers hold.
template <int D, int NR, int NQ>
struct FewSmem {
    static constexpr int kRows = 8 * NR;
    static constexpr int kCtas = D == 64 ? (NR == 1 ? 4 : 3) : NR == 2 && NQ == 2 ? 2 : 3;
    static constexpr int kStages = D == 128 && kCtas == 3 ? 2 : 3;  // steps
    static constexpr int kCodes = kStep * D;                     // of K or V
    static constexpr int kStage = 2 * kCodes + 2 * kStep * 4;
    static constexpr int kRing = kFewWarps * kStages * kStage;
    static constexpr int kMerge = kFewWarps * kRows * (D + 4) * 4;  // after the ring is done with
    static constexpr int kBytes = kRing > kMerge ? kRing : kMerge;
};

// The transposed 8 x 8 matrix of fp16 pairs that the warp holds.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Places of 16-byte chunk c of token row r in a stage, chosen so that the eight lanes that read together meet
// eight different places: rows 2i and 2i+1 for K, rows 0, 2, 4 and 6 for V.
template <int D>
__device__ __forceinline__ int k_at(int r, int c) { return r * D + (D == 128 ? (c ^ ((r & 1) << 2)) : c) * 16; }
template <int D>
__device__ __forceinline__ int v_at(int r, int c) { return r * D + (D == 128 ? (c ^ (r & 6)) : (c ^ ((r >> 1) & 3))) * 16; }

template <int D, int NR, int NQ, int NP>
__global__ void __launch_bounds__(kFewWarps * 32, FewSmem<D, NR, NQ>::kCtas) chunk_few_kernel(const ChunkParams p) {
    extern __shared__ __align__(16) uint8_t few_smem[];
    constexpr int KS = D / 16;      // steps of 16 dims of a product
    constexpr int CH = D / 64;      // 16-byte chunks of a K row that a lane holds
    constexpr int PER = D / 16;     // 16-byte chunks of a row
    constexpr int COPIES = kStep * PER / 32;  // chunks of K, and of V, that a lane copies
    constexpr int CLS = NR - 1;
    using S = FewSmem<D, NR, NQ>;
    constexpr int ROWS = S::kRows, STAGES = S::kStages;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, c = lane & 3;
    uint8_t* ring = few_smem + warp * STAGES * S::kStage;
    class_begins(p);
    const int units = p.head->units[CLS], span = p.head->span[CLS];
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int b = warp_find(p.first[CLS], p.B, unit);
        const ChunkRows R = chunk_rows(p, b);
        int each;
        const int rows = R.n * p.G, nrb = (rows + ROWS - 1) / ROWS, nsplit = chunk_splits(R.len, span, kStep, each);
        int rest = unit - p.first[CLS][b];
        const int rb = rest % nrb;
        rest /= nrb;
        const int hk = rest % p.Hkv, split = rest / p.Hkv;
        const int last_row = min(rows, (rb + 1) * ROWS) - 1;
        const int most = chunk_sees(p, R, static_cast<int>(p.by_g.div(static_cast<uint32_t>(last_row))));
        const int least = chunk_sees(p, R, static_cast<int>(p.by_g.div(static_cast<uint32_t>(rb * ROWS))));
        const int begin = split * each, end = min(min(begin + each, R.len), most);
        // ---- tokens into the ring. Lane l looks up token l of the step that is copied next.
        const int steps = end > begin ? (end - begin + kStep - 1) / kStep : 0;
        const int mine = steps > warp ? (steps - warp + kFewWarps - 1) / kFewWarps : 0;
        const int32_t* table = p.table + b * p.bt_stride;
        const int8_t* K = p.K + hk * p.kv_sh;
        const int8_t* V = p.V + hk * p.kv_sh;
        const float* ks = p.ks + hk * p.sc_sh;
        const float* vs = p.vs + hk * p.sc_sh;
        auto look_up = [&](int k, int& off) {  // block of this lane's token of its k-th step, -1: none
            const int t = begin + (warp + k * kFewWarps) * kStep + lane;
            if (k >= mine || t >= end) return -1;
            const int j = static_cast<int>(p.by_bs.div(static_cast<uint32_t>(t)));
            off = t - j * p.bs;
            const int id = table[j];
            if (id >= 0 && id < p.NB) return id;
            record_status(KVD_STATUS_BAD_BLOCK);
            return -1;
        };
        int next_off = 0, next_id = look_up(0, next_off);
        int ahead_off = 0, ahead_id = STAGES > 2 ? look_up(1, ahead_off) : -1;  // on its way together with the first
        auto fetch = [&](int k, bool first = false) {
            if (k < mine) {
                uint8_t* st = ring + (k % STAGES) * S::kStage;
                // where there is no token its scales are zeros, and any codes do
                const int id = max(next_id, 0), off = next_id < 0 ? 0 : next_off;
                const int64_t row = id * p.kv_sblk + off * p.kv_st, sc = id * p.sc_sblk + off;
#pragma unroll
                for (int u = 0; u < COPIES; ++u) {
                    const int i = lane + 32 * u, r = i / PER, ch = i % PER;
                    const int64_t at = __shfl_sync(0xffffffffu, row, r) + ch * 16;
                    async_copy<16>(st + k_at<D>(r, ch), K + at, true);
                    async_copy<16>(st + S::kCodes + v_at<D>(r, ch), V + at, true);
                }
                float* scales = reinterpret_cast<float*>(st + 2 * S::kCodes);
                async_copy<4>(scales + lane, ks + sc, next_id >= 0);
                async_copy<4>(scales + kStep + lane, vs + sc, next_id >= 0);
                if (first && STAGES > 2) {
                    next_id = ahead_id;
                    next_off = ahead_off;
                } else {
                    next_id = look_up(k + 1, next_off);
                }
            }
            async_commit();
        };
        // ---- queries: this lane's dims of row quad of each group, a power of two times them so that fp16 holds them
        uint32_t qb[NQ][NR][KS][2];
        float factor[NR];  // what the scores of row quad are multiplied with instead
        fetch(0, true);
        if (STAGES > 2) fetch(1);
#pragma unroll
        for (int e = 0; e < NR; ++e) {
            const int r = rb * ROWS + 8 * e + quad;
            const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(r))), g = r - i * p.G;
            const int64_t q_at = static_cast<int64_t>(R.t0 + i) * p.q_st + static_cast<int64_t>(hk * p.G + g) * p.q_sh;
            float x[CH * 16];
#pragma unroll
            for (int d = 0; d < CH * 16; ++d) x[d] = 0.f;
            if (r < rows) {
                if (p.vec_q) {
#pragma unroll
                    for (int h = 0; h < CH; ++h) {
                        const int64_t at = q_at + h * 64 + c * 16;
                        if constexpr (NQ == 2) {
                            const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.Q) + at);
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                const float4 v = src[y];
                                x[h * 16 + 4 * y] = v.x; x[h * 16 + 4 * y + 1] = v.y;
                                x[h * 16 + 4 * y + 2] = v.z; x[h * 16 + 4 * y + 3] = v.w;
                            }
                        } else {
                            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.Q) + at);
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const uint4 v = src[y];
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int z = 0; z < 4; ++z) {
                                    float2 f;
                                    if (p.flags & KVD_FLAG_Q_BF16)
                                        f = make_float2(__uint_as_float(w[z] << 16), __uint_as_float(w[z] & 0xffff0000u));
                                    else
                                        f = __half22float2(*reinterpret_cast<const __half2*>(&w[z]));
                                    x[h * 16 + 8 * y + 2 * z] = f.x;
                                    x[h * 16 + 8 * y + 2 * z + 1] = f.y;
                                }
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < CH; ++h)
#pragma unroll
                        for (int d = 0; d < 16; ++d) x[h * 16 + d] = load_q(p.Q, q_at + h * 64 + c * 16 + d, p.flags);
                }
            }
            float top = 0.f;
#pragma unroll
            for (int d = 0; d < CH * 16; ++d) top = fmaxf(top, fabsf(x[d]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // Two terms: whole numbers up to 2^11 and what is left. The first one's products with the codes add up without
            // loss below 2^24: always at 64 dims, at 128 unless nearly all of a row's have one sign. (Below 2^10, where
            // they always would, costs more than it saves: errors of 1.0e-6 against 7.3e-7 for scores of hundreds, 2.8e-7
            // against 3.3e-7 where all have one sign.)
            // One: below 2^15, products of 128 dims stay far from fp32's end.
            const int k = fit_exponent(top, NQ == 2 ? 11 : 15);
            const float f = pow2i(k);
            factor[e] = p.qscale * pow2i(-k);
#pragma unroll
            for (int s = 0; s < KS; ++s) {  // a word of four codes is a step: even dims in one pair, odd ones in the other
                const float* y = x + s * 4;
                const float a = y[0] * f, b = y[1] * f, c2 = y[2] * f, d = y[3] * f;
                if constexpr (NQ == 2) {
                    qb[0][e][s][0] = pack_half(rintf(a), rintf(c2));
                    qb[0][e][s][1] = pack_half(rintf(b), rintf(d));
                    qb[1][e][s][0] = pack_rest(a, c2, qb[0][e][s][0]);
                    qb[1][e][s][1] = pack_rest(b, d, qb[0][e][s][1]);
                } else {
                    qb[0][e][s][0] = pack_half(a, c2);
                    qb[0][e][s][1] = pack_half(b, d);
                }
            }
        }
        // the columns of this lane in the products: rows 2c and 2c + 1 of each group
        float rf[NR][2], m[NR][2], l[NR][2];
        int sees[NR][2];
        // Exponents of the four rows, a byte each, plus 127: value scales that a row has seen, times 2^ve, are below 2^7,
        // so that weights up to 2^8 fit fp16. (Registers are short here: 16 requests of 16 rows take 89 us, 93 with a word
        // for each and 96 with one exponent for all and a copy of the loop below for rows that differ; 86 with one alone.)
        uint32_t ve4 = 253u * 0x01010101u;
        auto scale_of = [&](int e, int y) { return __uint_as_float(__byte_perm(ve4, 0u, (2 * e + y) << 12 | 0x0444) >> 1); };
#pragma unroll
        for (int e = 0; e < NR; ++e)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                rf[e][y] = __shfl_sync(0xffffffffu, factor[e], 4 * (2 * c + y));
                const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(rb * ROWS + 8 * e + 2 * c + y)));
                // rows that are not there see what the last one does
                sees[e][y] = min(end, chunk_sees(p, R, min(i, R.n - 1)));
                m[e][y] = -INFINITY;
                l[e][y] = 0.f;
            }
        // ---- the walk
        float o[NR][D / 16][4];
#pragma unroll
        for (int e = 0; e < NR; ++e)
#pragma unroll
            for (int j = 0; j < D / 16; ++j) o[e][j][0] = o[e][j][1] = o[e][j][2] = o[e][j][3] = 0.f;
#pragma unroll 1
        for (int k = 0; k < mine; ++k) {
            async_wait<STAGES - 2>();
            __syncwarp();  // every lane's copies of step k are there, and step k - 1 has been read
            fetch(k + STAGES - 1);
            const uint8_t* st = ring + (k % STAGES) * S::kStage;
            const float* scales = reinterpret_cast<const float*>(st + 2 * S::kCodes);
            const int t0 = begin + (warp + k * kFewWarps) * kStep;
            // scores: s[mt][e][x] is token 16 mt + quad + 8 (x >> 1), row 2c + (x & 1) of group e
            float s[2][NR][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                for (int e = 0; e < NR; ++e) s[mt][e][0] = s[mt][e][1] = s[mt][e][2] = s[mt][e][3] = 0.f;
                // the second term's sum by itself: a sum is cut off, not rounded, behind every step, by a unit of its size
                float s2[NR][4] = {};
#pragma unroll
                for (int h = 0; h < CH; ++h) {
                    const uint4 a4 = *reinterpret_cast<const uint4*>(st + k_at<D>(mt * 16 + quad, h * 4 + c));
                    const uint4 b4 = *reinterpret_cast<const uint4*>(st + k_at<D>(mt * 16 + quad + 8, h * 4 + c));
                    const uint32_t wa[4] = {a4.x, a4.y, a4.z, a4.w}, wb[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t a[4] = {half_pair(wa[x]), half_pair(wb[x]), half_pair(wa[x] >> 8), half_pair(wb[x] >> 8)};
#pragma unroll
                        for (int e = 0; e < NR; ++e) {
                            mma_16816(s[mt][e], a, qb[0][e][h * 4 + x][0], qb[0][e][h * 4 + x][1]);
                            if constexpr (NQ == 2) mma_16816(s2[e], a, qb[1][e][h * 4 + x][0], qb[1][e][h * 4 + x][1]);
                        }
                    }
                }
                if constexpr (NQ == 2)
#pragma unroll
                    for (int e = 0; e < NR; ++e)
#pragma unroll
                        for (int x = 0; x < 4; ++x) s[mt][e][x] += s2[e][x];
            }
            float top[NR][2];
#pragma unroll
            for (int e = 0; e < NR; ++e) top[e][0] = top[e][1] = -INFINITY;
            const bool masked = t0 + kStep > min(least, end);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int t = 16 * mt + quad + 8 * half;
                    const float kq = scales[t];
#pragma unroll
                    for (int e = 0; e < NR; ++e)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            float v = s[mt][e][2 * half + y] * kq * rf[e][y];
                            if (masked && t0 + t >= sees[e][y]) v = -INFINITY;  // the row does not see the token
                            s[mt][e][2 * half + y] = v;
                            top[e][y] = fmaxf(top[e][y], v);
                        }
                }
            // largest value scale of the step, and the exponents that it asks for: a row's are its own where rows see
            // different tokens, so that no hidden one costs it bits. A scale that is not finite has no say, but makes
            // the sum of weights of the rows that see it NaN.
            float v_top = fabsf(scales[kStep + lane]);
            uint32_t fit4 = 0u;
            if (!masked) {
                int bits = __reduce_max_sync(0xffffffffu, __float_as_int(v_top));
                if (bits >= kInfBits) {
#pragma unroll
                    for (int e = 0; e < NR; ++e) l[e][0] = l[e][1] = NAN;
                    bits = __reduce_max_sync(0xffffffffu, v_top < INFINITY ? __float_as_int(v_top) : 0);
                }
                fit4 = (bits == 0 ? 253u : fit_exponent(__int_as_float(bits), 7) + 127u) * 0x01010101u;
            } else {
                const unsigned odd = __ballot_sync(0xffffffffu, !(v_top < INFINITY));
                if (!(v_top < INFINITY)) v_top = 0.f;
#pragma unroll
                for (int x = 1; x < 32; x <<= 1) {  // lane i: the largest of tokens 0 .. i
                    const float y = __shfl_up_sync(0xffffffffu, v_top, x);
                    if (lane >= x) v_top = fmaxf(v_top, y);
                }
#pragma unroll
                for (int e = 0; e < NR; ++e)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int lim = sees[e][y] - t0;
                        const float seen = __shfl_sync(0xffffffffu, v_top, min(max(lim, 1), 32) - 1);
                        fit4 |= (lim <= 0 || seen == 0.f ? 253u : fit_exponent(seen, 7) + 127u) << (8 * (2 * e + y));
                        if (odd & (lim >= 32 ? 0xffffffffu : lim <= 0 ? 0u : (1u << lim) - 1u)) l[e][y] = NAN;
                    }
            }
            fit4 = __vminu4(fit4, ve4);
            bool move = fit4 != ve4;
#pragma unroll
            for (int e = 0; e < NR; ++e)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    move |= top[e][y] > m[e][y] + (m[e][y] == -INFINITY ? 0.f : 8.f);
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int e = 0; e < NR; ++e)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        float to = top[e][y];
                        to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 4));
                        to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 8));
                        to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 16));
                        const bool go = to > m[e][y] + (m[e][y] == -INFINITY ? 0.f : 8.f);
                        const float f = go ? (m[e][y] == -INFINITY ? 0.f : ex2_fast(m[e][y] - to)) : 1.f;
                        const int at = 8 * (2 * e + y), fall = static_cast<int>(ve4 >> at & 0xffu) - static_cast<int>(fit4 >> at & 0xffu);
                        const float fo = fall > 126 ? 0.f : f * pow2i(-fall);
                        if (go) m[e][y] = to;
                        l[e][y] *= f;
#pragma unroll
                        for (int j = 0; j < D / 16; ++j) {
                            o[e][j][y] *= fo;
                            o[e][j][2 + y] *= fo;
                        }
                    }
                ve4 = fit4;
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                // weights of 16 tokens
                uint32_t pb[NP][NR][2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float vq = scales[kStep + 16 * mt + quad + 8 * half];
#pragma unroll
                    for (int e = 0; e < NR; ++e) {
                        float w[2];
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const float x = s[mt][e][2 * half + y];
                            const float pr = ex2_fast(x - (m[e][y] == -INFINITY ? 0.f : m[e][y]));
                            l[e][y] += pr;
                            w[y] = pr * (vq * scale_of(e, y));
                            if (masked && x == -INFINITY) w[y] = 0.f;  // a hidden token's scale may be anything
                        }
                        const uint32_t hi = pack_half(w[0], w[1]);
                        pb[0][e][half] = transposed(hi);
                        if constexpr (NP == 2) pb[1][e][half] = transposed(pack_rest(w[0], w[1], hi));
                    }
                }
                // values: tokens 2c, 2c+1, 2c+8, 2c+9 of the 16; dims quad * D/8 .. of each
                constexpr int W = D / 32;  // words of a lane's dims
                uint32_t v[4][W];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = mt * 16 + 2 * c + (x & 1) + (x >> 1) * 8;
                    const uint8_t* src = st + S::kCodes;
                    if constexpr (D == 128) {
                        const uint4 w = *reinterpret_cast<const uint4*>(src + v_at<D>(r, quad));
                        v[x][0] = w.x; v[x][1] = w.y; v[x][2] = w.z; v[x][3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(src + v_at<D>(r, quad >> 1) + (quad & 1) * 8);
                        v[x][0] = w.x; v[x][1] = w.y;
                    }
                }
#pragma unroll
                for (int y = 0; y < W; ++y)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {  // dims 4y + 2z and the next one: rows quad and quad + 8 of a product
                        const uint32_t lo = __byte_perm(v[0][y], v[1][y], z ? 0x7632 : 0x5410);
                        const uint32_t hi = __byte_perm(v[2][y], v[3][y], z ? 0x7632 : 0x5410);
                        const uint32_t a[4] = {half_pair(lo), half_pair(lo >> 8), half_pair(hi), half_pair(hi >> 8)};
#pragma unroll
                        for (int e = 0; e < NR; ++e) {
                            if constexpr (NP == 1) {
                                mma_16816(o[e][2 * y + z], a, pb[0][e][0], pb[0][e][1]);
                            } else {  // sums by themselves: a product cuts off what it adds to, towards zero
                                float sum[4] = {};
                                mma_16816(sum, a, pb[1][e][0], pb[1][e][1]);
                                mma_16816(sum, a, pb[0][e][0], pb[0][e][1]);
#pragma unroll
                                for (int x = 0; x < 4; ++x) o[e][2 * y + z][x] += sum[x];
                            }
                        }
                    }
            }
        }
        async_wait<0>();
        // ---- merge of the warps
        __syncthreads();  // every warp is done with its ring
        float* merge = reinterpret_cast<float*>(few_smem);  // [warp][row][D + 4]: dims, then m and l
#pragma unroll
        for (int e = 0; e < NR; ++e)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float sum = l[e][y];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const float back = pow2i(127 - static_cast<int>(ve4 >> (8 * (2 * e + y)) & 0xffu));
                float* row = merge + (warp * ROWS + 8 * e + 2 * c + y) * (D + 4);
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    *reinterpret_cast<float2*>(row + quad * (D / 8) + 2 * j) = make_float2(o[e][j][y] * back, o[e][j][2 + y] * back);
                if (quad == 0) *reinterpret_cast<float2*>(row + D) = make_float2(m[e][y], sum);
            }
        __syncthreads();
        const int slot = nsplit > 1 ? p.rec[CLS][b] + (hk * nrb + rb) * nsplit + split : -1;
        constexpr int TPR = kFewWarps * 32 / ROWS;  // threads a row, four dims at a time each
        const int r = threadIdx.x / TPR, tx = threadIdx.x % TPR, row = rb * ROWS + r;
        if (row < rows) {
            float M = -INFINITY, f[kFewWarps], L = 0.f;
            float2 ml[kFewWarps];
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                ml[w] = *reinterpret_cast<const float2*>(merge + (w * ROWS + r) * (D + 4) + D);
                M = fmaxf(M, ml[w].x);
            }
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                f[w] = ml[w].x == -INFINITY ? 0.f : ex2_fast(ml[w].x - M);
                L += ml[w].y * f[w];
            }
            const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(row))), g = row - i * p.G;
            const int64_t o_at = static_cast<int64_t>(R.t0 + i) * p.o_st + static_cast<int64_t>(hk * p.G + g) * p.o_sh;
            // a sum of weights that is 0 belongs to a row that sees nothing; NaN stays
            const float inv = slot >= 0 ? 1.f : L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int j = 0; j < D / 4 / TPR; ++j) {
                const int d = (tx + j * TPR) * 4;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(merge + (w * ROWS + r) * (D + 4) + d);
                    if (f[w] != 0.f) x = make_float4(fmaf(y.x, f[w], x.x), fmaf(y.y, f[w], x.y), fmaf(y.z, f[w], x.z), fmaf(y.w, f[w], x.w));
                }
                x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                if (slot >= 0) *reinterpret_cast<float4*>(p.part_o[CLS] + (static_cast<int64_t>(slot) * ROWS + r) * D + d) = x;
                else store_out4(p, o_at + d, x);
            }
            if (slot >= 0 && tx == 0) p.part_ml[CLS][static_cast<int64_t>(slot) * ROWS + r] = make_float2(M, L);
        }
        __syncthreads();  // the ring may be filled again
        if (slot >= 0) {  // the CTA that is last to write a record of the unit merges them
            __shared__ int s_last;
            if (threadIdx.x == 0) {  // releases this CTA's records, acquires the others'
                int before;
                asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(&p.arrived[CLS][slot - split]) : "memory");
                s_last = before == nsplit - 1;
            }
            __syncthreads();
            if (s_last)
                merge_records<D, ROWS / kFewWarps>(p, R, p.part_o[CLS], p.part_ml[CLS], slot - split, nsplit, ROWS, hk, rb * ROWS,
                                                   warp * (ROWS / kFewWarps), rows, lane);
        }
    }
    class_ends(p);
}

template <int D, int NR, int NQ, int NP>
cudaError_t launch_few(const ChunkParams& p, cudaStream_t st) {
    auto kern = chunk_few_kernel<D, NR, NQ, NP>;
    using S = FewSmem<D, NR, NQ>;
    static PerDeviceOnce once;
    cudaError_t e = once.run([kern] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.ctas[NR - 1]), 1, 1);
    cfg.blockDim = dim3(kFewWarps * 32, 1, 1);
    cfg.dynamicSmemBytes = S::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int D, int NR>
cudaError_t launch_few_of(const ChunkParams& p, cudaStream_t st) {
    const bool q16 = (p.flags & (KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16)) != 0, o16 = (p.flags & (KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16)) != 0;
    return q16 ? (o16 ? launch_few<D, NR, 1, 1>(p, st) : launch_few<D, NR, 1, 2>(p, st))
               : (o16 ? launch_few<D, NR, 2, 1>(p, st) : launch_few<D, NR, 2, 2>(p, st));
}

}  // namespace

int chunk_few_ctas(int D, int cls, bool q16) {
    if (D == 64) return cls ? FewSmem<64, 2, 1>::kCtas : FewSmem<64, 1, 1>::kCtas;
    return cls == 0 ? FewSmem<128, 1, 1>::kCtas : q16 ? FewSmem<128, 2, 1>::kCtas : FewSmem<128, 2, 2>::kCtas;
}

cudaError_t launch_chunk_few(const ChunkParams& p, int cls, cudaStream_t st, int* launches) {
    const cudaError_t e = p.D == 128 ? (cls ? launch_few_of<128, 2>(p, st) : launch_few_of<128, 1>(p, st))
                                     : (cls ? launch_few_of<64, 2>(p, st) : launch_few_of<64, 1>(p, st));
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace kvd
