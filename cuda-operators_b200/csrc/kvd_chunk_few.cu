// kvd_chunk_few.cu -- attention of packed new tokens over a paged cache for
// requests with few rows a KV head (single tokens, drafted tokens, short
// chunks): bound by the cache's bytes.
//
// A unit is (request, 16 rows of a KV head, stretch of tokens); its rows are
// the request's tokens times the group's heads, so a token's codes are read once
// for up to 16 of them. Each of the CTA's warps walks every fourth step of 32
// tokens with its own running maximum, sum and output: with s_j = (q . K_j)
// ks_j scale in base 2, p_j = 2^(s_j - m),
//   l = sum p_j,  o = sum (p_j vs_j) V_j,
// and the four are merged at the end. Codes come through a ring in shared memory
// that only this warp uses (16-byte cp.async, three steps ahead), are widened to
// fp16 exactly and multiplied with mma.m16n8k16: 16 rows are all that a unit has,
// where tcgen05's smallest tile is 64. The order of dims in q . K, and of
// dims over the output's columns, is whatever makes a lane's operands neighbours
// in memory; the scores' accumulators are the weights' operand as they lie.
#include "kvd_chunk.cuh"
#include "kvd_decode.cuh"
#include "kvd_tc.cuh"

namespace kvd {
namespace {

constexpr int kFewWarps = 4;
constexpr int kStep = kFewStep;
constexpr int kStages = 3;  // steps of a warp's ring

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

template <int D>
struct FewSmem {
    static constexpr int kCodes = kStep * D;                // one of K or V
    static constexpr int kStage = 2 * kCodes + 2 * kStep * 4;
    static constexpr int kRing = kFewWarps * kStages * kStage;
    static constexpr int kMerge = kFewWarps * kFewRows * (D + 4) * 4;  // after the ring is done with
    static constexpr int kBytes = kRing > kMerge ? kRing : kMerge;
};

// Places of 16-byte chunk c of token row r in a stage, chosen so that the eight lanes that read together meet
// eight different places: rows 2i and 2i+1 for K, rows 0, 2, 4 and 6 for V.
template <int D>
__device__ __forceinline__ int k_at(int r, int c) { return r * D + (D == 128 ? (c ^ ((r & 1) << 2)) : c) * 16; }
template <int D>
__device__ __forceinline__ int v_at(int r, int c) { return r * D + (D == 128 ? (c ^ (r & 6)) : (c ^ ((r >> 1) & 3))) * 16; }

template <int D, int NQ, int NP>
__global__ void __launch_bounds__(kFewWarps * 32, 2) chunk_few_kernel(const ChunkParams p) {
    extern __shared__ __align__(16) uint8_t few_smem[];
    constexpr int KS = D / 16;      // steps of 16 dims of a product
    constexpr int CH = D / 64;      // 16-byte chunks of a K row that a lane holds
    constexpr int PER = D / 16;     // 16-byte chunks of a row
    constexpr int COPIES = kStep * PER / 32;  // chunks of K, and of V, that a lane copies
    using S = FewSmem<D>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, c = lane & 3;
    uint8_t* ring = few_smem + warp * kStages * S::kStage;
    grid_dependency_wait();
    allow_dependents();
    const int units = p.head->few_units, span = p.head->few_span;
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int b = warp_find(p.few_first, p.B, unit);
        const ChunkRows R = chunk_rows(p, b);
        int each;
        const int rows = R.n * p.G, nrb = (rows + kFewRows - 1) / kFewRows, nsplit = chunk_splits(R.len, span, kStep, each);
        int rest = unit - p.few_first[b];
        const int rb = rest % nrb;
        rest /= nrb;
        const int hk = rest % p.Hkv, split = rest / p.Hkv;
        // the two rows of this lane: token of the request, head of the group, tokens that it sees
        int sees[2];
        int64_t q_at[2];
        bool there[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = rb * kFewRows + quad + 8 * e;
            const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(r))), g = r - i * p.G;
            there[e] = r < rows;
            sees[e] = chunk_sees(p, R, min(i, R.n - 1));  // rows that are not there see what the last one does
            q_at[e] = static_cast<int64_t>(R.t0 + i) * p.q_st + static_cast<int64_t>(hk * p.G + g) * p.q_sh;
        }
        const int last_row = min(rows, (rb + 1) * kFewRows) - 1;
        const int most = chunk_sees(p, R, static_cast<int>(p.by_g.div(static_cast<uint32_t>(last_row))));
        const int least = chunk_sees(p, R, static_cast<int>(p.by_g.div(static_cast<uint32_t>(rb * kFewRows))));
        const int begin = split * each, end = min(min(begin + each, R.len), most);
        // ---- tokens into the ring. Lane l looks up token l of the step that is copied next.
        const int steps = end > begin ? (end - begin + kStep - 1) / kStep : 0;
        const int mine = steps > warp ? (steps - warp + kFewWarps - 1) / kFewWarps : 0;
        const int32_t* table = p.table + b * p.bt_stride;
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
        auto fetch = [&](int k) {
            if (k < mine) {
                uint8_t* st = ring + (k % kStages) * S::kStage;
                const int64_t row = next_id < 0 ? -1 : next_id * p.kv_sblk + hk * p.kv_sh + next_off * p.kv_st;
                const int64_t sc = next_id < 0 ? 0 : next_id * p.sc_sblk + hk * p.sc_sh + next_off;
#pragma unroll
                for (int u = 0; u < COPIES; ++u) {
                    const int i = lane + 32 * u, r = i / PER, ch = i % PER;
                    const int64_t at = __shfl_sync(0xffffffffu, row, r);
                    const bool ok = at >= 0;
                    const int64_t from = (ok ? at : 0) + ch * 16;
                    async_copy<16>(st + k_at<D>(r, ch), p.K + from, ok);
                    async_copy<16>(st + S::kCodes + v_at<D>(r, ch), p.V + from, ok);
                }
                float* scales = reinterpret_cast<float*>(st + 2 * S::kCodes);
                async_copy<4>(scales + lane, p.ks + sc, next_id >= 0);
                async_copy<4>(scales + kStep + lane, p.vs + sc, next_id >= 0);
                next_id = look_up(k + 1, next_off);
            }
            async_commit();
        };
#pragma unroll 1
        for (int k = 0; k < kStages - 1; ++k) fetch(k);
        // ---- queries: this lane's dims of its rows, a power of two times them so that fp16 holds them
        uint32_t qa[NQ][KS][4];
        float rf[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x[CH * 16];
#pragma unroll
            for (int h = 0; h < CH; ++h)
#pragma unroll
                for (int d = 0; d < 16; ++d) x[h * 16 + d] = 0.f;
            if (there[e]) {
                if (p.vec_q) {
#pragma unroll
                    for (int h = 0; h < CH; ++h) {
                        const int64_t at = q_at[e] + h * 64 + c * 16;
                        if constexpr (NQ == 2) {
                            const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.Q) + at);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float4 v = src[i];
                                x[h * 16 + 4 * i] = v.x; x[h * 16 + 4 * i + 1] = v.y;
                                x[h * 16 + 4 * i + 2] = v.z; x[h * 16 + 4 * i + 3] = v.w;
                            }
                        } else {
                            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.Q) + at);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint4 v = src[i];
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int y = 0; y < 4; ++y) {
                                    float2 f;
                                    if (p.flags & KVD_FLAG_Q_BF16)
                                        f = make_float2(__uint_as_float(w[y] << 16), __uint_as_float(w[y] & 0xffff0000u));
                                    else
                                        f = __half22float2(*reinterpret_cast<const __half2*>(&w[y]));
                                    x[h * 16 + 8 * i + 2 * y] = f.x;
                                    x[h * 16 + 8 * i + 2 * y + 1] = f.y;
                                }
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < CH; ++h)
#pragma unroll
                        for (int d = 0; d < 16; ++d) x[h * 16 + d] = load_q(p.Q, q_at[e] + h * 64 + c * 16 + d, p.flags);
                }
            }
            float top = 0.f;
#pragma unroll
            for (int d = 0; d < CH * 16; ++d) top = fmaxf(top, fabsf(x[d]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int k = fit_exponent(top, 15);  // below 2^15: products of 128 dims stay far from fp32's end
            const float f = pow2i(k);
            rf[e] = p.qscale * pow2i(-k);
#pragma unroll
            for (int s = 0; s < KS; ++s) {  // a word of four codes is a step: even dims in one pair, odd ones in the other
                const float* y = x + s * 4;
                const uint32_t ev = pack_half(y[0] * f, y[2] * f), od = pack_half(y[1] * f, y[3] * f);
                qa[0][s][e] = ev;
                qa[0][s][2 + e] = od;
                if constexpr (NQ == 2) {
                    qa[1][s][e] = pack_rest(y[0] * f, y[2] * f, ev);
                    qa[1][s][2 + e] = pack_rest(y[1] * f, y[3] * f, od);
                }
            }
        }
        // ---- the walk
        float o[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        int ve = 126;  // value scales times 2^ve are below 2^7, so that weights up to 2^8 fit fp16
#pragma unroll 1
        for (int k = 0; k < mine; ++k) {
            async_wait<kStages - 2>();
            __syncwarp();  // every lane's copies of step k are there, and step k - 1 has been read
            fetch(k + kStages - 1);
            const uint8_t* st = ring + (k % kStages) * S::kStage;
            const float* scales = reinterpret_cast<const float*>(st + 2 * S::kCodes);
            const int t0 = begin + (warp + k * kFewWarps) * kStep;
            float s[kStep / 8][4];
#pragma unroll
            for (int n = 0; n < kStep / 8; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int h = 0; h < CH; ++h) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(st + k_at<D>(n * 8 + quad, h * 4 + c));
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t b0 = half_pair(w[x]), b1 = half_pair(w[x] >> 8);
                        mma_16816(s[n], qa[0][h * 4 + x], b0, b1);
                        if constexpr (NQ == 2) mma_16816(s[n], qa[1][h * 4 + x], b0, b1);
                    }
                }
            }
            // scores; -inf where a row does not see the token
            float top[2] = {-INFINITY, -INFINITY};
            const bool masked = t0 + kStep > min(least, end);
#pragma unroll
            for (int n = 0; n < kStep / 8; ++n) {
                const float2 kq = *reinterpret_cast<const float2*>(scales + n * 8 + 2 * c);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float v = s[n][x] * ((x & 1) ? kq.y : kq.x) * rf[x >> 1];
                    if (masked && t0 + n * 8 + 2 * c + (x & 1) >= min(sees[x >> 1], end)) v = -INFINITY;
                    s[n][x] = v;
                    top[x >> 1] = fmaxf(top[x >> 1], v);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
            }
            // largest value scale of the step (what is not finite has no say)
            float v_top = fabsf(scales[kStep + lane]);
            if (!(v_top < INFINITY)) v_top = 0.f;
            const int v_bits = __reduce_max_sync(0xffffffffu, __float_as_int(v_top));
            const int v_fit = v_bits == 0 ? 126 : fit_exponent(__int_as_float(v_bits), 7);
            const bool grow = v_fit < ve;
            bool move[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) move[e] = top[e] > m[e] + (m[e] == -INFINITY ? 0.f : 8.f);
            if (__any_sync(0xffffffffu, grow || move[0] || move[1])) {
                const float fv = grow ? (ve - v_fit > 126 ? 0.f : pow2i(v_fit - ve)) : 1.f;
                if (grow) ve = v_fit;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float f = move[e] ? (m[e] == -INFINITY ? 0.f : ex2_fast(m[e] - top[e])) : 1.f;
                    if (move[e]) m[e] = top[e];
                    l[e] *= f;
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        o[j][2 * e] *= f * fv;
                        o[j][2 * e + 1] *= f * fv;
                    }
                }
            }
            const float vf = pow2i(ve);
            // weights, and the sums of values
#pragma unroll
            for (int g = 0; g < kStep / 16; ++g) {
                uint32_t pa[NP][4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int n = 2 * g + half;
                    const float2 vq = *reinterpret_cast<const float2*>(scales + kStep + n * 8 + 2 * c);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float me = m[e] == -INFINITY ? 0.f : m[e];
                        const float p0 = ex2_fast(s[n][2 * e] - me), p1 = ex2_fast(s[n][2 * e + 1] - me);
                        l[e] += p0 + p1;
                        float w0 = p0 * (vq.x * vf), w1 = p1 * (vq.y * vf);
                        if (masked) {  // a hidden token's scale may be anything
                            if (s[n][2 * e] == -INFINITY) w0 = 0.f;
                            if (s[n][2 * e + 1] == -INFINITY) w1 = 0.f;
                        }
                        pa[0][2 * half + e] = pack_half(w0, w1);
                        if constexpr (NP == 2) pa[1][2 * half + e] = pack_rest(w0, w1, pa[0][2 * half + e]);
                    }
                }
                // tokens 2c, 2c+1, 2c+8, 2c+9 of these 16; dims quad * D/8 .. of each
                constexpr int W = D / 32;  // words of a lane's dims
                uint32_t v[4][W];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = g * 16 + 2 * c + (x & 1) + (x >> 1) * 8;
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
                for (int y = 0; y < W; ++y) {
                    const uint32_t lo01 = __byte_perm(v[0][y], v[1][y], 0x5410), lo23 = __byte_perm(v[0][y], v[1][y], 0x7632);
                    const uint32_t hi01 = __byte_perm(v[2][y], v[3][y], 0x5410), hi23 = __byte_perm(v[2][y], v[3][y], 0x7632);
                    const uint32_t b0[4] = {half_pair(lo01), half_pair(lo01 >> 8), half_pair(lo23), half_pair(lo23 >> 8)};
                    const uint32_t b1[4] = {half_pair(hi01), half_pair(hi01 >> 8), half_pair(hi23), half_pair(hi23 >> 8)};
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        mma_16816(o[4 * y + d], pa[0], b0[d], b1[d]);
                        if constexpr (NP == 2) mma_16816(o[4 * y + d], pa[1], b0[d], b1[d]);
                    }
                }
            }
        }
        async_wait<0>();
        // ---- merge of the warps. Column n of product j is dim n * D/8 + j.
        __syncthreads();  // every warp is done with its ring
        float* merge = reinterpret_cast<float*>(few_smem);  // [warp][row][D + 4]: dims, then m and l
        const float back = pow2i(-ve);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            float* row = merge + (warp * kFewRows + quad + 8 * e) * (D + 4);
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
                row[(2 * c) * (D / 8) + j] = o[j][2 * e] * back;
                row[(2 * c + 1) * (D / 8) + j] = o[j][2 * e + 1] * back;
            }
            if (c == 0) {
                row[D] = m[e];
                row[D + 1] = l[e];
            }
        }
        __syncthreads();
        const int slot = nsplit > 1 ? p.few_rec[b] + (hk * nrb + rb) * nsplit + split : -1;
        for (int r = warp; r < kFewRows; r += kFewWarps) {
            const int row = rb * kFewRows + r;
            if (row >= rows) break;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, merge[(w * kFewRows + r) * (D + 4) + D]);
            float f[kFewWarps], L = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float* src = merge + (w * kFewRows + r) * (D + 4);
                f[w] = src[D] == -INFINITY ? 0.f : ex2_fast(src[D] - M);
                L += src[D + 1] * f[w];
            }
            const int i = static_cast<int>(p.by_g.div(static_cast<uint32_t>(row))), g = row - i * p.G;
            const int64_t o_at = static_cast<int64_t>(R.t0 + i) * p.o_st + static_cast<int64_t>(hk * p.G + g) * p.o_sh;
            // a sum of weights that is 0 belongs to a row that sees nothing; NaN stays
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int d = lane; d < D; d += 32) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w)
                    if (f[w] != 0.f) x = fmaf(merge[(w * kFewRows + r) * (D + 4) + d], f[w], x);
                if (slot >= 0) p.few_o[(static_cast<int64_t>(slot) * kFewRows + r) * D + d] = x;
                else store_out(p.out, o_at + d, x * inv, p.flags);
            }
            if (slot >= 0 && lane == 0) p.few_ml[slot * kFewRows + r] = make_float2(M, L);
        }
        __syncthreads();  // the ring may be filled again
    }
}

template <int D, int NQ, int NP>
cudaError_t launch_few(const ChunkParams& p, cudaStream_t st) {
    auto kern = chunk_few_kernel<D, NQ, NP>;
    static PerDeviceOnce once;
    cudaError_t e = once.run([kern] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FewSmem<D>::kBytes);
    });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2u * device_sm_count(), 1, 1);
    cfg.blockDim = dim3(kFewWarps * 32, 1, 1);
    cfg.dynamicSmemBytes = FewSmem<D>::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

cudaError_t launch_chunk_few(const ChunkParams& p, cudaStream_t st, int* launches) {
    const bool q16 = (p.flags & (KVD_FLAG_Q_BF16 | KVD_FLAG_Q_F16)) != 0, o16 = (p.flags & (KVD_FLAG_OUT_BF16 | KVD_FLAG_OUT_F16)) != 0;
    cudaError_t e;
    if (p.D == 128)
        e = q16 ? (o16 ? launch_few<128, 1, 1>(p, st) : launch_few<128, 1, 2>(p, st))
                : (o16 ? launch_few<128, 2, 1>(p, st) : launch_few<128, 2, 2>(p, st));
    else
        e = q16 ? (o16 ? launch_few<64, 1, 1>(p, st) : launch_few<64, 1, 2>(p, st))
                : (o16 ? launch_few<64, 2, 1>(p, st) : launch_few<64, 2, 2>(p, st));
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace kvd
