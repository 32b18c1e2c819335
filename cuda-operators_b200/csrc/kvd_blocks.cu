// kvd_blocks.cu -- the paged serving step around the attention kernels: block
// tables and slot maps from request lengths, quantised writes and reads by
// slot, and the selection of blocks that a decode attends to.
//
// No reference counterpart (the reference's caches are dense and complete,
// kv_cache/new_kvint8.cu:83-84). This file must not be built with fast-math:
// the quantiser's divisions are IEEE.
#include "kvd_blocks.cuh"
#include "kvd_common.cuh"
#include "kvd_decode.cuh"
#include "kvd_quant.cuh"

namespace kvd {
namespace {

template <class... A, class... B>
cudaError_t launch_after(void (*kern)(A...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, B... args) {
    // Programmatic dependent of the kernel before it; every kernel here waits
    // (griddepcontrol.wait) before its first global access.
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

// ----------------------------------------------------------------------- plan
// Prefix sums over the requests (new tokens, blocks needed, blocks given back)
// place every slot, table entry and free-list entry independently, so after
// the sums all writes run in parallel. Every CTA makes the sums itself (8 bytes
// a request from L2, an exchange through shared memory a sum) and writes its
// share, a slot per thread where that many threads fit on the GPU. Bound:
// latency, a chain of three loads and the sums' barriers: 3.7 us for 8 requests
// and 8.7 us for 1,024 with 65,536 new tokens. Up to 256 requests a CTA has 256
// threads, above that 1,024: 8 requests took 3.3 us with 256 and 4.1 with 1,024,
// 512 take 5.5 and 4.8, 4,096 take 21 and 12. Lengths and the count may alias the
// inputs: the CTA that was last to read the inputs writes them, at its end; the
// others have counted themselves right after reading.
constexpr int kPlanMaxBatch = 8192;

struct PlanParams {
    kvd_paged_plan_desc d;
    const int32_t* seq_lens;
    const int32_t* new_lens;
    int32_t* table;
    int32_t* free_blocks;
    const int32_t* free_count;
    int64_t* slots;
    int32_t* starts;
    int32_t* lens_out;
    int32_t* count_out;
    unsigned int* ticket;
    FastDiv by_bs;
};

// Sums saturate at 2^31 - 1: lengths no pool can hold are refused, not wrapped.
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }

// Inclusive prefix sums of N values per thread over the block, on top of `carry`.
template <int N>
__device__ __forceinline__ void block_scan(uint32_t (&x)[N], const uint32_t (&carry)[N], uint32_t (*warp_sums)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x[i], o);
            if (lane >= o) x[i] = sat_add(x[i], y);
        }
    __syncthreads();  // the sums of the scan before are no longer read
    if (lane == 31)
#pragma unroll
        for (int i = 0; i < N; ++i) warp_sums[i][warp] = x[i];
    __syncthreads();
    uint32_t s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = lane < nw ? warp_sums[i][lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, s[i], o);
            if (lane >= o) s[i] = sat_add(s[i], y);
        }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t before = __shfl_sync(0xffffffffu, s[i], (warp - 1) & 31);
        x[i] = sat_add(x[i], warp > 0 ? sat_add(carry[i], before) : carry[i]);
    }
}

// First index in [0, n) whose inclusive sum is above v (n when there is none).
__device__ __forceinline__ int first_above(const uint32_t* sums, int n, uint32_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > v) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Shared memory of one request: four sums or lengths and a flag.
constexpr size_t kPlanBytes = 17;

__global__ void __launch_bounds__(1024) plan_kernel(const PlanParams p) {
    extern __shared__ uint32_t plan_smem[];
    __shared__ uint32_t warp_sums[2][32];
    __shared__ uint32_t s_popped;
    __shared__ int s_last;
    grid_dependency_wait();
    allow_dependents();
    const int B = p.d.batch, bs = p.d.block_size, MB = p.d.max_blocks_per_seq, NB = p.d.num_blocks;
    const int64_t cap = static_cast<int64_t>(MB) * bs;
    uint32_t* tok = plan_smem;   // [B] tokens up to and with request b
    uint32_t* need = tok + B;    // [B] blocks needed up to and with request b
    uint32_t* back = need + B;   // [B] blocks given back up to and with request b
    int32_t* held_len = reinterpret_cast<int32_t*>(back + B);  // [B] lengths
    uint8_t* okay = reinterpret_cast<uint8_t*>(held_len + B);  // [B] 0 refused, 1 or 2 served, 3 ends
    const uint32_t fc = static_cast<uint32_t>(min(max(0, *p.free_count), NB));
    auto blocks_of = [&](int tokens) {
        const int whole = static_cast<int>(p.by_bs.div(static_cast<uint32_t>(tokens)));
        return whole + (whole * bs != tokens);
    };
    uint32_t carry_t[1] = {0}, carry[2] = {0, 0};
    if (threadIdx.x == 0) s_popped = 0;
    int status = 0;
    for (int b0 = 0; b0 < B; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        const bool in = b < B;
        const int n = in ? p.new_lens[b] : 0;
        const int len = in ? static_cast<int>(min(static_cast<int64_t>(max(0, p.seq_lens[b])), cap)) : 0;
        uint32_t stop[1] = {n > 0 ? static_cast<uint32_t>(n) : 0u};
        block_scan<1>(stop, carry_t, warp_sums);
        const bool over =
            n > 0 && (len + static_cast<int64_t>(n) > cap || stop[0] > static_cast<uint32_t>(p.d.num_slots));
        const int held = blocks_of(len);
        const uint32_t nd = n > 0 && !over ? blocks_of(len + n) - held : 0;
        uint32_t sums[2] = {nd, n < 0 ? static_cast<uint32_t>(held) : 0u};
        block_scan<2>(sums, carry, warp_sums);
        if (in) {
            tok[b] = stop[0];
            need[b] = sums[0];
            back[b] = sums[1];
            held_len[b] = len;
            okay[b] = n < 0 ? 3 : over ? 0 : nd > 0 ? 2 : 1;  // 2: served if the blocks suffice
            if (over) status |= KVD_STATUS_CACHE_FULL;
        }
        __syncthreads();
        const int last = min(B, b0 + static_cast<int>(blockDim.x)) - 1;
        carry_t[0] = tok[last];
        carry[0] = need[last];
        carry[1] = back[last];
    }
    // the inputs are read: count this CTA
    if (threadIdx.x == 0) {
        s_last = 1;
        if (gridDim.x > 1) {
            __threadfence();
            s_last = atomicInc(p.ticket, gridDim.x - 1) == gridDim.x - 1;
            __threadfence();
        }
    }
    const uint32_t total = sat_add(fc, carry[1]);  // stack height with the ended requests' blocks on top
    uint32_t most = 0;
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        if (okay[b] != 2) continue;
        if (need[b] <= total) {
            most = max(most, need[b]);
        } else {
            okay[b] = 0;
            status |= KVD_STATUS_NO_BLOCKS;
        }
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_popped, most);
    __syncthreads();
    const uint32_t popped = s_popped, left = total - popped;
    // Entry i of the stack.
    auto stack = [&](uint32_t i) -> int {
        if (i < fc) return p.free_blocks[i];
        const int b = first_above(back, B, i - fc);
        const uint32_t before = b > 0 ? back[b - 1] : 0u;
        return p.table[b * p.d.block_table_stride + (i - fc - before)];
    };
    const uint32_t stride = gridDim.x * blockDim.x, me = blockIdx.x * blockDim.x + threadIdx.x;
    // slots
    const uint32_t tokens = min(tok[B - 1], static_cast<uint32_t>(p.d.num_slots));
    for (uint32_t t = me; t < static_cast<uint32_t>(p.d.num_slots); t += stride) {
        int64_t slot = -1;
        if (t < tokens) {
            const int b = first_above(tok, B, t);
            if (okay[b]) {
                const int len = held_len[b], held = blocks_of(len);
                const uint32_t pos = len + (t - (b > 0 ? tok[b - 1] : 0u));
                const int j = static_cast<int>(p.by_bs.div(pos));
                const int id = j < held ? p.table[b * p.d.block_table_stride + j]
                                        : stack(total - 1 - ((b > 0 ? need[b - 1] : 0u) + (j - held)));
                if (id >= 0 && id < NB) slot = static_cast<int64_t>(id) * bs + (pos - static_cast<uint32_t>(j) * bs);
                else status |= KVD_STATUS_BAD_BLOCK;
            }
        }
        p.slots[t] = slot;
    }
    // table entries of the new blocks
    for (uint32_t k = me; k < popped; k += stride) {
        const int b = first_above(need, B, k);
        const uint32_t before = b > 0 ? need[b - 1] : 0u;
        p.table[b * p.d.block_table_stride + blocks_of(held_len[b]) + (k - before)] = stack(total - 1 - k);
    }
    // ended requests' blocks that stay on the stack
    for (uint32_t i = fc + me; i < left; i += stride) {
        if (i < static_cast<uint32_t>(NB)) p.free_blocks[i] = stack(i);
        else status |= KVD_STATUS_BAD_BLOCK;  // more blocks than the pool has: some were given back twice
    }
    if (blockIdx.x == 0) {
        for (int b = threadIdx.x; b <= B; b += blockDim.x)
            p.starts[b] = b > 0 ? min(tok[b - 1], static_cast<uint32_t>(p.d.num_slots)) : 0;
        if (status) record_status(status);
    } else if (status & KVD_STATUS_BAD_BLOCK) {
        record_status(KVD_STATUS_BAD_BLOCK);
    }
    if (!s_last) return;
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        const int len = held_len[b];  // tokens of a served request: its share of the sums
        const uint32_t n = tok[b] - (b > 0 ? tok[b - 1] : 0u);
        p.lens_out[b] = okay[b] == 3 ? 0 : okay[b] ? len + static_cast<int>(n) : len;
    }
    if (threadIdx.x == 0) *p.count_out = static_cast<int32_t>(min(left, static_cast<uint32_t>(NB)));
}

// ------------------------------------------------------------- rows by slot
struct RowsParams {
    kvd_paged_rows_desc d;
    const void* k_rows;
    const void* v_rows;
    void* k_out;
    void* v_out;
    const int64_t* slots;
    int8_t* K;
    int8_t* V;
    float* ks;
    float* vs;
    int8_t* bounds;      // or nullptr
    float* bound_scale;
    int tile;            // tokens whose runs one CTA writes
    FastDiv by_bs, by_heads;
    int64_t n_slots;
};

// Block of a slot, -1 for one outside the pools.
__device__ __forceinline__ int block_of(const RowsParams& p, int64_t slot) {
    if (slot < 0 || slot >= p.n_slots) return -1;
    if (p.n_slots <= 0x7fffffffLL) return static_cast<int>(p.by_bs.div(static_cast<uint32_t>(slot)));
    return static_cast<int>(slot / p.d.block_size);
}

template <class T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen(float x) { return x; }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __half) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 1.5 * 2^23: adding it rounds a float below 2^22 to a whole number, ties to
// even, whose low byte is then the sum's low byte.
constexpr float kRound = 12582912.0f;

__device__ __forceinline__ uint32_t low_bytes(float2 a, float2 b) {
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                       __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}

// How a warp holds rows of D values: LPR lanes a row, 8 neighbouring values a
// lane, 32 / LPR rows at a time (D = 8 * LPR, 16-byte aligned rows); LPR = 0:
// any D <= 512, one row at a time, every 32nd value a lane.
template <int LPR>
struct Rows {
    static constexpr bool VEC = LPR > 0;
    static constexpr int LANES = VEC ? LPR : 32;  // lanes a row
    static constexpr int N = 32 / LANES;          // rows a warp holds
    static constexpr int E = VEC ? 8 : 16;        // values a lane
    static __device__ __forceinline__ int at(int l, int j) { return VEC ? l * 8 + j : l + 32 * j; }
    static __device__ __forceinline__ bool in(int l, int j, int D) { return VEC || l + 32 * j < D; }
    template <class T>
    static __device__ __forceinline__ void load(const T* row, int l, int D, float (&x)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = in(l, j, D) ? widen<T>(row[at(l, j)]) : 0.f;
    }
    static __device__ __forceinline__ void widen_codes(uint2 q, float (&x)[E]) {  // VEC
        float2 a, b;
        dequant4(q.x, a, b);
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
        dequant4(q.y, a, b);
        x[4] = a.x; x[5] = a.y; x[6] = b.x; x[7] = b.y;
    }
    static __device__ __forceinline__ void load_codes(const int8_t* row, int l, int D, float (&x)[E]) {
        if constexpr (VEC) {
            widen_codes(*reinterpret_cast<const uint2*>(row + l * 8), x);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) x[j] = in(l, j, D) ? static_cast<float>(row[at(l, j)]) : 0.f;
        }
    }
    template <class T>
    static __device__ __forceinline__ void store(T* row, int l, int D, const float (&x)[E]) {
        if constexpr (VEC && sizeof(T) == 4) {
            float4* out = reinterpret_cast<float4*>(row + l * 8);
            __stcs(out, make_float4(x[0], x[1], x[2], x[3]));
            __stcs(out + 1, make_float4(x[4], x[5], x[6], x[7]));
        } else if constexpr (VEC) {
            __stcs(reinterpret_cast<uint4*>(row + l * 8),
                   make_uint4(narrow2(x[0], x[1], T()), narrow2(x[2], x[3], T()), narrow2(x[4], x[5], T()),
                              narrow2(x[6], x[7], T())));
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (in(l, j, D)) row[at(l, j)] = narrow<T>(x[j]);
        }
    }
    // x: codes as whole floats
    static __device__ __forceinline__ void store_codes(int8_t* row, int l, int D, const float (&x)[E]) {
        if constexpr (VEC) {
            float2 e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = make_float2(x[2 * j] + kRound, x[2 * j + 1] + kRound);
            *reinterpret_cast<uint2*>(row + l * 8) = make_uint2(low_bytes(e[0], e[1]), low_bytes(e[2], e[3]));
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (in(l, j, D)) row[at(l, j)] = static_cast<int8_t>(x[j]);
        }
    }
    static __device__ __forceinline__ float amax(float a) {  // over the lanes of a row
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        return a;
    }
};

// A lane's 8 neighbouring values of a row, as loaded: words, so that they stay
// in registers.
template <class T>
struct Pack {
    static constexpr int W = static_cast<int>(sizeof(T)) * 2;  // 32-bit words
    uint32_t w[W];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < W; ++j) w[j] = 0u;
    }
    __device__ __forceinline__ void load(const T* x) {
#pragma unroll
        for (int j = 0; j < W; j += 4) {
            const uint4 q = __ldcs(reinterpret_cast<const uint4*>(x) + j / 4);
            w[j] = q.x; w[j + 1] = q.y; w[j + 2] = q.z; w[j + 3] = q.w;
        }
    }
    // values 2j and 2j + 1 as floats
    __device__ __forceinline__ float2 pair(int j) const {
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
        else return widen2(w[j], T());
    }
    static __device__ __forceinline__ float2 widen2(uint32_t x, __nv_bfloat16) {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
    static __device__ __forceinline__ float2 widen2(uint32_t x, __half) {
        return __half22float2(*reinterpret_cast<const __half2*>(&x));
    }
    static __device__ __forceinline__ float2 widen2(uint32_t x, float) { return make_float2(__uint_as_float(x), 0.f); }
    // bits of the largest magnitude as a float: ordered like magnitudes, infinities and NaN on top
    __device__ __forceinline__ uint32_t most() const {
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < W; ++j) m = max(m, w[j] & 0x7fffffffu);
            return m;
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
            return __float_as_uint(widen2(max(m & 0xffffu, m >> 16), T()).x);
        }
    }
};

// Any row by the rule of kvd_quant.cuh, divided value by value: x becomes the
// codes (as floats); returns the scale of the lane's row. All lanes call it.
template <int LPR>
__device__ __forceinline__ float quantise_divided(float (&x)[Rows<LPR>::E]) {
    using R = Rows<LPR>;
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < R::E; ++j) a = fmaxf(a, fabsf(x[j]));  // a NaN is left out
    a = R::amax(a);
    const float s = a == 0.f ? 0.f : a / 127.0f;
#pragma unroll
    for (int j = 0; j < R::E; ++j) x[j] = a == 0.f ? 0.f : fminf(fmaxf(rintf(x[j] / s), -127.0f), 127.0f);
    return s;
}

// Quotients x / s, correctly rounded, then rounded to whole numbers, plus
// kRound; ns = -s, yy = 1 / s rounded. q = x y, and twice q += (x - q s) y by
// fused multiply-adds (Markstein, IBM J. Res. Dev. 34, 1990: the second step
// starts from a neighbour of the quotient and an exact remainder). For
// magnitudes whose remainders and reciprocals are normal numbers.
__device__ __forceinline__ float2 quotient(float2 x, float2 ns, float2 yy) {
    float2 q = __fmul2_rn(x, yy);
    q = __ffma2_rn(__ffma2_rn(q, ns, x), yy, q);
    q = __ffma2_rn(__ffma2_rn(q, ns, x), yy, q);
    return __fadd2_rn(q, make_float2(kRound, kRound));
}

// The same for 16-bit values, by the reciprocal in two parts, y + ye with
// ye = (1 - s y) y: q = x y + (x ye), three operations instead of six. Equal to
// the division's codes for all pairs of 8-bit and of 11-bit significands of
// value and maximum and all exponents between them (checked exhaustively).
__device__ __forceinline__ float2 quotient16(float2 x, float2 yy, float2 ye) {
    return __fadd2_rn(__ffma2_rn(x, yy, __fmul2_rn(x, ye)), make_float2(kRound, kRound));
}

// The K and V rows that a warp holds (LPR lanes each), by the rule of
// kvd_quant.cuh: code words, the scales of the lane's rows, and in `code` the
// K codes as floats.
//  * Even lanes reduce and divide for K, odd lanes for V, so both rows' scales
//    and reciprocals cost one row's work; 8 or more lanes share a row.
//  * Every quotient x / s has to be the correctly rounded one (for 16-bit rows
//    it often lies on a half exactly, where the code depends on its last bit):
//    quotient() gives it in packed pairs and without a branch.
//  * Rows that are not finite, or so small or large that a remainder or
//    reciprocal leaves the normal numbers, are divided instead.
template <class T, int LPR>
__device__ __forceinline__ void quantise_pair(const Pack<T>& pk, const Pack<T>& pv, float2 (&code)[4], uint2& kw,
                                              uint2& vw, float& sk, float& sv) {
    const int lane = threadIdx.x & 31;
    const bool even = (lane & 1) == 0;
    const uint32_t mk = pk.most(), mv = pv.most();
    uint32_t m = max(even ? mk : mv, __shfl_xor_sync(0xffffffffu, even ? mv : mk, 1));
#pragma unroll
    for (int o = 2; o < LPR; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool plain = m == 0 || (m >= 0x21800000u && m <= 0x5d800000u);  // 2^-60 .. 2^60
    if (!__all_sync(0xffffffffu, plain)) {
        float k[8], v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 a = pk.pair(j), b = pv.pair(j);
            k[2 * j] = a.x; k[2 * j + 1] = a.y; v[2 * j] = b.x; v[2 * j + 1] = b.y;
        }
        sk = quantise_divided<LPR>(k);
        sv = quantise_divided<LPR>(v);
        float2 e[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            code[j] = make_float2(k[2 * j], k[2 * j + 1]);
            e[j] = make_float2(k[2 * j] + kRound, k[2 * j + 1] + kRound);
            e[4 + j] = make_float2(v[2 * j] + kRound, v[2 * j + 1] + kRound);
        }
        kw = make_uint2(low_bytes(e[0], e[1]), low_bytes(e[2], e[3]));
        vw = make_uint2(low_bytes(e[4], e[5]), low_bytes(e[6], e[7]));
        return;
    }
    // m / 127 by one such step: equal to the division for all 2^23 significands
    const float a = __uint_as_float(m), y127 = 1.0f / 127.0f;
    float s = a * y127;
    s = fmaf(fmaf(s, -127.0f, a), y127, s);
    const float y = m == 0 ? 0.f : 1.0f / s;
    const int mine = lane & ~1;
    sk = __shfl_sync(0xffffffffu, s, mine);
    sv = __shfl_sync(0xffffffffu, s, mine + 1);
    const float yk = __shfl_sync(0xffffffffu, y, mine), yv = __shfl_sync(0xffffffffu, y, mine + 1);
    auto row = [](const Pack<T>& x, float s1, float y1, float2 (&e)[4]) {
        const float ye = fmaf(-s1, y1, 1.0f) * y1;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            e[j] = sizeof(T) == 2 ? quotient16(x.pair(j), make_float2(y1, y1), make_float2(ye, ye))
                                  : quotient(x.pair(j), make_float2(-s1, -s1), make_float2(y1, y1));
    };
    float2 e[4];
    row(pk, sk, yk, e);
#pragma unroll
    for (int j = 0; j < 4; ++j) code[j] = __fadd2_rn(e[j], make_float2(-kRound, -kRound));
    kw = make_uint2(low_bytes(e[0], e[1]), low_bytes(e[2], e[3]));
    row(pv, sv, yv, e);
    vw = make_uint2(low_bytes(e[0], e[1]), low_bytes(e[2], e[3]));
}

constexpr int kRowWarps = 4;

// Writes: a run is a maximal stretch of tokens in one block, skipped tokens
// (slot -1) aside. One CTA per (tile of tokens, KV head) takes the runs that
// start in its tile, one after the other, its warps the rows of a run in turn.
// A run's key bounds are then the maximum and minimum over values that the CTA
// holds in registers (and the block's earlier tokens, read from the pool), so
// the bounds cost no second pass and no exchange between CTAs. Heads are the
// fast index of the grid: CTAs that run together read neighbouring rows. The
// first rows are loaded beside the slots, before the run is known.
// Bound: latency. For long maps no resource is full: 59 % of the issue slots,
// 24 % of the DRAM rate, a third of the warps at 24 an SM, so too little is under
// way (32,768 bf16 rows x 8 heads of 128 in blocks of 64 take 70.9 us, 58.5
// without bounds; their 204 MB would take 31 at the copy rate). For short ones it
// is the chain of dependent loads (256 decode rows in a pool of 512 blocks of 16:
// 6.2 us, 3.4 without bounds). A refused prompt's slots of -1 are looked through
// 32 at a time behind a run and 128 in front of one, a load after the other:
// 30,000 of them between prompts of 1,990 tokens cost 235 us (8,000: 56 to 58).
// CTAs of four warps: six an SM (80 registers, 52 to 104 bytes spilled); five,
// seven and eight took 93, 89 and 93 us when six took 82. CTAs of one: 20 an SM
// (4 to 32 bytes spilled), 256 decode rows 5.9 us when 24 took 7.0.
template <class T, int LPR, int W>
__global__ void __launch_bounds__(32 * W, LPR ? (W == 1 ? 20 : 24 / W) : 1) write_kernel(const RowsParams p) {
    using R = Rows<LPR>;
    constexpr int E = R::E, STEP = W * R::N;
    extern __shared__ float write_smem[];  // [W][2][D] bounds of each warp
    __shared__ int s_odd[W];
    grid_dependency_wait();
    allow_dependents();
    const kvd_paged_rows_desc& d = p.d;
    const int D = d.head_dim, bs = d.block_size, nt = d.num_tokens;
    const int tile = static_cast<int>(p.by_heads.div(blockIdx.x));
    const int h = blockIdx.x - tile * d.num_kv_heads;
    const int t0 = tile * p.tile, t1 = min(nt, t0 + p.tile);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / R::LANES, l = lane % R::LANES;
    const T* k_rows = static_cast<const T*>(p.k_rows) + h * d.row_stride_h;
    const T* v_rows = static_cast<const T*>(p.v_rows) + h * d.row_stride_h;
    const int r0 = warp * R::N + sub;  // this lane's row of the STEP that the CTA holds
    // V's rows and codes lie at fixed distances from K's
    const int64_t v_rows_at = reinterpret_cast<const char*>(v_rows) - reinterpret_cast<const char*>(k_rows);
    const int64_t v_codes_at = p.V - p.K;
    const int64_t v_scales_at = reinterpret_cast<char*>(p.vs) - reinterpret_cast<char*>(p.ks);
    Pack<T> pk, pv;  // this lane's part of the next row
    auto fetch = [&](const T* row) {
        if constexpr (R::VEC) {
            pk.load(row);
            pv.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + v_rows_at));
        }
    };
    auto slot_at = [&](int v) -> int64_t { return v >= 0 && v < nt ? p.slots[v] : -1; };
    bool fresh = false;  // the next token with a slot is known to start a run
    int t = t0;
    while (t < t1) {  // every warp finds the same runs
        const int64_t here = slot_at(t + lane), s0 = __shfl_sync(0xffffffffu, here, 0);
        int64_t ahead = slot_at(t + 1 + lane);
        const T* next_row = k_rows + static_cast<int64_t>(t + r0) * d.row_stride_t + l * 8;
        if (t + r0 < nt) fetch(next_row);
        else if constexpr (R::VEC) { pk.clear(); pv.clear(); }
        const int blk = block_of(p, s0);
        if (blk < 0) {  // on to the next token with a slot
            const bool valid = here >= 0 && here < p.n_slots;
            const uint32_t some = __ballot_sync(0xffffffffu, valid);
            const int skip = some ? __ffs(some) - 1 : 32;
            if (lane < skip && here != -1) record_status(KVD_STATUS_BAD_BLOCK);
            t += skip;
            continue;
        }
        const int64_t base = static_cast<int64_t>(blk) * bs;
        const int first = static_cast<int>(s0 - base);
        // up to the first later token of another block; `last` is the run's last token with a slot
        int end = t + 1, last = t, held = 1;
        bool plain = true;
        for (;;) {
            const int v = end + lane;
            const bool valid = ahead >= 0 && ahead < p.n_slots;
            const bool mine = valid && ahead >= base && ahead < base + bs;
            if (ahead != -1 && !valid) record_status(KVD_STATUS_BAD_BLOCK);
            const uint32_t stop = __ballot_sync(0xffffffffu, v >= nt || (valid && !mine));
            const uint32_t before = stop ? (1u << (__ffs(stop) - 1)) - 1u : 0xffffffffu;
            const uint32_t mb = __ballot_sync(0xffffffffu, mine) & before;
            plain &= (__ballot_sync(0xffffffffu, mine && ahead != s0 + (v - t)) & before) == 0;
            held += __popc(mb);
            if (mb) last = end + 31 - __clz(mb);
            if (stop) {
                end += __ffs(stop) - 1;
                break;
            }
            end += 32;
            ahead = slot_at(end + lane);
        }
        plain &= held == last - t + 1;  // token i of the run has place first + i - t
        if (!fresh) {
            // A run that started in an earlier tile is its CTA's: look for the token with a slot before
            // t (tokens of a block come in order, so place 0 starts a run), 128 tokens at a time
            // because refused requests leave long gaps.
            fresh = true;
            bool goes_on = false;
            for (int u = t - 1; first > 0 && u >= 0; u -= 128) {
                int64_t s[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) s[x] = slot_at(u - 32 * x - lane);
                uint32_t found = 0;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (found) break;
                    const bool valid = s[x] >= 0 && s[x] < p.n_slots;
                    found = __ballot_sync(0xffffffffu, valid);
                    if (found)
                        goes_on = __shfl_sync(0xffffffffu, s[x] >= base && s[x] < base + bs, __ffs(found) - 1);
                }
                if (found) break;
            }
            if (goes_on) {
                t = end;
                continue;
            }
        }
        float hi[E], lo[E];
        bool odd = false;  // a token scale that is not finite
#pragma unroll
        for (int j = 0; j < E; ++j) { hi[j] = -INFINITY; lo[j] = INFINITY; }
        int8_t* K = p.K + blk * d.kv_stride_block + h * d.kv_stride_h;
        int8_t* V = p.V + blk * d.kv_stride_block + h * d.kv_stride_h;
        float* ks = p.ks + blk * d.sc_stride_block + h * d.sc_stride_h;
        float* vs = p.vs + blk * d.sc_stride_block + h * d.sc_stride_h;
        auto widen_bounds = [&](const float (&c)[E], float s) {
            odd |= !isfinite(s);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const float v = c[j] * s;
                hi[j] = fmaxf(hi[j], v);
                lo[j] = fminf(lo[j], v);
            }
        };
        // the rows in hand, to code row `ko` with scale `so`
        auto put = [&](bool in, int8_t* ko, float* so) {
            if constexpr (R::VEC) {
                float2 code[4];
                uint2 kw, vw;
                float sk, sv;
                quantise_pair<T, LPR>(pk, pv, code, kw, vw, sk, sv);
                if (!in) return;
                *reinterpret_cast<uint2*>(ko) = kw;
                *reinterpret_cast<uint2*>(ko + v_codes_at) = vw;
                if (l == 0) {
                    *so = sk;
                    *reinterpret_cast<float*>(reinterpret_cast<char*>(so) + v_scales_at) = sv;
                }
                if (p.bounds) {
                    odd |= !isfinite(sk);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 v = __fmul2_rn(code[j], make_float2(sk, sk));
                        hi[2 * j] = fmaxf(hi[2 * j], v.x);
                        lo[2 * j] = fminf(lo[2 * j], v.x);
                        hi[2 * j + 1] = fmaxf(hi[2 * j + 1], v.y);
                        lo[2 * j + 1] = fminf(lo[2 * j + 1], v.y);
                    }
                }
            }
        };
        auto earlier = [&](int o) {  // a token that an earlier call wrote
            float c[E];
            R::load_codes(K + o * d.kv_stride_t, l, D, c);
            widen_bounds(c, ks[o]);
        };
        if (p.bounds) {
#pragma unroll 2
            for (int o = r0; o < first; o += STEP) earlier(o);
        }
        if (R::VEC && plain) {  // consecutive places: pointers advance, the next rows load meanwhile
            int8_t* ko = K + static_cast<int64_t>(first + r0) * d.kv_stride_t + l * 8;
            float* so = ks + first + r0;
            for (int left = last - t + 1; left > 0; left -= STEP) {
                const Pack<T> ck = pk, cv = pv;
                const bool more = left - STEP > r0;
                next_row += STEP * d.row_stride_t;
                Pack<T> nk = ck, nv = cv;
                if (more) {
                    nk.load(next_row);
                    nv.load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(next_row) + v_rows_at));
                }
                put(left > r0, ko, so);
                pk = nk;
                pv = nv;
                ko += STEP * d.kv_stride_t;
                so += STEP;
            }
        } else {
            for (int i0 = t; i0 <= last; i0 += STEP) {
                const int i = i0 + r0;
                const int64_t s = i <= last ? p.slots[i] : -1;
                const bool in = s >= base && s < base + bs;
                const int o = in ? static_cast<int>(s - base) : 0;
                const int64_t row = static_cast<int64_t>(min(i, nt - 1)) * d.row_stride_t;
                if constexpr (R::VEC) {
                    fetch(k_rows + row + l * 8);
                    put(in, K + o * d.kv_stride_t + l * 8, ks + o);
                } else {
                    float xk[E], xv[E];
                    R::load(k_rows + row, l, D, xk);
                    R::load(v_rows + row, l, D, xv);
                    const float sk = quantise_divided<LPR>(xk), sv = quantise_divided<LPR>(xv);
                    if (!in) continue;
                    R::store_codes(K + o * d.kv_stride_t, l, D, xk);
                    R::store_codes(V + o * d.kv_stride_t, l, D, xv);
                    if (l == 0) { ks[o] = sk; vs[o] = sv; }
                    if (p.bounds) widen_bounds(xk, sk);
                }
            }
        }
        if (p.bounds && !plain) {  // places left out between the run's tokens hold earlier ones
            for (int i = t + r0; i < last; i += STEP) {
                const int64_t s = p.slots[i];
                if (s < base || s >= base + bs) continue;
                int next = i + 1;
                while (next < last && (p.slots[next] < base || p.slots[next] >= base + bs)) ++next;
                for (int o = static_cast<int>(s - base) + 1, stop = static_cast<int>(p.slots[next] - base); o < stop; ++o)
                    earlier(o);
            }
        }
        if (p.bounds) {
            __syncwarp();
#pragma unroll
            for (int x = R::LANES; x < 32; x <<= 1) {  // over the rows that the warp held
                odd |= __shfl_xor_sync(0xffffffffu, odd, x);
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    hi[j] = fmaxf(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], x));
                    lo[j] = fminf(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], x));
                }
            }
            if constexpr (W > 1) {
                float* mine = write_smem + warp * 2 * D;
                if (sub == 0) {
#pragma unroll
                    for (int j = 0; j < E; ++j)
                        if (R::in(l, j, D)) { mine[R::at(l, j)] = hi[j]; mine[D + R::at(l, j)] = lo[j]; }
                }
                if (lane == 0) s_odd[warp] = odd;
                __syncthreads();
            }
            if (warp == 0) {
                float most = 0.f;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    if (!R::in(l, j, D)) { hi[j] = lo[j] = 0.f; continue; }
#pragma unroll
                    for (int w = 1; w < W; ++w) {
                        hi[j] = fmaxf(hi[j], write_smem[w * 2 * D + R::at(l, j)]);
                        lo[j] = fminf(lo[j], write_smem[w * 2 * D + D + R::at(l, j)]);
                    }
                    most = fmaxf(most, fmaxf(fabsf(hi[j]), fabsf(lo[j])));
                }
                for (int w = 1; w < W; ++w) odd |= s_odd[w] != 0;
                most = R::amax(most);
                const float step = odd ? NAN : most / 127.0f;
                int8_t* bound = p.bounds + (static_cast<int64_t>(blk) * d.num_kv_heads + h) * 2 * D;
                // the upper row as the negated lower row of the negated values; with two or more
                // rows of lanes a warp, the first rounds one and the second the other
                auto lower = [&](float (&x)[E], bool flip, int8_t* out) {
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const float v = flip ? -x[j] : x[j];
                        const float f = step > 0.f ? fminf(fmaxf(floorf(v / step), -127.f), 127.f) : 0.f;
                        x[j] = flip ? -f : f;
                    }
                    R::store_codes(out, l, D, x);
                };
                if constexpr (R::N > 1) {
#pragma unroll
                    for (int j = 0; j < E; ++j) lo[j] = sub == 0 ? hi[j] : lo[j];
                    if (sub < 2) lower(lo, sub == 0, bound + sub * D);
                } else {
                    lower(hi, true, bound);
                    lower(lo, false, bound + D);
                }
                if (lane == 0) p.bound_scale[static_cast<int64_t>(blk) * d.num_kv_heads + h] = step;
            }
            if constexpr (W > 1) __syncthreads();  // the bounds rows are written again
        }
        t = end;
    }
}

// Reads: rows (token, head) in order, a warp holding U times R::N neighbours,
// their codes as loaded until all loads are under way. 16-bit outputs: two
// rows a lane take 43.9 us for 32,768 x 8 rows of 128 (201 MB, 4.6 TB/s; a
// plain copy of 134 MB, as many bytes written, takes 41.9), one 47.2, three
// 46.1; 32-bit ones: two take 7.9 us for 2,000 x 8 rows, one 6.2. Bound: HBM,
// two thirds of the bytes being writes.
template <class T, int LPR>
constexpr int kReadRows = LPR && sizeof(T) == 2 ? 2 : 1;

template <class T, int LPR>
__global__ void __launch_bounds__(32 * kRowWarps) read_kernel(const RowsParams p) {
    using R = Rows<LPR>;
    constexpr int E = R::E, U = kReadRows<T, LPR>;
    grid_dependency_wait();
    allow_dependents();
    const kvd_paged_rows_desc& d = p.d;
    const int D = d.head_dim, H = d.num_kv_heads;
    const int lane = threadIdx.x & 31, sub = lane / R::LANES, l = lane % R::LANES;
    const uint32_t rows = static_cast<uint32_t>(d.num_tokens) * H;
    const uint32_t step = gridDim.x * kRowWarps * (R::N * U);
    const int64_t v_codes_at = p.V - p.K, v_rows_at = static_cast<char*>(p.v_out) - static_cast<char*>(p.k_out);
    for (uint32_t r0 = (blockIdx.x * kRowWarps + (threadIdx.x >> 5)) * (R::N * U); r0 < rows; r0 += step) {
        uint2 kw[U], vw[U];      // VEC
        float xk[E], xv[E];      // otherwise (U = 1)
        float sk[U], sv[U];
        T* out[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t r = r0 + u * R::N + sub;
            out[u] = nullptr;
            kw[u] = vw[u] = make_uint2(0u, 0u);
            sk[u] = sv[u] = 0.f;
            if constexpr (!R::VEC) {
#pragma unroll
                for (int j = 0; j < E; ++j) xk[j] = xv[j] = 0.f;
            }
            if (r >= rows) continue;
            const int t = static_cast<int>(p.by_heads.div(r)), h = static_cast<int>(r) - t * H;
            out[u] = static_cast<T*>(p.k_out) + t * d.row_stride_t + h * d.row_stride_h;
            const int64_t slot = p.slots[t];
            const int blk = block_of(p, slot);
            if (blk < 0) {
                if (slot != -1 && h == 0 && l == 0) record_status(KVD_STATUS_BAD_BLOCK);
                continue;
            }
            const int64_t o = slot - static_cast<int64_t>(blk) * d.block_size;
            const int8_t* at = p.K + blk * d.kv_stride_block + h * d.kv_stride_h + o * d.kv_stride_t;
            const int64_t sc = blk * d.sc_stride_block + h * d.sc_stride_h + o;
            if constexpr (R::VEC) {
                kw[u] = *reinterpret_cast<const uint2*>(at + l * 8);
                vw[u] = *reinterpret_cast<const uint2*>(at + v_codes_at + l * 8);
            } else {
                R::load_codes(at, l, D, xk);
                R::load_codes(at + v_codes_at, l, D, xv);
            }
            sk[u] = p.ks[sc];
            sv[u] = p.vs[sc];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!out[u]) continue;
            if constexpr (R::VEC) {
                R::widen_codes(kw[u], xk);
                R::widen_codes(vw[u], xv);
            }
#pragma unroll
            for (int j = 0; j < E; ++j) { xk[j] *= sk[u]; xv[j] *= sv[u]; }
            R::store(out[u], l, D, xk);
            R::store(reinterpret_cast<T*>(reinterpret_cast<char*>(out[u]) + v_rows_at), l, D, xv);
        }
    }
}

template <class T, int LPR>
cudaError_t launch_rows(RowsParams& p, bool write, cudaStream_t st) {
    const kvd_paged_rows_desc& d = p.d;
    const int64_t rows = static_cast<int64_t>(d.num_tokens) * d.num_kv_heads;
    if (write) {
        // One warp a CTA, or four that share a run. In us, bf16 rows of 8 heads x 128, one warp | four, for
        // rows that each lie in a block of their own (decode: a run of one and the block's earlier tokens)
        // and for whole blocks (prompt), anywhere in a pool of 131,072 tokens:
        //   block_size   decode 256  decode 1,000   prompt 250   prompt 5,000  prompt 20,000
        //       16         7.6 | 17     21 | 56      6.3 |  7.2     13 | 22       38 | 62
        //       32         9.1 | 18     25 | 62      9.1 |  7.9     18 | 17       35 | 44
        //       64          12 | 20     38 | 68       15 |  9.4     27 | 17       34 | 38
        //      128          19 | 21     67 | 88       25 |  13      41 | 23       57 | 43
        // Between, blocks of 33 to 127 tokens, calls of up to 64 rows an SM are taken for decode steps, which
        // gain more by it than a prompt loses (1,000 tokens in blocks of 64: 38 | 68 against 19 | 11).
        const bool one = LPR && (d.block_size <= 32 || (d.block_size < 128 && rows <= 64 * device_sm_count()));
        // Tiles: about the CTAs that the GPU holds at once (20 of one warp an SM), or twice as many (6 of four):
        // with 10 or 40 of one warp 1,000 decode rows took 31 or 19 us, 5,000 prompt rows 16 or 18; with 6 or
        // 24 of four 256 decode rows in blocks of 128 took 28 or 24 us, 20,000 prompt rows 40 or 47.
        const int64_t per = rows / ((one ? 20 : 12) * device_sm_count());
        const int most = d.block_size < 64 ? 64 : d.block_size > 256 ? 256 : d.block_size;
        p.tile = static_cast<int>(per < 1 ? 1 : per > most ? most : per);
        const int64_t grid = static_cast<int64_t>((d.num_tokens + p.tile - 1) / p.tile) * d.num_kv_heads;
        if (one)
            return launch_after(write_kernel<T, LPR, 1>, static_cast<unsigned>(grid), 32, 0, st, p);
        return launch_after(write_kernel<T, LPR, kRowWarps>, static_cast<unsigned>(grid), 32 * kRowWarps,
                            sizeof(float) * kRowWarps * 2 * d.head_dim, st, p);
    }
    const int64_t per = kRowWarps * Rows<LPR>::N * kReadRows<T, LPR>;
    int64_t grid = (rows + per - 1) / per;
    const int64_t most = static_cast<int64_t>(device_sm_count()) * 16;
    if (grid > most) grid = most;
    return launch_after(read_kernel<T, LPR>, static_cast<unsigned>(grid), 32 * kRowWarps, 0, st, p);
}

template <class T>
cudaError_t launch_rows_t(RowsParams& p, bool write, bool vec, cudaStream_t st) {
    if (vec && p.d.head_dim == 64) return launch_rows<T, 8>(p, write, st);
    if (vec && p.d.head_dim == 128) return launch_rows<T, 16>(p, write, st);
    if (vec && p.d.head_dim == 256) return launch_rows<T, 32>(p, write, st);
    return launch_rows<T, 0>(p, write, st);
}

bool rows_ok(const kvd_paged_rows_desc* d) {
    if (!d || d->num_tokens < 0 || d->num_kv_heads < 1 || d->head_dim < 1 || d->head_dim > 512) return false;
    if (d->block_size < 1 || d->num_blocks < 1) return false;
    if (static_cast<int64_t>(d->num_tokens) * d->num_kv_heads > 0x7fff0000LL) return false;
    return d->flags == 0 || d->flags == KVD_FLAG_Q_BF16 || d->flags == KVD_FLAG_Q_F16;
}

cudaError_t rows_call(RowsParams& p, const void* a, const void* b, bool write, cudaStream_t st) {
    const kvd_paged_rows_desc& d = p.d;
    p.by_bs = FastDiv(d.block_size);
    p.by_heads = FastDiv(d.num_kv_heads);
    p.n_slots = static_cast<int64_t>(d.num_blocks) * d.block_size;
    // vector access: every row of values and of codes starts on 16 bytes
    const int64_t es = d.flags ? 2 : 4;
    auto al = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    const bool vec = al(a) && al(b) && al(p.K) && al(p.V) && al(p.bounds) &&
                     (((d.row_stride_t | d.row_stride_h) * es) & 15) == 0 &&
                     ((d.kv_stride_block | d.kv_stride_h | d.kv_stride_t) & 15) == 0;
    cudaError_t e;
    if (d.flags & KVD_FLAG_Q_BF16) e = launch_rows_t<__nv_bfloat16>(p, write, vec, st);
    else if (d.flags & KVD_FLAG_Q_F16) e = launch_rows_t<__half>(p, write, vec, st);
    else e = launch_rows_t<float>(p, write, vec, st);
    if (e == cudaSuccess) ++*launch_counter();
    return e;
}

// --------------------------------------------------------------------- select
// Two kernels: scores (kvd_score_tc.cu, or score_any_kernel for other shapes),
// spread evenly over the GPU whatever the lengths are, then one CTA per
// (request, KV head) that finds the threshold and writes the table.

// Scores for head dims other than 64, 128 and 256 and groups of more than 64
// heads: a warp a CTA, query codes in shared memory, as many heads at a time as
// 48 KB hold (95 of 512 dims). Bound: instructions; 16 x 512 blocks x 8 KV heads in
// groups of 4 take 97 us at head_dim 96 and 94 at 128, by tensor cores 12.
__global__ void __launch_bounds__(32) score_any_kernel(const SelectParams p, int heads) {
    extern __shared__ int8_t any_smem[];  // [heads][D] codes, padded to 4, then [heads] scales
    const kvd_block_select_desc& d = p.d;
    const int D = d.head_dim, H = d.num_kv_heads, G = d.num_q_heads / H, lane = threadIdx.x;
    float* scale = reinterpret_cast<float*>(any_smem + ((heads * D + 3) & ~3));
    const int chunks = (d.max_blocks_per_seq + 15) / 16, items = d.batch * H * chunks;
    grid_dependency_wait();
    allow_dependents();
    for (int it = blockIdx.x; it < items; it += gridDim.x) {  // 16 blocks of a row each
        ScoreItem I;
        I.row = it / chunks;
        I.i0 = (it - I.row * chunks) * 16;
        I.b = I.row / H;
        I.h = I.row - I.b * H;
        int n;
        select_len(d, I.b, n);
        if (n <= d.budget || I.i0 >= n) continue;
        I.m = min(16, n - I.i0);
        const int32_t* table = d.block_table + I.b * d.block_table_stride + I.i0;
        const int id = lane < I.m ? pool_id(d, table, lane) : -1;  // of this lane's block
        float best = -INFINITY;                                    // its score over the heads so far
        for (int g0 = 0; g0 < G; g0 += heads) {
            const int m = min(heads, G - g0);
            __syncwarp();
            for (int g = 0; g < m; ++g) {
                const int64_t q0 = I.b * d.q_stride_b + static_cast<int64_t>(I.h * G + g0 + g) * d.q_stride_h;
                float x[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = lane + 32 * j < D ? load_q(p.Q, q0 + lane + 32 * j, d.flags) : 0.f;
                const float s = quantise_divided<0>(x);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (lane + 32 * j < D) any_smem[g * D + lane + 32 * j] = static_cast<int8_t>(x[j]);
                if (lane == 0) scale[g] = s;
            }
            __syncwarp();
            for (int i = 0; i < I.m; ++i) {
                const int64_t at = static_cast<int64_t>(max(__shfl_sync(0xffffffffu, id, i), 0)) * H + I.h;
                const int8_t* r = p.bounds + at * (2 * D);
                for (int g = 0; g < m; ++g) {
                    int acc = 0;
                    for (int x = lane; x < D; x += 32) {
                        const int c = any_smem[g * D + x];
                        acc += c * (c > 0 ? r[x] : r[D + x]);
                    }
                    const float v = static_cast<float>(__reduce_add_sync(0xffffffffu, acc)) * scale[g];
                    if (lane == i) best = fmaxf(best, isnan(v) ? INFINITY : v);
                }
            }
        }
        if (lane < I.m)
            p.keys[static_cast<int64_t>(I.row) * d.max_blocks_per_seq + I.i0 + lane] =
                id < 0 ? kNoBlockKey : score_key(best * p.bound_scale[static_cast<int64_t>(id) * H + I.h]);
    }
}

// Threshold and table of one row per CTA. The keys are binned evenly between
// the lowest and highest finite score, which puts the threshold into a bin of
// few keys as a rule; their ranks then give it exactly. Where the bin holds
// too many (equal or very uneven scores), 8-bit radix passes over the keys
// find it instead. Each warp owns a stretch of the row's blocks, so the places
// of its blocks follow from counts. A row of up to 16 blocks a thread is held in
// registers, keys and pool ids, from one load to the end; longer rows are read
// again from L2. 256 threads where the table has up to 4,096 blocks a row, above
// that 1,024. Bound: latency, three loads in a row and seven barriers, and for
// many rows the instructions (57 % of the issue slots, four CTAs an SM).
// With the scores, 64 requests x 8 heads x up to 4,096 blocks take 89.4 us, 11 of
// them here: 100 when rows are read again, 93 by radix passes alone, 97 with 1,024
// threads a row. One request of 256 blocks a head takes 7.7 us (9.0 with 1,024
// threads), of 4,096 blocks 11.4 (11.0), of 8,192 15.4 (37 with 256).
constexpr int kPickEach = 16;  // keys a thread holds

template <int THREADS>
struct PickShared {
    static constexpr int WARPS = THREADS / 32;
    uint32_t hist[THREADS];  // a bin a thread
    uint32_t list[THREADS];  // keys whose ranks are counted, a thread each
    uint32_t range[2][WARPS];
    uint32_t scan[WARPS];
    uint32_t pick[3], found[2], listed;
    uint32_t count[2][WARPS];
};

// Sum of a number of each warp in front of this one.
template <int WARPS>
__device__ __forceinline__ uint32_t before_warp(const uint32_t (&of)[WARPS]) {
    const int lane = threadIdx.x & 31;
    return __reduce_add_sync(0xffffffffu, lane < static_cast<int>(threadIdx.x >> 5) ? of[lane % WARPS] : 0u);
}

// The bin (a thread each) that the need-th best key lies in: pick = bin, keys above it, keys in it.
template <int THREADS>
__device__ __forceinline__ void find_bin(PickShared<THREADS>& s, uint32_t need) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bin = THREADS - 1 - tid;
    const uint32_t mine = s.hist[bin];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) s.scan[warp] = upto;
    __syncthreads();
    upto += before_warp(s.scan);
    if (upto >= need && upto - mine < need) {
        s.pick[0] = bin;
        s.pick[1] = upto - mine;
        s.pick[2] = mine;
    }
    __syncthreads();
}

template <bool KEPT, int THREADS>
__device__ __forceinline__ void pick_row(const SelectParams& p, PickShared<THREADS>& s, int row, int n,
                                         const int32_t* table) {
    constexpr int WARPS = THREADS / 32;
    const kvd_block_select_desc& d = p.d;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t* all = p.keys + static_cast<int64_t>(row) * d.max_blocks_per_seq;
    int32_t* out = p.sel_table + static_cast<int64_t>(row) * d.budget;
    const int seg = ((n + WARPS - 1) / WARPS + 31) & ~31;  // KEPT: at most 32 * kPickEach
    const int s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
    const int lo = d.first, hi = n - d.last;  // scored blocks: [lo, hi); the others are always selected
    // Keys of blocks that are always selected and of places past the end: above and below all others.
    constexpr uint32_t kAlways = 0xffffffffu, kOutside = 0u;
    auto key_at = [&](int i) {
        const uint32_t k = i < s1 ? all[i] : kOutside;
        return i < s1 && (i < lo || i >= hi) ? kAlways : k;
    };
    auto scored = [](uint32_t k) { return k - 1u < kAlways - 1u; };
    uint32_t key[kPickEach], bins[kPickEach / 2] = {};  // bins: 16 bits a key
    int id[kPickEach];
    if constexpr (KEPT) {
#pragma unroll
        for (int j = 0; j < kPickEach; ++j) {
            const int i = s0 + 32 * j + lane;
            key[j] = key_at(i);
            id[j] = i < s1 ? table[i] : 0;
        }
    }
    // fn(j, key) for this warp's blocks s0 + 32 j + lane in order, all lanes together
    auto each = [&](auto fn) {
        if constexpr (KEPT) {
#pragma unroll
            for (int j = 0; j < kPickEach; ++j) {
                if (s0 + 32 * j >= s1) break;
                fn(j, key[j]);
            }
        } else {
#pragma unroll 4
            for (int j = 0; s0 + 32 * j < s1; ++j) fn(j, key_at(s0 + 32 * j + lane));
        }
    };
    constexpr uint32_t kInf = 0xff800000u, kNegInf = 0x007fffffu;  // keys of +inf and -inf
    uint32_t kmin = 0xffffffffu, kmax = 0u;
    each([&](int, uint32_t k) {
        if (k - (kNegInf + 1) < kInf - (kNegInf + 1)) {
            kmin = min(kmin, k);
            kmax = max(kmax, k);
        }
    });
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (lane == 0) { s.range[0][warp] = kmin; s.range[1][warp] = kmax; }
    __syncthreads();
    kmin = __reduce_min_sync(0xffffffffu, s.range[0][lane % WARPS]);
    kmax = __reduce_max_sync(0xffffffffu, s.range[1][lane % WARPS]);
    // Bin of a key: scores clamped to the finite ones' range, evenly divided, rounded by the addition
    // of 2^23 (a bin a thread). It never falls where the key rises. A range that is empty, or whose
    // width or reciprocal overflows, leaves few bins in use, with products that may be infinite or
    // NaN: those all end in the last bin.
    const bool some = kmin <= kmax;
    const float least = some ? key_score(kmin) : 0.f, most = some ? key_score(kmax) : 0.f, width = most - least;
    const float per = width > 0.f ? (THREADS - 1.5f) / width : 0.f;
    auto bin_of = [&](uint32_t k) -> uint32_t {
        const float s = fminf(fmaxf(key_score(k), least), most);  // the key of no block stands for a NaN: least
        return min(__float_as_uint(fmaf(s - least, per, 8388608.0f)) - 0x4b000000u, THREADS - 1u);
    };
    uint32_t need = static_cast<uint32_t>(d.budget - d.first - d.last);
    uint32_t threshold = kAlways - 1u, at_it = 0;  // selected: above the threshold, and the first at_it at it
    if (need > 0) {
        each([&](int j, uint32_t k) {
            const uint32_t bin = bin_of(k);
            if constexpr (KEPT) bins[j / 2] |= bin << (j % 2 * 16);
            if (scored(k)) atomicAdd(&s.hist[bin], 1u);
        });
        __syncthreads();
        find_bin(s, need);
        const uint32_t bin = s.pick[0], in_bin = s.pick[2];
        if (in_bin <= THREADS) {
            const uint32_t rest = need - s.pick[1];
            each([&](int j, uint32_t k) {
                bool here;
                if constexpr (KEPT) here = (bins[j / 2] >> (j % 2 * 16) & 0xffffu) == bin;
                else here = bin_of(k) == bin;
                if (here && scored(k)) s.list[atomicAdd(&s.listed, 1u)] = k;
            });
            __syncthreads();
            if (tid < static_cast<int>(in_bin)) {
                const uint32_t k = s.list[tid];
                uint32_t more = 0, same = 0;
#pragma unroll 4
                for (uint32_t j = 0; j < in_bin; ++j) {
                    more += s.list[j] > k;
                    same += s.list[j] == k;
                }
                if (more < rest && more + same >= rest) {
                    s.found[0] = k;
                    s.found[1] = rest - more;
                }
            }
            __syncthreads();
            threshold = s.found[0];
            at_it = s.found[1];
        } else {
            uint32_t mask = 0, prefix = 0;
            for (int sh = 24; sh >= 0; sh -= 8) {
                s.hist[tid] = 0u;
                __syncthreads();
                each([&](int, uint32_t k) {
                    if (scored(k) && (k & mask) == prefix) atomicAdd(&s.hist[(k >> sh) & 255u], 1u);
                });
                __syncthreads();
                find_bin(s, need);
                prefix |= s.pick[0] << sh;
                mask |= 255u << sh;
                need -= s.pick[1];
            }
            threshold = prefix;
            at_it = need;
        }
    }
    uint32_t above = 0, equal = 0;
    each([&](int, uint32_t k) {
        above += k > threshold;
        equal += k == threshold;
    });
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) { s.count[0][warp] = above; s.count[1][warp] = equal; }
    __syncthreads();
    above = before_warp(s.count[0]);
    equal = before_warp(s.count[1]);
    const uint32_t below = (1u << lane) - 1u;
    each([&](int j, uint32_t k) {
        const int i = s0 + 32 * j + lane;
        int block = 0;
        if constexpr (KEPT) block = id[j];
        else if (i < s1) block = table[i];
        const bool up = k > threshold, eq = k == threshold;
        const uint32_t ub = __ballot_sync(0xffffffffu, up), eb = __ballot_sync(0xffffffffu, eq);
        if ((ub | eb) == 0) return;
        const uint32_t e = equal + __popc(eb & below);
        if (up || (eq && e < at_it)) out[above + __popc(ub & below) + min(e, at_it)] = block;
        above += __popc(ub);
        equal += __popc(eb);
    });
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) pick_kernel(const SelectParams p) {
    __shared__ PickShared<THREADS> s;
    const kvd_block_select_desc& d = p.d;
    const int row = blockIdx.x, b = row / d.num_kv_heads;
    const int tid = threadIdx.x, k = d.budget;
    s.hist[tid] = 0u;
    if (tid == 0) s.listed = 0u;
    grid_dependency_wait();
    allow_dependents();
    int n;
    const int len = select_len(d, b, n);
    const int32_t* table = d.block_table + b * d.block_table_stride;
    if (tid == 0) p.sel_lens[row] = n <= k ? len : (k - n) * d.block_size + len;
    if (n <= k) {  // everything
        for (int i = tid; i < k; i += THREADS) {
            p.sel_table[static_cast<int64_t>(row) * k + i] = i < n ? table[i] : -1;
            if (i < n) pool_id(d, table, i);
        }
    } else if (n <= THREADS * kPickEach) {
        pick_row<true, THREADS>(p, s, row, n, table);
    } else {
        pick_row<false, THREADS>(p, s, row, n, table);
    }
}

cudaError_t launch_select(const SelectParams& p, cudaStream_t st) {
    const kvd_block_select_desc& d = p.d;
    const int64_t rows = static_cast<int64_t>(d.batch) * d.num_kv_heads;
    cudaError_t e;
    if (d.max_blocks_per_seq > d.budget) {  // else every row takes all its blocks
        if (score_tc_ok(p)) {
            e = launch_score_tc(p, st);
        } else {
            const int64_t items = rows * ((d.max_blocks_per_seq + 15) / 16), most = static_cast<int64_t>(device_sm_count()) * 16;
            const int G = d.num_q_heads / d.num_kv_heads, most_heads = (48 * 1024 - 4) / (d.head_dim + 4);
            const int heads = G < most_heads ? G : most_heads;
            const size_t smem = ((static_cast<size_t>(heads) * d.head_dim + 3) & ~size_t(3)) + sizeof(float) * heads;
            if (items > 0x7fff0000LL) return cudaErrorInvalidValue;
            e = launch_after(score_any_kernel, static_cast<unsigned>(items < most ? items : most), 32, smem, st, p, heads);
        }
        if (e != cudaSuccess) return e;
        ++*launch_counter();
    }
    if (d.max_blocks_per_seq <= 256 * kPickEach)
        e = launch_after(pick_kernel<256>, static_cast<unsigned>(rows), 256, 0, st, p);
    else
        e = launch_after(pick_kernel<1024>, static_cast<unsigned>(rows), 1024, 0, st, p);
    if (e == cudaSuccess) ++*launch_counter();
    return e;
}

}  // namespace
}  // namespace kvd

using namespace kvd;

namespace {
bool plan_ok(const kvd_paged_plan_desc* d) {
    if (!d || d->batch < 1 || d->batch > kPlanMaxBatch || d->block_size < 1 || d->num_blocks < 1) return false;
    if (d->max_blocks_per_seq < 1 || d->num_slots < 0 || d->num_slots == 0x7fffffff) return false;
    if (d->block_table_stride < d->max_blocks_per_seq) return false;
    return static_cast<int64_t>(d->max_blocks_per_seq) * d->block_size <= 0x7fffffffLL;
}
}  // namespace

extern "C" size_t kvd_paged_plan_workspace_size(const kvd_paged_plan_desc* desc) { return plan_ok(desc) ? 16 : 0; }

extern "C" cudaError_t kvd_paged_plan_launch(const kvd_paged_plan_desc* desc, const int32_t* seq_lens,
                                             const int32_t* new_lens, int32_t* block_table, int32_t* free_blocks,
                                             const int32_t* free_count, int64_t* slot_map, int32_t* token_starts,
                                             int32_t* seq_lens_out, int32_t* free_count_out, void* workspace,
                                             size_t workspace_bytes, cudaStream_t stream) {
    *launch_counter() = 0;
    if (!plan_ok(desc) || !seq_lens || !new_lens || !block_table || !free_blocks || !free_count || !token_starts ||
        !seq_lens_out || !free_count_out || (!slot_map && desc->num_slots > 0))
        return cudaErrorInvalidValue;
    if (!workspace || workspace_bytes < kvd_paged_plan_workspace_size(desc) ||
        (reinterpret_cast<uintptr_t>(workspace) & 3) != 0)
        return cudaErrorInvalidValue;
    PlanParams p{*desc, seq_lens, new_lens, block_table, free_blocks, free_count, slot_map, token_starts,
                 seq_lens_out, free_count_out, static_cast<unsigned int*>(workspace),
                 FastDiv(static_cast<uint32_t>(desc->block_size))};
    const unsigned block = desc->batch <= 256 ? 256 : 1024;
    const size_t smem = static_cast<size_t>(desc->batch) * kPlanBytes;
    static PerDeviceOnce once;
    cudaError_t e = once.run([] {
        return cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kPlanMaxBatch * kPlanBytes);
    });
    if (e != cudaSuccess) return e;
    int64_t grid = (static_cast<int64_t>(desc->num_slots) + block - 1) / block;
    if (grid > device_sm_count()) grid = device_sm_count();
    if (grid < 1) grid = 1;
    e = launch_after(plan_kernel, static_cast<unsigned>(grid), block, smem, stream, p);
    if (e == cudaSuccess) *launch_counter() = 1;
    return e;
}

extern "C" cudaError_t kvd_paged_write_launch(const kvd_paged_rows_desc* desc, const void* k_new, const void* v_new,
                                              const int64_t* slot_map, int8_t* K_pool, int8_t* V_pool,
                                              float* k_scale_pool, float* v_scale_pool, int8_t* bounds,
                                              float* bound_scale, cudaStream_t stream) {
    *launch_counter() = 0;
    if (!rows_ok(desc)) return cudaErrorInvalidValue;
    if (desc->num_tokens == 0) return cudaSuccess;
    if (!k_new || !v_new || !slot_map || !K_pool || !V_pool || !k_scale_pool || !v_scale_pool ||
        (bounds == nullptr) != (bound_scale == nullptr))
        return cudaErrorInvalidValue;
    RowsParams p{*desc, k_new, v_new, nullptr, nullptr, slot_map, K_pool, V_pool, k_scale_pool, v_scale_pool,
                 bounds, bound_scale, 1, FastDiv(), FastDiv(), 0};
    return rows_call(p, k_new, v_new, true, stream);
}

extern "C" cudaError_t kvd_paged_read_launch(const kvd_paged_rows_desc* desc, const int64_t* slot_map,
                                             const int8_t* K_pool, const int8_t* V_pool, const float* k_scale_pool,
                                             const float* v_scale_pool, void* k_out, void* v_out,
                                             cudaStream_t stream) {
    *launch_counter() = 0;
    if (!rows_ok(desc)) return cudaErrorInvalidValue;
    if (desc->num_tokens == 0) return cudaSuccess;
    if (!slot_map || !K_pool || !V_pool || !k_scale_pool || !v_scale_pool || !k_out || !v_out)
        return cudaErrorInvalidValue;
    RowsParams p{*desc, nullptr, nullptr, k_out, v_out, slot_map, const_cast<int8_t*>(K_pool),
                 const_cast<int8_t*>(V_pool), const_cast<float*>(k_scale_pool), const_cast<float*>(v_scale_pool),
                 nullptr, nullptr, 1, FastDiv(), FastDiv(), 0};
    return rows_call(p, k_out, v_out, false, stream);
}

namespace {
bool select_ok(const kvd_block_select_desc* p) {
    if (!p) return false;
    const kvd_block_select_desc& d = *p;
    if (d.batch < 1 || d.num_q_heads < 1 || d.num_kv_heads < 1 || d.num_q_heads % d.num_kv_heads != 0 ||
        d.head_dim < 1 || d.head_dim > 512 || d.block_size < 1 || d.num_blocks < 1)
        return false;
    if (d.max_blocks_per_seq < 1 || d.block_table_stride < d.max_blocks_per_seq ||
        static_cast<int64_t>(d.max_blocks_per_seq) * d.block_size > 0x7fffffffLL)
        return false;
    if (d.budget < 1 || d.first < 0 || d.last < 1 || d.first > d.budget - d.last) return false;
    // the kernels step over blocks and entries in ints, up to 1,024 threads and a tile past the last
    if (d.max_blocks_per_seq > 0x40000000 || d.budget > 0x40000000) return false;
    if (static_cast<int64_t>(d.batch) * d.num_kv_heads > 0x7fffffffLL) return false;
    return d.flags == 0 || d.flags == KVD_FLAG_Q_BF16 || d.flags == KVD_FLAG_Q_F16;
}
}  // namespace

extern "C" size_t kvd_block_select_workspace_size(const kvd_block_select_desc* desc) {
    if (!select_ok(desc) || desc->max_blocks_per_seq <= desc->budget) return 0;
    return static_cast<size_t>(desc->batch) * desc->num_kv_heads * desc->max_blocks_per_seq * sizeof(uint32_t);
}

extern "C" cudaError_t kvd_block_select_launch(const kvd_block_select_desc* desc, const void* Q, const int8_t* bounds,
                                               const float* bound_scale, int32_t* sel_table, int32_t* sel_lens,
                                               void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    *launch_counter() = 0;
    if (!select_ok(desc) || !Q || !bounds || !bound_scale || !sel_table || !sel_lens || !desc->seq_lens ||
        !desc->block_table)
        return cudaErrorInvalidValue;
    const size_t want = kvd_block_select_workspace_size(desc);
    if (want > 0 && (!workspace || workspace_bytes < want || (reinterpret_cast<uintptr_t>(workspace) & 3) != 0))
        return cudaErrorInvalidValue;
    const SelectParams p{*desc, Q, bounds, bound_scale, sel_table, sel_lens, static_cast<uint32_t*>(workspace)};
    return launch_select(p, stream);
}
