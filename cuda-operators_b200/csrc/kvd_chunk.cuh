// kvd_chunk.cuh -- shared by the kernels of attention of packed new tokens over
// a paged cache (kvd_paged_prefill_launch): parameters, the plan of their work,
// the records of work that is split along the tokens, and the widening of codes.
#pragma once

#include <cstdint>

#include "kvd_common.cuh"

namespace kvd {

// Requests by their rows (new tokens times heads of a group) of a KV head: up to 8, few, many. Each class has a
// kernel of its own.
constexpr int kClasses = 3;
constexpr int kMany = 2;

// Work of a call, in the workspace: this, then for each class two arrays of B + 1 entries.
struct ChunkHead {
    uint64_t ready;           // the call's stamp once the plan is there
    int32_t units[kClasses];  // units: blocks of rows x KV heads x stretches of tokens
    int32_t span[kClasses];   // tokens of a stretch at most
    int32_t recs[kClasses];   // records of units whose tokens are split
    int32_t ticket;           // units of many rows that have been taken
    int32_t ended;            // CTAs of the last class's kernel that have ended
    int32_t pad[3];
};
static_assert(sizeof(ChunkHead) % 16 == 0, "alignment");

struct ChunkParams {
    const void* Q;
    const int8_t* K;
    const int8_t* V;
    const float* ks;
    const float* vs;
    void* out;
    const int32_t* seq_lens;
    const int32_t* starts;
    const int32_t* table;
    int B, Hq, Hkv, G, D, T, bs, NB, MB, causal;
    int64_t bt_stride;
    int64_t kv_sblk, kv_sh, kv_st, sc_sblk, sc_sh, q_st, q_sh, o_st, o_sh;
    float qscale;  // softmax_scale * log2(e)
    uint32_t flags;
    FastDiv by_bs, by_g;
    int vec_q, vec_out;  // rows on 16-byte boundaries
    // plan
    ChunkHead* head;
    int32_t* first[kClasses];   // [B + 1] units in front of request b's
    int32_t* rec[kClasses];     // [B + 1] records in front of request b's
    float* part_o[kClasses];    // records: [slot][unit_rows][D] sums of weighted values
    float2* part_ml[kClasses];  // and [slot][unit_rows] (reference in base 2, sum of weights)
    int unit_rows[kClasses];
    int ctas[kClasses];         // CTAs that run at once
    int32_t* arrived[kMany];    // [slot] units of the classes with few rows that have written their records
    int max_recs[kClasses];     // room for records
    float4* aside;              // [CTA][2][D / 4][128] sums that the kernel for many rows puts aside
    int aside_tiles;            // after how many tiles
    uint64_t stamp;             // of the call: no other has it
    int follows;                // the kernel before this one reads the same plan
    int last;                   // no kernel of a class comes after this one
    int tiny_most, few_most;    // rows up to which a request is of the first class, of the second
};

constexpr int kFewStep = 32;     // tokens of a step of the kernels for few rows
constexpr int kFewMinSpan = 256; // tokens that a split has at least
constexpr int kTileMinSpan = 512;
// What a unit costs beside its tokens, in tokens.
constexpr float kFewExtra = 512.f, kTileExtra = 400.f;
constexpr int kTile = 128;       // tokens of a tile of the kernel for many rows
// A product of 16 tokens on the tensor cores cuts the sum that it adds to off, towards zero: 32,768 tokens of values
// above zero, in one stretch of two terms, came out 1.07e-4 too small. So a warpgroup puts its sums aside, added with
// rounding, and starts again from zero after this many of its tiles, 64 products of a 32-bit output (1.5e-6 then),
// 512 of a 16-bit one. Powers of two.
constexpr int kAsideTiles = 4, kAsideTiles16 = 64;

// The kernels of the classes write nothing that the others read, so one need not wait until the one before it ends: it
// takes the SMs that the other leaves. What puts its reads behind the plan, and with it behind all that the plan has
// waited for, is the stamp that the plan releases and this acquires. A kernel that does not find the stamp waits for
// the one before it. No stamp is left over from a call before: calls have stamps of their own, and a captured one, which
// keeps its stamp, takes it back when its last class ends. Every kernel ends after the one before it, so whoever
// waits for the last waits for all.
__device__ __forceinline__ void class_begins(const ChunkParams& p) {
    if (p.follows) {
        __shared__ int s_ready;
        if (threadIdx.x == 0) {
            unsigned long long stamp;
            asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(stamp) : "l"(&p.head->ready) : "memory");
            s_ready = stamp == p.stamp;
        }
        __syncthreads();
        if (!s_ready) grid_dependency_wait();
    } else {
        grid_dependency_wait();
    }
    allow_dependents();
}
__device__ __forceinline__ void class_ends(const ChunkParams& p) {
    if (!p.follows) return;
    grid_dependency_wait();
    // (the last kernel's CTAs have all seen the stamp when each has counted itself, and earlier kernels have ended)
    if (p.last && threadIdx.x == 0 && atomicAdd(&p.head->ended, 1) == static_cast<int>(gridDim.x) - 1) p.head->ready = 0;
}

// Rows [t0, t0 + n) of request b and its tokens.
struct ChunkRows {
    int t0, n, len;
};

__device__ __forceinline__ ChunkRows chunk_rows(const ChunkParams& p, int b) {
    ChunkRows r;
    r.t0 = min(max(0, p.starts[b]), p.T);
    r.n = min(max(r.t0, p.starts[b + 1]), p.T) - r.t0;
    r.len = static_cast<int>(min(static_cast<int64_t>(max(0, p.seq_lens[b])), static_cast<int64_t>(p.MB) * p.bs));
    return r;
}

// Tokens that row i of a request sees: the first of them, this many.
__device__ __forceinline__ int chunk_sees(const ChunkParams& p, const ChunkRows& r, int i) {
    return p.causal ? max(0, min(r.len, r.len - r.n + i + 1)) : r.len;
}

__device__ __forceinline__ int chunk_class(const ChunkParams& p, int rows) {
    return rows <= p.tiny_most ? 0 : rows <= p.few_most ? 1 : kMany;
}

// Splits of a request's tokens, and the tokens of each (a multiple of `step`).
__device__ __forceinline__ int chunk_splits(int len, int span, int step, int& each) {
    const int n = max(1, (len + span - 1) / span);
    each = ((len + n - 1) / n + step - 1) / step * step;
    return max(1, (len + each - 1) / max(1, each));
}

// The last i in [0, n) with first[i] <= x, by a whole warp: 32 places a round.
__device__ __forceinline__ int warp_find(const int32_t* first, int n, int x) {
    const int lane = threadIdx.x & 31;
    int lo = 0;
    while (n > 1) {
        const int step = (n + 31) >> 5, at = lane * step;
        const unsigned ok = __ballot_sync(0xffffffffu, at < n && first[lo + min(at, n - 1)] <= x);
        const int k = ok ? 31 - __clz(ok) : 0;  // the places ascend
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// 2^k as a float, -126 <= k <= 127.
__device__ __forceinline__ float pow2i(int k) { return __int_as_float((k + 127) << 23); }

// Codes as fp16. A code c is the byte c + 128 once its sign bit is flipped; 0x6400 | byte is the fp16
// 1024 + byte, exactly, and 1152 from it leaves c. Even bytes of a word give one pair, odd ones the other.
__device__ __forceinline__ uint32_t half_pair(uint32_t bytes_0_2) {
    uint32_t x = (bytes_0_2 & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Two floats as a pair of fp16, and what the rounding left of them as another.
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack_half(a - f.x, b - f.y);
}

// Exponent k such that |x| 2^k < 2^top, for the largest |x| of a row or of value scales. Zero, infinities
// and NaN have none: k = 0. k stays where 2^k and 2^-k are normal.
__device__ __forceinline__ int fit_exponent(float most, int top) {
    const int e = static_cast<int>(__float_as_uint(most) >> 23);  // most >= 0
    if (most == 0.f || e == 255) return 0;
    return min(max(top - (e - 126), -126), 126);
}

// Four neighbouring dims of an output row.
__device__ __forceinline__ void store_out4(const ChunkParams& p, int64_t at, float4 x) {
    if (!p.vec_out) {
        store_out(p.out, at, x.x, p.flags);
        store_out(p.out, at + 1, x.y, p.flags);
        store_out(p.out, at + 2, x.z, p.flags);
        store_out(p.out, at + 3, x.w, p.flags);
    } else if (p.flags & KVD_FLAG_OUT_BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else if (p.flags & KVD_FLAG_OUT_F16) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(pack_half(x.x, x.y), pack_half(x.z, x.w));
    } else {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = x;
    }
}

// N rows from r0 on (of the unit's; row0: its first one of the request's) of a split unit, by a warp: the records
// slot, slot + 1, .. of its splits, weighed by their references.
template <int D, int N>
__device__ __forceinline__ void merge_records(const ChunkParams& p, const ChunkRows& R, const float* o, const float2* ml, int slot,
                                              int nsplit, int unit_rows, int hk, int row0, int r0, int rows, int lane) {
    constexpr int E = D / 32;  // neighbouring dims a lane
    float M[N], L[N] = {}, acc[N][E] = {};
    int64_t at[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        at[i] = static_cast<int64_t>(slot) * unit_rows + min(r0 + i, rows - 1 - row0);  // the last one again where there is none
        M[i] = -INFINITY;
        for (int s = lane; s < nsplit; s += 32) M[i] = fmaxf(M[i], __ldcg(&ml[at[i] + static_cast<int64_t>(s) * unit_rows]).x);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) M[i] = fmaxf(M[i], __shfl_xor_sync(0xffffffffu, M[i], x));
    }
#pragma unroll 4
    for (int s = 0; s < nsplit; ++s) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t rec = at[i] + static_cast<int64_t>(s) * unit_rows;
            const float2 v = __ldcg(&ml[rec]);
            float x[E];
            if constexpr (E == 4) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(o + rec * D) + lane);
                x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
            } else {
                const float2 y = __ldcg(reinterpret_cast<const float2*>(o + rec * D) + lane);
                x[0] = y.x; x[1] = y.y;
            }
            const float f = v.x == -INFINITY ? 0.f : exp2f(v.x - M[i]);
            L[i] = fmaf(v.y, f, L[i]);
#pragma unroll
            for (int d = 0; d < E; ++d)
                if (f != 0.f) acc[i][d] = fmaf(x[d], f, acc[i][d]);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = row0 + r0 + i;
        if (row >= rows) break;
        const int t = static_cast<int>(p.by_g.div(static_cast<uint32_t>(row))), g = row - t * p.G;
        const int64_t to = static_cast<int64_t>(R.t0 + t) * p.o_st + static_cast<int64_t>(hk * p.G + g) * p.o_sh + lane * E;
        const float inv = L[i] == 0.f ? 0.f : 1.f / L[i];  // no token in sight: 0; NaN stays
#pragma unroll
        for (int d = 0; d < E; ++d) store_out(p.out, to + d, acc[i][d] * inv, p.flags);
    }
}

cudaError_t launch_chunk_few(const ChunkParams& p, int cls, cudaStream_t st, int* launches);
int chunk_few_ctas(int D, int cls, bool q16);  // CTAs of an SM
cudaError_t launch_chunk_tile(const ChunkParams& p, cudaStream_t st, int* launches);

}  // namespace kvd
