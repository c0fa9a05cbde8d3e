// rows.cuh -- kernels on token rows: tokens sorted by expert and back (with
// the gradients), rows into 8 bits with a scale for each 128 columns, SwiGLU
// into 8-bit rows and its gradient.
//
// All of them read each input once and write each output once and compute
// little: memory bounds them from a few hundred rows on, launch latency below.
// A thread holds 8 neighbouring columns (one 16-byte load of a 16-bit type,
// one 8-byte store of codes); 16 neighbouring threads hold a block of 128, so
// a block's largest magnitude is four shuffles inside a half warp and no value
// is read twice.  Everything between load and store is in 32 bits.
//
// 8-bit rows: for each block of 128 columns scale = max(amax / 448, 2^-126),
// code = e4m3(v / scale), round to nearest even.  448 is e4m3's largest
// number, so no code saturates.  The lower bound keeps the scale of a block of
// zeros (or of denormals) a normal number.  A NaN or an infinity in a block
// makes its scale NaN: the whole block stands for NaN, and its neighbours are
// untouched.
//
// Both divisions are a product with the rounded reciprocal and one correction
// by the exact remainder (Markstein's theorem: rounded like the division), 3
// operations for two values in place of some 20 with branches.
// (Blocks of scales below 2^-90, where the remainder is not exact, are divided.)
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace qrm {

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;
constexpr float kFp8MinScale = 1.17549435e-38f;   // 2^-126

// ------------------------------------------------------------ eight columns

struct Vec8 {
    float v[8];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Eight columns as they are stored: what a thread keeps of a load in flight.
template <typename T>
struct Raw8 {
    uint32_t w[2 * sizeof(T)];
};

// the n <= 8 columns at p (the others are 0); `wide`: p is on a 16-byte boundary
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* __restrict__ p, int n, bool wide) {
    Raw8<T> r;
    if (wide && n == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p) + i);
            r.w[4 * i] = a.x; r.w[4 * i + 1] = a.y; r.w[4 * i + 2] = a.z; r.w[4 * i + 3] = a.w;
        }
    } else {
        T h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = i < n ? p[i] : from_f32<T>(0.f);
        memcpy(r.w, h, sizeof h);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ float column(const Raw8<T>& r, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[i]);
    T h[2];
    memcpy(h, &r.w[i / 2], 4);
    return to_f32(h[i & 1]);
}
template <typename T>
__device__ __forceinline__ Vec8 load8(const T* __restrict__ p, int n, bool wide) {
    const Raw8<T> raw = load_raw8(p, n, wide);
    Vec8 r;
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = column(raw, i);
    return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, const Vec8& r, int n, bool wide) {
    if (wide && n == 8) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p)[0] = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const T h[2] = {from_f32<T>(r.v[2 * i]), from_f32<T>(r.v[2 * i + 1])};
                memcpy(&w[i], h, 4);
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = from_f32<T>(r.v[i]);
    }
}

// ------------------------------------------------------------ 8-bit blocks

// largest magnitude; a NaN stays one
__device__ __forceinline__ float amax3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// two f32 in one operation
typedef uint64_t Pair;
__device__ __forceinline__ Pair pair(float x, float y) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpair(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// scale = max(amax / 448, 2^-126): the quotient by reciprocal and remainder, as below
__device__ __forceinline__ float block_scale(float amax) {
    constexpr float r = 1.f / kFp8Max;
    const float q = amax * r;
    return max_nan(fmaf(-fmaf(q, kFp8Max, -amax), r, q), kFp8MinScale);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// How the values of one block are turned into codes: the scale and, for pairs,
// the scale and minus its rounded reciprocal.
struct Quant {
    Pair s, nr;
};
__device__ __forceinline__ Quant quant(float scale) {
    const float nr = -1.f / scale;
    return {pair(scale, scale), pair(nr, nr)};
}
// Codes of the pair whose negated values nv holds: v / s rounded, from
// q = v r, e = q s - v (exact) and q - e r.  With the signs placed so, a zero
// keeps its sign.
__device__ __forceinline__ uint32_t codes2(Pair nv, const Quant& z) {
    const Pair q = mul2(nv, z.nr);
    const float2 f = unpair(fma2(fma2(q, z.s, nv), z.nr, q));
    return e4m3x2(f.x, f.y);
}
struct Pairs8 {   // eight values, negated where they are to become codes
    Pair p[4];
};
__device__ __forceinline__ uint2 codes8(const Pairs8& v, const Quant& z) {
    return make_uint2(codes2(v.p[0], z) | (codes2(v.p[1], z) << 16), codes2(v.p[2], z) | (codes2(v.p[3], z) << 16));
}

// The remainder of a value below 2^-103 is rounded to a denormal, and a tie may
// then go to the wrong side.  Such values have codes (the smallest tie is 2^-10
// of the scale) only where the scale is below 2^-92: those blocks are divided.
// The check costs 0.3 us of 64 in gather_rows_fp8, 0.4 of 145 in the combine's
// gradient and 0.4 of 67 in SwiGLU's, at the sizes stated there.
constexpr float kFp8Tiny = 8.077935669463161e-28f;   // 2^-90
static __device__ __noinline__ uint2 codes8_divided(const Pairs8 v, float scale) {
    uint32_t w[4];
#pragma unroll 1
    for (int i = 0; i < 4; i++) {
        const float2 f = unpair(v.p[i]);
        w[i] = e4m3x2(f.x / -scale, f.y / -scale);
    }
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// The largest magnitude among eight values, then in the block of 128 that a
// half warp holds (8 columns a thread), in each of its threads.  All 32 lanes
// take part.
__device__ __forceinline__ float amax8(const Pairs8& v) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpair(v.p[i]);
        m = amax3(m, f.x, f.y);
    }
    return m;
}
__device__ __forceinline__ float half_warp_max(float m) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Eight stored columns, negated, as f32 (the sign bits are turned over where
// two 16-bit values still share a word)
template <typename T>
__device__ __forceinline__ Pairs8 negated(const Raw8<T>& r) {
    Pairs8 v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            v.p[i] = pair(-__uint_as_float(r.w[2 * i]), -__uint_as_float(r.w[2 * i + 1]));
        } else {
            const uint32_t w = r.w[i] ^ 0x80008000u;
            T h[2];
            memcpy(h, &w, 4);
            v.p[i] = pair(to_f32(h[0]), to_f32(h[1]));
        }
    }
    return v;
}
template <typename T>
__device__ __forceinline__ Pairs8 values8(const Raw8<T>& r) {
    Pairs8 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v.p[i] = pair(column(r, 2 * i), column(r, 2 * i + 1));
    return v;
}

__device__ __forceinline__ void store_codes8(uint8_t* __restrict__ p, uint2 c, int n, bool wide) {
    if (wide && n == 8) {
        *reinterpret_cast<uint2*>(p) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
}

// columns that a thread at column c holds of `cols`, at most `most`
__device__ __forceinline__ int columns_at(int c, int cols, int most = 8) { return min(max(cols - c, 0), most); }

// ------------------------------------------------------------ tokens sorted by expert
// A stable counting sort of the n = T k assignments by expert in one launch:
// one CTA, or a cluster of 8 for more than 4096 assignments.  Each warp owns a
// run of assignments and counts them by expert in its own row of shared memory
// (the lowest lane of those with one expert adds), the rows and then the CTAs'
// totals are summed up in order, and the same walk gives each assignment its
// place.  No atomics: the order inside an expert is the assignments' own.
// The lanes with one expert are found by a vote for each bit of its number.
// Latencies bound it (8 SMs, a few passes over shared memory, two cluster
// barriers): 10.5 to 12 us at 32768 assignments to 256 experts, 14.6 with one
// load in flight instead of four; 4 us at 8 assignments.
constexpr int kSortMaxExperts = 1024;
constexpr int kSortCluster = 8;
constexpr int kSortOwnSmem = 32 * sizeof(int32_t);   // bytes beside the dynamic ones: a sum of each warp

// lanes whose e is this lane's; bits: of the largest e and of -1
__device__ __forceinline__ uint32_t lanes_with(int e, int bits) {
    uint32_t same = 0xffffffffu;
#pragma unroll 4
    for (int b = 0; b < bits; b++) {
        const bool one = e >> b & 1;
        const uint32_t v = __ballot_sync(0xffffffffu, one);
        same &= one ? v : ~v;
    }
    return same;
}

template <int C>   // CTAs
__global__ void __launch_bounds__(1024)
sort_tokens_kernel(const int32_t* __restrict__ idx, long long n, int first, int E, int bits, int32_t* __restrict__ perm,
                   int32_t* __restrict__ pos, int32_t* __restrict__ offsets) {
    pdl_start();
    extern __shared__ int32_t sort_sm[];
    const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int32_t* total = sort_sm;            // [E] this CTA's count of each expert
    int32_t* start = sort_sm + E;        // [E] place of this CTA's first assignment of each expert
    int32_t* count = sort_sm + 2 * E;    // [W][E] each warp's count, then its running place
    __shared__ int32_t warp_sum[kSortOwnSmem / sizeof(int32_t)];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = C > 1 ? (int)cluster.block_rank() : 0;

    for (int i = threadIdx.x; i < W * E; i += blockDim.x) count[i] = 0;
    const long long per = ((n + (long long)C * W - 1) / ((long long)C * W) + 31) & ~31ll;
    const long long a0 = ((long long)rank * W + warp) * per, a1 = a0 + per < n ? a0 + per : n;
    int32_t* mine = count + warp * E;
    __syncthreads();
    auto expert = [&](long long i) {   // -1: none of these
        const uint32_t e = i < a1 ? (uint32_t)idx[i] - (uint32_t)first : ~0u;
        return e < (uint32_t)E ? (int)e : -1;
    };
    for (long long a = a0; a < a1; a += 128) {
        int e[4];   // loads in flight together
#pragma unroll
        for (int u = 0; u < 4; u++) e[u] = expert(a + 32 * u + lane);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (a + 32 * u >= a1) break;
            const uint32_t same = lanes_with(e[u], bits);
            if (e[u] >= 0 && lane == __ffs(same) - 1) mine[e[u]] += __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int32_t sum = 0;
        for (int w0 = 0; w0 < W; w0 += 8) {   // W is a multiple of 8
            int32_t c[8];
#pragma unroll
            for (int w = 0; w < 8; w++) c[w] = count[(w0 + w) * E + e];
#pragma unroll
            for (int w = 0; w < 8; w++) {
                count[(w0 + w) * E + e] = sum;
                sum += c[w];
            }
        }
        total[e] = sum;
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    // places: experts in order, inside an expert the CTAs in order
    int32_t before = 0;   // assignments of the experts already passed
    for (int e0 = 0; e0 < E; e0 += blockDim.x) {
        const int e = e0 + threadIdx.x;
        int32_t sum = 0, lower = 0;
        if (e < E) {
            int32_t c[C];
#pragma unroll
            for (int r = 0; r < C; r++) c[r] = C > 1 ? cluster.map_shared_rank(total, r)[e] : total[e];
#pragma unroll
            for (int r = 0; r < C; r++) {
                if (r < rank) lower += c[r];
                sum += c[r];
            }
        }
        int32_t scan = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        int32_t v = lane < W ? warp_sum[lane] : 0, lane_sum = v;   // every warp sums the warps up for itself
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        const int32_t at = before + scan - sum + __shfl_sync(0xffffffffu, v - lane_sum, warp);
        if (e < E) {
            start[e] = at + lower;
            if (rank == 0) offsets[e] = at;
        }
        before += __shfl_sync(0xffffffffu, v, 31);
        __syncthreads();
    }
    if (rank == 0 && threadIdx.x == 0) offsets[E] = before;
    if (C > 1) cluster.barrier_arrive();   // this CTA has read the others' totals
    for (long long a = a0; a < a1; a += 128) {
        int e[4];
#pragma unroll
        for (int u = 0; u < 4; u++) e[u] = expert(a + 32 * u + lane);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (a + 32 * u >= a1) break;
            const long long i = a + 32 * u + lane;
            const uint32_t same = lanes_with(e[u], bits);
            const int32_t at = e[u] >= 0 ? start[e[u]] + mine[e[u]] + __popc(same & ((1u << lane) - 1u)) : -1;
            __syncwarp();
            if (e[u] >= 0 && lane == __ffs(same) - 1) mine[e[u]] += __popc(same);
            __syncwarp();
            if (i < a1) {
                pos[i] = at;
                if (at >= 0) perm[at] = (int32_t)i;
            }
        }
    }
    for (long long i = before + (long long)rank * blockDim.x + threadIdx.x; i < n; i += (long long)C * blockDim.x)
        perm[i] = -1;
    if (C > 1) cluster.barrier_wait();   // and they this one's
}

// ------------------------------------------------------------ rows out and back
// blockIdx.x is the token or row, blockIdx.y the piece of its columns that the
// CTA's threads hold.  Positions are compared unsigned, so -1 is out too.

// rows[pos[t, j]] = x[t] for every slot j whose row is in [0, n_rows)
template <typename T>
__global__ void __launch_bounds__(256)
gather_rows_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ pos, int k, int d, uint32_t n_rows,
                   T* __restrict__ rows, long long ld_rows, bool wide) {
    pdl_start();
    const int t = blockIdx.x, c = (blockIdx.y * blockDim.x + threadIdx.x) * 8, n = columns_at(c, d);
    if (!n) return;
    pos += (size_t)t * k;
    x += t * ld_x + c;
    if (wide && n == 8) {   // the bits as they are
        const Raw8<T> v = load_raw8(x, 8, true);
#pragma unroll 4
        for (int j = 0; j < k; j++) {
            const uint32_t p = pos[j];
            if (p >= n_rows) continue;
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++)
                reinterpret_cast<uint4*>(rows + p * ld_rows + c)[i] = make_uint4(v.w[4 * i], v.w[4 * i + 1], v.w[4 * i + 2], v.w[4 * i + 3]);
        }
    } else {
        for (int j = 0; j < k; j++) {
            const uint32_t p = pos[j];
            if (p >= n_rows) continue;
            for (int i = 0; i < n; i++) rows[p * ld_rows + c + i] = x[i];
        }
    }
}

// 16 columns in 8 bits: their codes, given the 8 threads' block
struct Codes16 {
    uint2 lo, hi;
    float scale;
};
template <typename T>
__device__ __forceinline__ Codes16 quantize16(const T* __restrict__ x, int n, bool wide) {
    const Pairs8 a = negated(load_raw8(x, min(n, 8), wide)), b = negated(load_raw8(x + 8, max(n - 8, 0), wide));
    float m = amax3(amax8(a), amax8(b), 0.f);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    Codes16 r;
    r.scale = block_scale(m);
    if (r.scale < kFp8Tiny) {
        r.lo = codes8_divided(a, r.scale);
        r.hi = codes8_divided(b, r.scale);
    } else {
        const Quant z = quant(r.scale);
        r.lo = codes8(a, z);
        r.hi = codes8(b, z);
    }
    return r;
}
__device__ __forceinline__ void store_codes16(uint8_t* __restrict__ p, const Codes16& q, int n, bool wide) {
    if (wide && n == 16) {
        *reinterpret_cast<uint4*>(p) = make_uint4(q.lo.x, q.lo.y, q.hi.x, q.hi.y);
    } else {
        store_codes8(p, q.lo, min(n, 8), false);
        store_codes8(p + 8, q.hi, n - 8, false);
    }
}

// the same into 8 bits: a token's row is quantised once for all its slots.  A
// thread holds 16 columns: the slots' addresses and checks were most of what
// it did with 8.  Memory bounds it: 4096 tokens x 8 slots of 7168 bf16 columns
// in 51 us, 5.8 TB/s (69 us with 8 columns and positions in 64 bits).
template <typename T>
__global__ void __launch_bounds__(256)
gather_rows_fp8_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ pos, int k, int d,
                       uint32_t n_rows, uint8_t* __restrict__ codes, long long ld_c, float* __restrict__ scales,
                       long long ld_s, bool wide_x, bool wide_c) {
    pdl_start();
    const int t = blockIdx.x, c = (blockIdx.y * blockDim.x + threadIdx.x) * 16, n = columns_at(c, d, 16);
    pos += (size_t)t * k;
    const Codes16 q = quantize16(x + t * ld_x + c, n, wide_x);
    if (!n) return;
    const bool lead = (threadIdx.x & 7) == 0;
#pragma unroll 4
    for (int j = 0; j < k; j++) {
        const uint32_t p = pos[j];
        if (p >= n_rows) continue;
        store_codes16(codes + p * ld_c + c, q, n, wide_c);
        if (lead) scales[p * ld_s + c / kFp8Block] = q.scale;
    }
}

// out[t] = add[t] + sum_j w[t, j] rows[pos[t, j]], in slot order; w NULL: 1.
// The CTAs walk the tokens; a token's first positions and weights come while
// the one before it is summed up (a lane holds a slot's), so one wait for
// memory a token is left.  2048 tokens x 6 slots of 4096 bf16 columns on the
// residual stream: 24.9 us, 5.4 TB/s (55 us with one CTA a token and four
// widened rows in registers).
template <typename T>
__global__ void __launch_bounds__(256, 4)
combine_rows_kernel(const T* __restrict__ rows, long long ld_rows, uint32_t n_rows, const int32_t* __restrict__ pos,
                    const float* __restrict__ w, uint32_t tokens, int k, int d, const T* __restrict__ add, long long ld_add,
                    T* __restrict__ out, long long ld_out, bool wide) {
    pdl_start();
    constexpr int S = sizeof(T) == 4 ? 4 : 8;   // rows whose loads are in flight: 32 registers
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8, n = columns_at(c, d), lane = threadIdx.x & 31;
    uint32_t t = blockIdx.x;   // (unsigned: a step past the last of 2^31 - 1 tokens stays a number past it)
    uint32_t p_next = ~0u;
    float w_next = 1.f;
    auto ahead = [&](uint32_t at) {   // slots lane < min(k, S) of token `at`
        if (at < tokens && lane < S && lane < k) {
            p_next = pos[(size_t)at * k + lane];
            if (w) w_next = w[(size_t)at * k + lane];
        }
    };
    ahead(t);
    for (; t < tokens; t += gridDim.x) {
        Pairs8 acc;
#pragma unroll
        for (int i = 0; i < 4; i++) acc.p[i] = 0;
        Raw8<T> first;
        if (add) first = load_raw8(add + t * ld_add + c, n, wide);
        for (int j0 = 0; j0 < k; j0 += S) {
            uint32_t p_lane = p_next;
            float w_lane = w_next;
            if (j0) {
                const int j = j0 + lane;
                p_lane = lane < S && j < k ? (uint32_t)pos[(size_t)t * k + j] : ~0u;
                w_lane = w && lane < S && j < k ? w[(size_t)t * k + j] : 1.f;
            }
            Raw8<T> r[S];
            uint32_t held = 0;
#pragma unroll
            for (int j = 0; j < S; j++) {
                const uint32_t p = __shfl_sync(0xffffffffu, p_lane, j);
                if (j0 + j >= k || p >= n_rows) continue;
                held |= 1u << j;
                r[j] = load_raw8(rows + p * ld_rows + c, n, wide);
            }
            if (j0 == 0) {
                ahead(t + gridDim.x);
                if (add) acc = values8(first);
            }
#pragma unroll
            for (int j = 0; j < S; j++) {
                const float wj = __shfl_sync(0xffffffffu, w_lane, j);
                if (held >> j & 1) {
                    const Pair wp = pair(wj, wj);
                    const Pairs8 v = values8(r[j]);
#pragma unroll
                    for (int i = 0; i < 4; i++) acc.p[i] = fma2(wp, v.p[i], acc.p[i]);
                }
            }
        }
        Vec8 o;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = unpair(acc.p[i]);
            o.v[2 * i] = f.x;
            o.v[2 * i + 1] = f.y;
        }
        store8(out + t * ld_out + c, o, n, wide);
    }
}

// The gradient of combine_rows: drows[pos[t, j]] = w[t, j] dout[t] (T or 8
// bits) and dw[t, j] = <dout[t], rows[pos[t, j]]>.  One CTA per token, up to
// eight slots at a time, one or more of the eight warps to a slot, so a slot's
// sum stays in its warps and a thread has few registers (which keeps enough
// loads in flight).  dout goes through shared memory, 8192 columns at a time.
// Rounding does not change an order, so the largest magnitude of w dout is the
// rounded product of |w| and dout's: it is looked for once for all slots, and
// each (slot, block)'s scale and reciprocal are computed by one thread.
// 4096 tokens x 8 slots of 7168 bf16 columns into 8 bits: 145 us, 5.3 TB/s
// (594 us with all slots in each thread, a maximum and divisions for each).
constexpr int kGradCols = 8192;

// The codes of one slot's blocks with a tiny scale once more, by division, over
// what the same threads have written (a choice for each eight columns where they
// are written cost 8 us).
static __device__ __noinline__ void divide_tiny(const float4* g, const float2* sc, float minus_w, int cols, int c, int step,
                                         uint8_t* codes, bool wide) {
    const Pair wp = pair(minus_w, minus_w);
#pragma unroll 1
    for (; c < cols; c += step) {
        const float s = sc[c / kFp8Block].x;
        if (!(s < kFp8Tiny)) continue;
        Pairs8 v;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float4 x = g[c / 4 + i];
            v.p[2 * i] = mul2(wp, pair(x.x, x.y));
            v.p[2 * i + 1] = mul2(wp, pair(x.z, x.w));
        }
        store_codes8(codes + c, codes8_divided(v, s), columns_at(c, cols), wide);
    }
}

// FAST: every row of every array starts on its widest access, d is a multiple of 8
template <typename T, bool FP8, bool FAST>
__global__ void __launch_bounds__(256)
combine_grad_kernel(const T* __restrict__ dout, long long ld_dout, const T* __restrict__ rows, long long ld_rows,
                    uint32_t n_rows, const int32_t* __restrict__ pos, const float* __restrict__ w, int k, int d,
                    T* __restrict__ drows, uint8_t* __restrict__ codes, long long ld_d, float* __restrict__ scales,
                    long long ld_s, float* __restrict__ dw, bool wide, bool wide_d) {
    pdl_start();
    constexpr int S = 8, NB = kGradCols / kFp8Block;
    constexpr int U = sizeof(T) == 4 ? 2 : 4;   // row loads in flight
    extern __shared__ float4 g_sm[];            // min(d, kGradCols) columns of dout, in whole blocks
    __shared__ float amax[NB];
    __shared__ float2 sc[S][NB];                // scale, minus its reciprocal
    __shared__ float part[S];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x;
    pos += (size_t)t * k;
    if (w) w += (size_t)t * k;
    dout += t * ld_dout;
    for (int j0 = 0; j0 < k; j0 += S) {
        const int slots = min(S, k - j0), each = S / slots;   // warps to a slot
        const int slot = warp / each, mine = warp - slot * each;
        const bool busy = slot < slots;
        const uint32_t p = busy ? (uint32_t)pos[j0 + slot] : ~0u;
        const bool held = p < n_rows;
        const float wn = !busy ? 0.f : w ? -w[j0 + slot] : -1.f;   // minus the weight
        Pair dot = 0;
        for (int base = 0; base < d; base += kGradCols) {
            const int cols = min(kGradCols, d - base), blocks = (cols + kFp8Block - 1) / kFp8Block;
            for (int c = threadIdx.x * 8; c < blocks * kFp8Block; c += 256 * 8) {   // whole half warps
                const Pairs8 g = values8(load_raw8(dout + base + c, columns_at(c, cols), wide));
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float2 x = unpair(g.p[2 * i]), y = unpair(g.p[2 * i + 1]);
                    g_sm[c / 4 + i] = make_float4(x.x, x.y, y.x, y.y);
                }
                if constexpr (FP8) {
                    float m = amax8(g);   // a half warp's columns are one block: its threads stay together
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffu << (lane & 16), m, o));
                    if ((lane & 15) == 0) amax[c / kFp8Block] = m;
                }
            }
            __syncthreads();
            if constexpr (FP8) {
                for (int i = threadIdx.x; i < slots * blocks; i += 256) {
                    const int j = i / blocks, b = i - j * blocks;
                    const float s = block_scale(__fmul_rn(w ? fabsf(w[j0 + j]) : 1.f, amax[b]));
                    sc[j][b] = make_float2(s, -1.f / s);
                    const uint32_t q = pos[j0 + j];
                    if (q < n_rows) scales[q * ld_s + base / kFp8Block + b] = s;
                }
                __syncthreads();
            }
            if (held) {
                const Pair wp = pair(wn, wn);
                float least = 1.f;   // of the scales that this thread meets, if below
                const T* from = rows + p * ld_rows + base;
                for (int c0 = (mine * 32 + lane) * 8; c0 < cols; c0 += each * 256 * U) {
                    Raw8<T> r[U];
                    if (dw)
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            const int c = c0 + u * each * 256;
                            if (!FAST) r[u] = load_raw8(from + c, columns_at(c, cols), wide);
                            else if (c < cols) r[u] = load_raw8(from + c, 8, true);
                        }
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int c = c0 + u * each * 256, n = FAST ? 8 : columns_at(c, cols);
                        if (c >= cols) break;
                        Pairs8 g;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const float4 x = g_sm[c / 4 + i];
                            g.p[2 * i] = pair(x.x, x.y);
                            g.p[2 * i + 1] = pair(x.z, x.w);
                        }
                        Pairs8 v;   // minus w dout
#pragma unroll
                        for (int i = 0; i < 4; i++) v.p[i] = mul2(wp, g.p[i]);
                        if constexpr (FP8) {
                            const float2 s = sc[slot][c / kFp8Block];
                            least = fminf(least, s.x);
                            store_codes8(codes + p * ld_d + base + c, codes8(v, Quant{pair(s.x, s.x), pair(s.y, s.y)}), n, FAST || wide_d);
                        } else {
                            Vec8 o;
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float2 f = unpair(v.p[i]);
                                o.v[2 * i] = -f.x;
                                o.v[2 * i + 1] = -f.y;
                            }
                            store8(drows + p * ld_d + base + c, o, n, FAST || wide_d);
                        }
                        if (dw) {
                            const Pairs8 x = values8(r[u]);
#pragma unroll
                            for (int i = 0; i < 4; i++) dot = fma2(g.p[i], x.p[i], dot);
                        }
                    }
                }
                if (FP8 && least < kFp8Tiny)
                    divide_tiny(g_sm, sc[slot], wn, cols, (mine * 32 + lane) * 8, each * 256, codes + p * ld_d + base, FAST || wide_d);
            }
            __syncthreads();   // before the next columns, or slots
        }
        if (dw) {
            const float2 f = unpair(dot);
            float sum = f.x + f.y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) part[warp] = sum;
            __syncthreads();
            if (threadIdx.x < slots) {
                float v = 0.f;
                for (int i = 0; i < each; i++) v += part[threadIdx.x * each + i];
                dw[(size_t)t * k + j0 + threadIdx.x] = v;   // 0 for a slot without a row
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------ rows into 8 bits
// (n_dev: how many of the rows there are, on the device)

template <typename T>
__global__ void __launch_bounds__(256)
quantize_fp8_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ n_dev, int cols,
                    uint8_t* __restrict__ codes, long long ld_c, float* __restrict__ scales, long long ld_s, bool wide_x,
                    bool wide_c) {
    pdl_start();
    const int t = blockIdx.x, c = (blockIdx.y * blockDim.x + threadIdx.x) * 16, n = columns_at(c, cols, 16);
    if (n_dev && t >= *n_dev) return;
    const Codes16 q = quantize16(x + t * ld_x + c, n, wide_x);
    if (!n) return;
    store_codes16(codes + t * ld_c + c, q, n, wide_c);
    if ((threadIdx.x & 7) == 0) scales[t * ld_s + c / kFp8Block] = q.scale;
}

// One CTA of 256 threads per 128 x 128 block of a weight matrix (rows x cols,
// dense): thread i holds 8 columns of every 16th row.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_fp8_weights_kernel(const T* __restrict__ w, int rows, int cols, uint8_t* __restrict__ codes,
                            float* __restrict__ scales, bool wide) {
    pdl_start();
    __shared__ float top[8];
    const int r0 = blockIdx.y * kFp8Block, c = blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8;
    const long long base = (long long)blockIdx.z * rows * cols;
    const int n = columns_at(c, cols);
    Pairs8 v[8];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = r0 + (threadIdx.x >> 4) + 16 * i;
        v[i] = negated(load_raw8(w + base + (long long)r * cols + c, r < rows ? n : 0, wide));
        m = max_nan(m, amax8(v[i]));
    }
    m = half_warp_max(m);
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16));
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) m = max_nan(m, top[i]);
    const float s = block_scale(m);
    const Quant z = quant(s);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r < rows && n)
            store_codes8(codes + base + (long long)r * cols + c, s < kFp8Tiny ? codes8_divided(v[i], s) : codes8(v[i], z), n, wide);
    }
    if (threadIdx.x == 0)
        scales[((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

// ------------------------------------------------------------ SwiGLU
// gu [rows][2f]: the gate's f columns, then the up projection's.  With
// limit L > 0 the gate is cut off above L and up to [-L, L] first.
//   h = g sigma(g) u
//   dg = dh u (sigma(g) + g sigma(g) (1 - sigma(g))), 0 where the gate was cut off
//   du = dh g sigma(g), 0 where up was cut off
// Two columns at a time.  sigma(g) = num / (1 + e) with e = exp(-|g|), which
// never overflows, and num = 1 or e by g's sign.  e is 2^x for x = -|g| log2 e
// with the rounding of that product made good (x + lo is exact to 2^-45 or so),
// so only the two approximate instructions' own errors remain (2 ulp and 1 ulp).
// |g| is cut off at 128 there, where e is 0 in f32 already: from 2^128 / log2 e
// on x would be infinite, and the good made of it not a number.
struct Swiglu2 {
    Pair g, u, sig;   // after the cut-offs
};
constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = (float)(1.4426950408889634074 - (double)kLog2e);
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kGateMost = 128.f;
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool LIMIT>
__device__ __forceinline__ Swiglu2 swiglu2(float2 gate, float2 up, float limit) {
    if (LIMIT) {   // a NaN stays one
        gate = make_float2(min_nan(gate.x, limit), min_nan(gate.y, limit));
        up = make_float2(max_nan(min_nan(up.x, limit), -limit), max_nan(min_nan(up.y, limit), -limit));
    }
    const Pair a = pair(min_nan(fabsf(gate.x), kGateMost), min_nan(fabsf(gate.y), kGateMost)), l2e = pair(-kLog2e, -kLog2e);
    const Pair x = mul2(a, l2e);
    const float2 xf = unpair(x);
    const Pair lo = fma2(a, pair(-kLog2eLow, -kLog2eLow), fma2(a, l2e, pair(-xf.x, -xf.y)));
    const Pair e0 = pair(exp2_approx(xf.x), exp2_approx(xf.y));
    const float2 e = unpair(fma2(mul2(e0, lo), pair(kLn2, kLn2), e0));
    const float2 r = make_float2(reciprocal_approx(1.f + e.x), reciprocal_approx(1.f + e.y));
    Swiglu2 s;
    s.g = pair(gate.x, gate.y);
    s.u = pair(up.x, up.y);
    s.sig = mul2(pair(gate.x < 0.f ? e.x : 1.f, gate.y < 0.f ? e.y : 1.f), pair(r.x, r.y));
    return s;
}
__device__ __forceinline__ Pair negative(Pair p) { return p ^ 0x8000000080000000ull; }

// The CTAs walk the rows; a row's loads are on their way while the one before
// it is computed.  The gradient takes 63 us for 16384 rows of 2048 bf16 columns
// with a limit, 4.3 TB/s (67 us under sustained load), the forward 43 us: issue slots (74 % busy) bound it, some 50 operations
// a value; two rows ahead, or more CTAs of fewer registers, change nothing.
template <typename T, bool LIMIT>
__global__ void __launch_bounds__(256)
swiglu_fp8_kernel(const T* __restrict__ gu, long long ld, int rows, const int32_t* __restrict__ n_dev, int f, float limit,
                  uint8_t* __restrict__ codes, long long ld_c, float* __restrict__ scales, long long ld_s, bool wide,
                  bool wide_c) {
    pdl_start();
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8, n = columns_at(c, f);
    if (n_dev) rows = max(min(rows, *n_dev), 0);
    const uint32_t end = rows;
    uint32_t t = blockIdx.x;   // (unsigned, as in combine_rows_kernel)
    if (t >= end) return;
    gu += c;
    Raw8<T> g = load_raw8(gu + t * ld, n, wide), u = load_raw8(gu + t * ld + f, n, wide);   // absent columns are 0, and h there
    for (;;) {
        const uint32_t next = t + gridDim.x;
        Raw8<T> g1 = g, u1 = u;
        if (next < end) {
            g1 = load_raw8(gu + next * ld, n, wide);
            u1 = load_raw8(gu + next * ld + f, n, wide);
        }
        Pairs8 h;   // negated
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const Swiglu2 p = swiglu2<LIMIT>(make_float2(column(g, 2 * i), column(g, 2 * i + 1)),
                                             make_float2(column(u, 2 * i), column(u, 2 * i + 1)), limit);
            h.p[i] = mul2(mul2(p.g, p.sig), negative(p.u));
        }
        const float s = block_scale(half_warp_max(amax8(h)));
        if (n) {
            store_codes8(codes + t * ld_c + c, s < kFp8Tiny ? codes8_divided(h, s) : codes8(h, quant(s)), n, wide_c);
            if ((threadIdx.x & 15) == 0) scales[t * ld_s + c / kFp8Block] = s;
        }
        if (next >= end) return;
        t = next;
        g = g1;
        u = u1;
    }
}

// f is a multiple of 128 here, so no block of the 2f columns holds both halves
template <typename T, bool LIMIT>
__global__ void __launch_bounds__(256)
swiglu_fp8_grad_kernel(const T* __restrict__ gu, long long ld, const T* __restrict__ dh, long long ld_dh, int rows,
                       const int32_t* __restrict__ n_dev, int f, float limit, uint8_t* __restrict__ codes, long long ld_c,
                       float* __restrict__ scales, long long ld_s, bool wide, bool wide_c) {
    pdl_start();
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8, n = columns_at(c, f);
    if (n_dev) rows = max(min(rows, *n_dev), 0);
    const uint32_t end = rows;
    uint32_t t = blockIdx.x;   // (unsigned, as in combine_rows_kernel)
    if (t >= end) return;
    gu += c;
    dh += c;
    Raw8<T> g = load_raw8(gu + t * ld, n, wide), u = load_raw8(gu + t * ld + f, n, wide), d = load_raw8(dh + t * ld_dh, n, wide);
    for (;;) {
        const uint32_t next = t + gridDim.x;
        Raw8<T> g1 = g, u1 = u, d1 = d;
        if (next < end) {
            g1 = load_raw8(gu + next * ld, n, wide);
            u1 = load_raw8(gu + next * ld + f, n, wide);
            d1 = load_raw8(dh + next * ld_dh, n, wide);
        }
        Pairs8 dg, du;   // negated
        const Pair one = pair(1.f, 1.f), minus = pair(-1.f, -1.f);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 gate = make_float2(column(g, 2 * i), column(g, 2 * i + 1)), up = make_float2(column(u, 2 * i), column(u, 2 * i + 1));
            const Swiglu2 p = swiglu2<LIMIT>(gate, up, limit);
            const Pair nd = pair(-column(d, 2 * i), -column(d, 2 * i + 1));
            // u sigma (1 + g (1 - sigma)) and g sigma, times minus dh
            dg.p[i] = mul2(mul2(nd, p.u), mul2(p.sig, fma2(p.g, fma2(p.sig, minus, one), one)));
            du.p[i] = mul2(nd, mul2(p.g, p.sig));
            if (LIMIT) {   // nothing comes back through a cut-off
                float2 a = unpair(dg.p[i]), b = unpair(du.p[i]);
                a = make_float2(gate.x > limit ? 0.f : a.x, gate.y > limit ? 0.f : a.y);
                b = make_float2(fabsf(up.x) > limit ? 0.f : b.x, fabsf(up.y) > limit ? 0.f : b.y);
                dg.p[i] = pair(a.x, a.y);
                du.p[i] = pair(b.x, b.y);
            }
        }
        const float sg = block_scale(half_warp_max(amax8(dg))), su = block_scale(half_warp_max(amax8(du)));
        if (n) {
            uint2 cg, cu;
            if (fminf(sg, su) < kFp8Tiny) {
                cg = codes8_divided(dg, sg);
                cu = codes8_divided(du, su);
            } else {
                cg = codes8(dg, quant(sg));
                cu = codes8(du, quant(su));
            }
            store_codes8(codes + t * ld_c + c, cg, n, wide_c);
            store_codes8(codes + t * ld_c + f + c, cu, n, wide_c);
            if ((threadIdx.x & 15) == 0) {
                scales[t * ld_s + c / kFp8Block] = sg;
                scales[t * ld_s + (f + c) / kFp8Block] = su;
            }
        }
        if (next >= end) return;
        t = next;
        g = g1;
        u = u1;
        d = d1;
    }
}

}  // namespace qrm
