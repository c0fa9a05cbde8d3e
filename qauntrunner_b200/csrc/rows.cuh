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
// operations a value in place of some 10 with a branch.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// v / s given r = 1 / s, both rounded (in this order a zero keeps its sign)
__device__ __forceinline__ float divided(float v, float s, float r) {
    const float q = v * r;
    return fmaf(-fmaf(q, s, -v), r, q);
}
__device__ __forceinline__ float block_scale(float amax) {
    return max_nan(divided(amax, kFp8Max, 1.f / kFp8Max), kFp8MinScale);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// The largest magnitude of the block that this half warp's 16 threads hold (8
// columns each), in every one of them.  All 32 lanes take part.
__device__ __forceinline__ float half_warp_amax(const Vec8& r) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max_nan(m, fabsf(r.v[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
__device__ __forceinline__ float half_warp_scale(const Vec8& r) { return block_scale(half_warp_amax(r)); }

// r = 1 / scale
__device__ __forceinline__ uint2 codes8(const Vec8& v, float scale, float r) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = e4m3x2(divided(v.v[2 * i], scale, r), divided(v.v[2 * i + 1], scale, r));
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
__device__ __forceinline__ uint2 codes8(const Vec8& v, float scale) { return codes8(v, scale, 1.f / scale); }

__device__ __forceinline__ void store_codes8(uint8_t* __restrict__ p, uint2 c, int n, bool wide) {
    if (wide && n == 8) {
        *reinterpret_cast<uint2*>(p) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
}

// columns that a thread at column c holds of `cols`
__device__ __forceinline__ int columns_at(long long c, long long cols) {
    return c >= cols ? 0 : (int)(cols - c < 8 ? cols - c : 8);
}

// ------------------------------------------------------------ tokens sorted by expert
// A stable counting sort of the n = T k assignments by expert in one launch:
// one CTA, or a cluster of 8 for more than 4096 assignments.  Each warp owns a
// run of assignments and counts them by expert in its own row of shared memory
// (lanes with one expert found by match.any; the lowest of them adds), the
// rows and then the CTAs' totals are summed up in order, and the same walk
// gives each assignment its place.  No atomics: the order inside an expert is
// the assignments' own.
constexpr int kSortMaxExperts = 1024;
constexpr int kSortCluster = 8;

__global__ void __launch_bounds__(1024)
sort_tokens_kernel(const int32_t* __restrict__ idx, long long n, int first, int E, int32_t* __restrict__ perm,
                   int32_t* __restrict__ pos, int32_t* __restrict__ offsets) {
    extern __shared__ int32_t sort_sm[];
    const int W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int32_t* total = sort_sm;            // [E] this CTA's count of each expert
    int32_t* start = sort_sm + E;        // [E] place of this CTA's first assignment of each expert
    int32_t* count = sort_sm + 2 * E;    // [W][E] each warp's count, then its running place
    __shared__ int32_t warp_sum[32];
    __shared__ int32_t all;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();

    for (int i = threadIdx.x; i < W * E; i += blockDim.x) count[i] = 0;
    __syncthreads();
    const long long per = ((n + (long long)C * W - 1) / ((long long)C * W) + 31) & ~31ll;
    const long long a0 = ((long long)rank * W + warp) * per, a1 = a0 + per < n ? a0 + per : n;
    int32_t* mine = count + warp * E;
    for (long long a = a0; a < a1; a += 32) {
        const long long i = a + lane;
        int e = i < a1 ? idx[i] - first : -1;
        if (e < 0 || e >= E) e = -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int32_t sum = 0;
        for (int w = 0; w < W; w++) {
            const int32_t c = count[w * E + e];
            count[w * E + e] = sum;
            sum += c;
        }
        total[e] = sum;
    }
    cluster.sync();
    // places: experts in order, inside an expert the CTAs in order
    int32_t before = 0;   // assignments of the experts already passed
    for (int e0 = 0; e0 < E; e0 += blockDim.x) {
        const int e = e0 + threadIdx.x;
        int32_t sum = 0, lower = 0;
        if (e < E)
            for (int c = 0; c < C; c++) {
                const int32_t t = cluster.map_shared_rank(total, c)[e];
                if (c < rank) lower += t;
                sum += t;
            }
        int32_t scan = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        if (warp == 0) {
            int32_t v = lane < W ? warp_sum[lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (lane < W) warp_sum[lane] = v;
            if (lane == 31) all = v;
        }
        __syncthreads();
        const int32_t at = before + scan - sum + (warp ? warp_sum[warp - 1] : 0);
        if (e < E) {
            start[e] = at + lower;
            if (rank == 0) offsets[e] = at;
        }
        before += all;
        __syncthreads();
    }
    if (rank == 0 && threadIdx.x == 0) offsets[E] = before;
    cluster.sync();   // the totals have been read everywhere, the starts are written
    for (long long a = a0; a < a1; a += 32) {
        const long long i = a + lane;
        int e = i < a1 ? idx[i] - first : -1;
        if (e < 0 || e >= E) e = -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const int32_t at = e >= 0 ? start[e] + mine[e] + __popc(same & ((1u << lane) - 1u)) : -1;
        __syncwarp();
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
        if (i < a1) {
            pos[i] = at;
            if (at >= 0) perm[at] = (int32_t)i;
        }
    }
    for (long long i = before + (long long)rank * blockDim.x + threadIdx.x; i < n; i += (long long)C * blockDim.x)
        perm[i] = -1;
}

// ------------------------------------------------------------ rows out and back
// One unit of work = one token x the columns that a CTA's threads hold.

// rows[pos[t, j]] = x[t] for every slot j whose row is in [0, n_rows)
template <typename T>
__global__ void gather_rows_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ pos, long long T_,
                                   int k, long long d, int segments, long long n_rows, T* __restrict__ rows,
                                   long long ld_rows, bool wide) {
    for (long long u = blockIdx.x; u < T_ * segments; u += gridDim.x) {
        const long long t = u / segments;
        const long long c = ((u - t * segments) * blockDim.x + threadIdx.x) * 8;
        const int n = columns_at(c, d);
        if (!n) continue;
        if (wide && n == 8) {   // the bits as they are
            constexpr int W = sizeof(T) / 2;
            uint4 v[W];
#pragma unroll
            for (int i = 0; i < W; i++) v[i] = __ldg(reinterpret_cast<const uint4*>(x + t * ld_x + c) + i);
            for (int j = 0; j < k; j++) {
                const long long p = pos[t * k + j];
                if (p < 0 || p >= n_rows) continue;
#pragma unroll
                for (int i = 0; i < W; i++) reinterpret_cast<uint4*>(rows + p * ld_rows + c)[i] = v[i];
            }
        } else {
            for (int j = 0; j < k; j++) {
                const long long p = pos[t * k + j];
                if (p < 0 || p >= n_rows) continue;
                for (int i = 0; i < n; i++) rows[p * ld_rows + c + i] = x[t * ld_x + c + i];
            }
        }
    }
}

// the same into 8 bits: a token's row is quantised once for all its slots
template <typename T>
__global__ void gather_rows_fp8_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ pos,
                                       long long T_, int k, long long d, int segments, long long n_rows,
                                       uint8_t* __restrict__ codes, long long ld_c, float* __restrict__ scales,
                                       long long ld_s, bool wide_x, bool wide_c) {
    for (long long u = blockIdx.x; u < T_ * segments; u += gridDim.x) {
        const long long t = u / segments;
        const long long c = ((u - t * segments) * blockDim.x + threadIdx.x) * 8;
        const int n = columns_at(c, d);
        const Vec8 v = load8(x + t * ld_x + c, n, wide_x);
        const float s = half_warp_scale(v);
        if (!n) continue;
        const uint2 q = codes8(v, s);
        const bool lead = (threadIdx.x & 15) == 0;
        for (int j = 0; j < k; j++) {
            const long long p = pos[t * k + j];
            if (p < 0 || p >= n_rows) continue;
            store_codes8(codes + p * ld_c + c, q, n, wide_c);
            if (lead) scales[p * ld_s + c / kFp8Block] = s;
        }
    }
}

// out[t] = add[t] + sum_j w[t, j] rows[pos[t, j]], in slot order; w NULL: 1
template <typename T>
__global__ void combine_rows_kernel(const T* __restrict__ rows, long long ld_rows, long long n_rows,
                                    const int32_t* __restrict__ pos, const float* __restrict__ w, long long T_, int k,
                                    long long d, int segments, const T* __restrict__ add, long long ld_add,
                                    T* __restrict__ out, long long ld_out, bool wide) {
    constexpr int S = sizeof(T) == 4 ? 4 : 8;   // rows at a time: 32 registers
    for (long long u = blockIdx.x; u < T_ * segments; u += gridDim.x) {
        const long long t = u / segments;
        const long long c = ((u - t * segments) * blockDim.x + threadIdx.x) * 8;
        const int n = columns_at(c, d);
        if (!n) continue;
        Vec8 acc;
        if (add) acc = load8(add + t * ld_add + c, n, wide);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) acc.v[i] = 0.f;
        for (int j0 = 0; j0 < k; j0 += S) {   // their loads in flight together
            Raw8<T> r[S];
            float wj[S];
            uint32_t held = 0;
#pragma unroll
            for (int j = 0; j < S; j++) {
                if (j0 + j >= k) break;
                const long long p = pos[t * k + j0 + j];
                if (p < 0 || p >= n_rows) continue;
                held |= 1u << j;
                r[j] = load_raw8(rows + p * ld_rows + c, n, wide);
                wj[j] = w ? w[t * k + j0 + j] : 1.f;
            }
#pragma unroll
            for (int j = 0; j < S; j++)
                if (held >> j & 1)
#pragma unroll
                    for (int i = 0; i < 8; i++) acc.v[i] = fmaf(wj[j], column(r[j], i), acc.v[i]);
        }
        store8(out + t * ld_out + c, acc, n, wide);
    }
}

// The gradient of combine_rows: drows[pos[t, j]] = w[t, j] dout[t] (T or 8
// bits) and dw[t, j] = <dout[t], rows[pos[t, j]]>.  One CTA per token: dw
// needs the whole row.  Eight slots at a time, whose sums stay in registers.
// Rounding does not change an order, so the largest magnitude of w dout is the
// rounded product of |w| and dout's: it is looked for once for all slots, and
// the eight slots' scales and reciprocals are computed by eight lanes of the
// half warp, one each, and handed round.
template <typename T, bool FP8>
__global__ void __launch_bounds__(512, 2)
combine_grad_kernel(const T* __restrict__ dout, long long ld_dout, const T* __restrict__ rows,
                                    long long ld_rows, long long n_rows, const int32_t* __restrict__ pos,
                                    const float* __restrict__ w, long long T_, int k, long long d, T* __restrict__ drows,
                                    uint8_t* __restrict__ codes, long long ld_d, float* __restrict__ scales,
                                    long long ld_s, float* __restrict__ dw, bool wide, bool wide_d) {
    constexpr int S = 8, B = sizeof(T) == 4 ? 2 : 4;   // slots; rows' loads in flight
    __shared__ float part[S][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    for (long long t = blockIdx.x; t < T_; t += gridDim.x) {
        for (int j0 = 0; j0 < k; j0 += S) {
            float dot[S];
            int p[S];
            float wj[S];
#pragma unroll
            for (int j = 0; j < S; j++) {
                dot[j] = 0.f;
                wj[j] = 0.f;
                p[j] = j0 + j < k ? pos[t * k + j0 + j] : -1;
                if (p[j] >= n_rows) p[j] = -1;
                if (p[j] >= 0) wj[j] = w ? w[t * k + j0 + j] : 1.f;
            }
            float w_lane = 0.f;   // slot lane & 7
            if (FP8)
#pragma unroll
                for (int j = 0; j < S; j++)
                    if ((lane & 7) == j) w_lane = fabsf(wj[j]);
            for (long long c0 = 0; c0 < d; c0 += (long long)blockDim.x * 8) {
                const long long c = c0 + threadIdx.x * 8;
                const int n = columns_at(c, d);
                const Vec8 g = load8(dout + t * ld_dout + c, n, wide);
                float s_lane = 0.f, r_lane = 0.f;
#pragma unroll
                for (int jb = 0; jb < S; jb += B) {
                    Raw8<T> r[B];
                    if (dw)
#pragma unroll
                        for (int j = 0; j < B; j++)
                            if (p[jb + j] >= 0) r[j] = load_raw8(rows + p[jb + j] * ld_rows + c, n, wide);
                    if (FP8 && jb == 0) {
                        s_lane = block_scale(__fmul_rn(w_lane, half_warp_amax(g)));
                        r_lane = 1.f / s_lane;
                    }
#pragma unroll
                    for (int u = 0; u < B; u++) {
                        const int j = jb + u;
                        if (p[j] < 0) continue;   // the same for all threads of the CTA
                        Vec8 v;
#pragma unroll
                        for (int i = 0; i < 8; i++) v.v[i] = __fmul_rn(wj[j], g.v[i]);
                        if constexpr (FP8) {
                            const float s = __shfl_sync(0xffffffffu, s_lane, j, 16), q = __shfl_sync(0xffffffffu, r_lane, j, 16);
                            if (n) {
                                store_codes8(codes + p[j] * ld_d + c, codes8(v, s, q), n, wide_d);
                                if ((threadIdx.x & 15) == 0) scales[p[j] * ld_s + c / kFp8Block] = s;
                            }
                        } else if (n) {
                            store8(drows + p[j] * ld_d + c, v, n, wide_d);
                        }
                        if (dw)
#pragma unroll
                            for (int i = 0; i < 8; i++) dot[j] = fmaf(g.v[i], column(r[u], i), dot[j]);
                    }
                }
            }
            if (!dw) continue;
#pragma unroll
            for (int j = 0; j < S; j++) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
                if (lane == 0) part[j][warp] = dot[j];
            }
            __syncthreads();
            if (warp < S && j0 + warp < k) {
                float v = lane < warps ? part[warp][lane] : 0.f;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (lane == 0) dw[t * k + j0 + warp] = v;   // 0 for a slot without a row
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------ rows into 8 bits

template <typename T>
__global__ void quantize_fp8_kernel(const T* __restrict__ x, long long ld_x, long long rows,
                                    const int32_t* __restrict__ n_dev, long long cols, int segments,
                                    uint8_t* __restrict__ codes, long long ld_c, float* __restrict__ scales,
                                    long long ld_s, bool wide_x, bool wide_c) {
    if (n_dev) rows = min(rows, (long long)max(*n_dev, 0));
    for (long long u = blockIdx.x; u < rows * segments; u += gridDim.x) {
        const long long t = u / segments;
        const long long c = ((u - t * segments) * blockDim.x + threadIdx.x) * 8;
        const int n = columns_at(c, cols);
        const Vec8 v = load8(x + t * ld_x + c, n, wide_x);
        const float s = half_warp_scale(v);
        if (!n) continue;
        store_codes8(codes + t * ld_c + c, codes8(v, s), n, wide_c);
        if ((threadIdx.x & 15) == 0) scales[t * ld_s + c / kFp8Block] = s;
    }
}

// One CTA of 256 threads per 128 x 128 block of a weight matrix (rows x cols,
// dense): thread i holds 8 columns of every 16th row.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_fp8_weights_kernel(const T* __restrict__ w, long long rows, long long cols, uint8_t* __restrict__ codes,
                            float* __restrict__ scales, bool wide) {
    __shared__ float top[8];
    const long long r0 = (long long)blockIdx.y * kFp8Block, c = (long long)blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8;
    const long long base = (long long)blockIdx.z * rows * cols;
    const int n = columns_at(c, cols);
    Vec8 v[8];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const long long r = r0 + (threadIdx.x >> 4) + 16 * i;
        v[i] = load8(w + base + r * cols + c, r < rows ? n : 0, wide);
#pragma unroll
        for (int q = 0; q < 8; q++) m = max_nan(m, fabsf(v[i].v[q]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) m = max_nan(m, top[i]);
    const float s = block_scale(m);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const long long r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r < rows && n) store_codes8(codes + base + r * cols + c, codes8(v[i], s), n, wide);
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
struct Swiglu {
    float g, u, sig;
    bool g_in, u_in;
};
__device__ __forceinline__ Swiglu swiglu_parts(float gate, float up, float limit) {
    Swiglu r;
    r.g_in = r.u_in = true;
    r.g = gate;
    r.u = up;
    if (limit > 0.f) {
        r.g_in = !(gate > limit);
        r.u_in = !(fabsf(up) > limit);
        if (!r.g_in) r.g = limit;                       // a NaN stays one
        if (!r.u_in) r.u = copysignf(limit, up);
    }
    const float e = expf(-fabsf(r.g));   // never overflows
    r.sig = __fdividef(r.g < 0.f ? e : 1.f, 1.f + e);   // the divisor is in [1, 2]: within 2 ulp
    return r;
}

template <typename T>
__global__ void swiglu_fp8_kernel(const T* __restrict__ gu, long long ld, long long rows,
                                  const int32_t* __restrict__ n_dev, long long f, int segments, float limit,
                                  uint8_t* __restrict__ codes, long long ld_c, float* __restrict__ scales, long long ld_s,
                                  bool wide, bool wide_c) {
    if (n_dev) rows = min(rows, (long long)max(*n_dev, 0));
    for (long long x = blockIdx.x; x < rows * segments; x += gridDim.x) {
        const long long t = x / segments;
        const long long c = ((x - t * segments) * blockDim.x + threadIdx.x) * 8;
        const int n = columns_at(c, f);
        const Vec8 g = load8(gu + t * ld + c, n, wide), u = load8(gu + t * ld + f + c, n, wide);
        Vec8 h;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const Swiglu p = swiglu_parts(g.v[i], u.v[i], limit);
            h.v[i] = i < n ? p.g * p.sig * p.u : 0.f;
        }
        const float s = half_warp_scale(h);
        if (!n) continue;
        store_codes8(codes + t * ld_c + c, codes8(h, s), n, wide_c);
        if ((threadIdx.x & 15) == 0) scales[t * ld_s + c / kFp8Block] = s;
    }
}

// f is a multiple of 128 here, so no block of the 2f columns holds both halves
template <typename T>
__global__ void swiglu_fp8_grad_kernel(const T* __restrict__ gu, long long ld, const T* __restrict__ dh, long long ld_dh,
                                       long long rows, const int32_t* __restrict__ n_dev, long long f, int segments,
                                       float limit, uint8_t* __restrict__ codes, long long ld_c,
                                       float* __restrict__ scales, long long ld_s, bool wide, bool wide_c) {
    if (n_dev) rows = min(rows, (long long)max(*n_dev, 0));
    for (long long x = blockIdx.x; x < rows * segments; x += gridDim.x) {
        const long long t = x / segments;
        const long long c = ((x - t * segments) * blockDim.x + threadIdx.x) * 8;
        const int n = columns_at(c, f);
        const Vec8 g = load8(gu + t * ld + c, n, wide), u = load8(gu + t * ld + f + c, n, wide);
        const Vec8 d = load8(dh + t * ld_dh + c, n, wide);
        Vec8 dg, du;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const Swiglu p = swiglu_parts(g.v[i], u.v[i], limit);
            const float silu = p.g * p.sig;
            dg.v[i] = i < n && p.g_in ? d.v[i] * p.u * (p.sig * (1.f + p.g * (1.f - p.sig))) : 0.f;
            du.v[i] = i < n && p.u_in ? d.v[i] * silu : 0.f;
        }
        const float sg = half_warp_scale(dg), su = half_warp_scale(du);
        if (!n) continue;
        store_codes8(codes + t * ld_c + c, codes8(dg, sg), n, wide_c);
        store_codes8(codes + t * ld_c + f + c, codes8(du, su), n, wide_c);
        if ((threadIdx.x & 15) == 0) {
            scales[t * ld_s + c / kFp8Block] = sg;
            scales[t * ld_s + (f + c) / kFp8Block] = su;
        }
    }
}

}  // namespace qrm
