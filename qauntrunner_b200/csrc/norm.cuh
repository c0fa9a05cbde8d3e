// norm.cuh -- root-mean-square norm of token rows, the residual's addition in
// front of it, and its gradient.
//
//   s = x + add, rounded to the activations' type;  inv = 1 / sqrt(mean(s^2) + eps)
//   y = s inv w, in the activations' type, in 8-bit rows or in 4-bit rows
//   dx = inv (g - n mean(g n)) + add,  dw = sum over the rows of dy n,  with n = s inv, g = dy w
//
// The norm is that of the sum as it is stored, so the gradient needs nothing
// else of the forward: a row's two sums (s^2 and g s) come in the one pass that
// reads it.  Everything between load and store is in 32 bits, rounded once.
//
// Memory bounds both from some hundred rows on.  A CTA holds a row in
// registers, 8 neighbouring columns to a load, so that each row is read once.
// Rows that do not fit (more than 16384 columns, 8192 in the gradient) are read
// twice by the same kernels' last form (V = 0).
#pragma once
#include "rows4.cuh"

namespace qrm {

enum NormOut { kNormTyped = 0, kNorm8 = 1, kNorm4 = 2 };

constexpr int kNormThreads = 512;        // most of a CTA of the forward
constexpr int kNormGradThreads = 1024;   // of the gradient, one chunk of 8 columns each

// N sums over the CTA's threads, in every one of them; the order is fixed
template <int N>
__device__ __forceinline__ void cta_sum(float (&v)[N], float (*scratch)[32]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        if (lane == 0) scratch[i][warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        float t = lane < warps ? scratch[i][lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        v[i] = t;
    }
}

// eight columns that this kernel may have written (no read-only path)
template <typename T>
__device__ __forceinline__ Vec8 load8_again(const T* p, int n) {
    Vec8 r;
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = i < n ? to_f32(*const_cast<const volatile T*>(p + i)) : 0.f;
    return r;
}
template <>
__device__ __forceinline__ Vec8 load8_again(const __half* p, int n) {
    Vec8 r;
#pragma unroll
    for (int i = 0; i < 8; i++)
        r.v[i] = i < n ? __half2float(__ushort_as_half(*reinterpret_cast<const volatile unsigned short*>(p + i))) : 0.f;
    return r;
}
template <>
__device__ __forceinline__ Vec8 load8_again(const __nv_bfloat16* p, int n) {
    Vec8 r;
#pragma unroll
    for (int i = 0; i < 8; i++)
        r.v[i] = i < n ? __bfloat162float(__ushort_as_bfloat16(*reinterpret_cast<const volatile unsigned short*>(p + i))) : 0.f;
    return r;
}

template <typename T>
struct NormArgs {
    const T *x, *add;        // add: NULL, or what is added
    const float* w;          // NULL: 1
    T *sum, *y;              // NULL: not wanted
    uint8_t* codes;
    void* scales;            // f32, or e8m0 bytes
    long long ld_x, ld_add, ld_sum, ld_y, ld_c, ld_s;
    int d;
    float eps;
    bool wide, wide_w, wide_c;   // rows (weights, codes) start on 16 (16, 8 or 4) bytes
};

// s of eight columns, as it is stored
template <typename T>
__device__ __forceinline__ Vec8 norm_sum(const NormArgs<T>& a, const Raw8<T>& x, const Raw8<T>& add) {
    Vec8 v;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v.v[i] = column(x, i);
        if (a.add) v.v[i] = to_f32(from_f32<T>(v.v[i] + column(add, i)));
    }
    return v;
}
// y of eight columns at c, of which n exist, to where it goes.  All 32 lanes take part.
template <typename T, int OUT>
__device__ __forceinline__ void norm_out(const NormArgs<T>& a, long long t, const Vec8& s, const Vec8& w, float inv, int c, int n) {
    Vec8 y;
#pragma unroll
    for (int i = 0; i < 8; i++) y.v[i] = s.v[i] * inv * w.v[i];
    if (OUT == kNormTyped || a.y) {
        if (n) store8(a.y + t * a.ld_y + c, y, n, a.wide);
    }
    if (OUT == kNorm8) {
        Pairs8 neg;
#pragma unroll
        for (int i = 0; i < 4; i++) neg.p[i] = pair(2 * i < n ? -y.v[2 * i] : 0.f, 2 * i + 1 < n ? -y.v[2 * i + 1] : 0.f);
        const float scale = block_scale(half_warp_max(amax8(neg)));
        if (n) {
            store_codes8(a.codes + t * a.ld_c + c, scale < kFp8Tiny ? codes8_divided(neg, scale) : codes8(neg, quant(scale)), n, a.wide_c);
            if ((threadIdx.x & 15) == 0) static_cast<float*>(a.scales)[t * a.ld_s + c / kFp8Block] = scale;
        }
    } else if (OUT == kNorm4) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            y.v[i] = i < n ? y.v[i] : 0.f;
            m = max(m, magnitude(y.v[i]));
        }
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const uint32_t scale = fp4_scale(m), q = e2m1x8(y.v, scale);
        if (c / kFp4Block * kFp4Block < a.d) {   // codes past the last column, 0, up to the block's end
            uint8_t* to = a.codes + t * a.ld_c + c / 2;
            if (a.wide_c) {
                *reinterpret_cast<uint32_t*>(to) = q;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) to[i] = (uint8_t)(q >> (8 * i));
            }
            if ((threadIdx.x & 3) == 0) static_cast<uint8_t*>(a.scales)[t * a.ld_s + c / kFp4Block] = (uint8_t)scale;
        }
    }
}
__device__ __forceinline__ Vec8 norm_weight(const float* w, int c, int n, bool wide) {
    if (w) return load8(w + c, n, wide);
    Vec8 one;
#pragma unroll
    for (int i = 0; i < 8; i++) one.v[i] = 1.f;
    return one;
}

// A row of V chunks of 8 columns a thread (0: of any length, read twice).  sum
// may be x or add, y any of them: a thread has read a column before it writes it.
template <typename T, int OUT, int V>
__global__ void __launch_bounds__(kNormThreads)
rms_norm_kernel(const __grid_constant__ NormArgs<T> a) {
    pdl_start();
    __shared__ float scratch[1][32];
    const long long t = blockIdx.x;
    const T* x = a.x + t * a.ld_x;
    const T* add = a.add ? a.add + t * a.ld_add : nullptr;
    float total[1] = {0.f};
    const int step = 8 * blockDim.x, c0 = 8 * threadIdx.x;
    if constexpr (V > 0) {
        Raw8<T> raw[V], more[V];
        Vec8 s[V], w[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * step, n = columns_at(c, a.d);
            raw[i] = load_raw8(x + c, n, a.wide);
            more[i] = add ? load_raw8(add + c, n, a.wide) : raw[i];
        }
#pragma unroll
        for (int i = 0; i < V; i++) w[i] = norm_weight(a.w, c0 + i * step, columns_at(c0 + i * step, a.d), a.wide_w);
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * step, n = columns_at(c, a.d);
            s[i] = norm_sum(a, raw[i], more[i]);
            if (a.sum && n) store8(a.sum + t * a.ld_sum + c, s[i], n, a.wide);
#pragma unroll
            for (int j = 0; j < 8; j++) total[0] = fmaf(s[i].v[j], s[i].v[j], total[0]);
        }
        cta_sum(total, scratch);
        const float inv = 1.f / sqrtf(total[0] / (float)a.d + a.eps);
#pragma unroll
        for (int i = 0; i < V; i++) norm_out<T, OUT>(a, t, s[i], w[i], inv, c0 + i * step, columns_at(c0 + i * step, a.d));
    } else {
        for (int c = c0; c < a.d; c += step) {
            const int n = columns_at(c, a.d);
            const Raw8<T> raw = load_raw8(x + c, n, a.wide);
            const Vec8 s = norm_sum(a, raw, add ? load_raw8(add + c, n, a.wide) : raw);
            if (a.sum) store8(a.sum + t * a.ld_sum + c, s, n, a.wide);
#pragma unroll
            for (int j = 0; j < 8; j++) total[0] = fmaf(s.v[j], s.v[j], total[0]);
        }
        cta_sum(total, scratch);
        const float inv = 1.f / sqrtf(total[0] / (float)a.d + a.eps);
        for (int base = 0; base < a.d; base += step) {   // whole warps: a block's lanes meet in norm_out
            const int c = base + c0, n = columns_at(c, a.d);
            Vec8 s;
            if (a.sum) {
                s = load8_again(a.sum + t * a.ld_sum + c, n);
            } else {
                const Vec8 u = load8_again(x + c, n);
                s = u;
                if (add) {
                    const Vec8 v = load8_again(add + c, n);
#pragma unroll
                    for (int j = 0; j < 8; j++) s.v[j] = to_f32(from_f32<T>(u.v[j] + v.v[j]));
                }
            }
            norm_out<T, OUT>(a, t, s, norm_weight(a.w, c, n, a.wide_w), inv, c, n);
        }
    }
}

template <typename T>
struct NormGradArgs {
    const T *dy, *x, *add;   // add: NULL, or the gradient that the residual stream brings
    const float* w;
    T* dx;
    float* part;             // [gridDim.x][d] sums over a CTA's rows, or NULL
    long long ld_dy, ld_x, ld_add, ld_dx;
    int rows, d;
    float eps;
    bool wide, wide_w, wide_part;
};

// The CTAs walk the rows, so that a thread keeps its columns' weights and their
// sums over the rows in registers; a row's loads are on their way while the one
// before it is worked on.
template <typename T, int V>
__global__ void __launch_bounds__(kNormGradThreads)
rms_norm_grad_kernel(const __grid_constant__ NormGradArgs<T> a) {
    pdl_start();
    __shared__ float scratch[2][2][32];   // two rows' turns
    int turn = 0;
    if constexpr (V == 1) {
        const int c = 8 * threadIdx.x, n = columns_at(c, a.d);
        const Vec8 w = norm_weight(a.w, c, n, a.wide_w);
        Vec8 dw;
#pragma unroll
        for (int j = 0; j < 8; j++) dw.v[j] = 0.f;
        uint32_t t = blockIdx.x;   // (unsigned: a step past the last of 2^31 - 1 rows stays a number past it)
        Raw8<T> x = load_raw8(a.x + t * a.ld_x + c, n, a.wide), dy = load_raw8(a.dy + t * a.ld_dy + c, n, a.wide);
        for (; t < (uint32_t)a.rows; turn ^= 1) {
            const uint32_t next = t + gridDim.x;
            Raw8<T> x1 = x, dy1 = dy, add = x;
            if (a.add) add = load_raw8(a.add + t * a.ld_add + c, n, a.wide);
            if (next < (uint32_t)a.rows) {
                x1 = load_raw8(a.x + next * a.ld_x + c, n, a.wide);
                dy1 = load_raw8(a.dy + next * a.ld_dy + c, n, a.wide);
            }
            float sums[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float s = column(x, j), g = column(dy, j) * w.v[j];
                sums[0] = fmaf(s, s, sums[0]);
                sums[1] = fmaf(g, s, sums[1]);
            }
            cta_sum(sums, scratch[turn]);   // (one barrier a row: the turns keep a row's sums from the next one's)
            const float inv = 1.f / sqrtf(sums[0] / (float)a.d + a.eps);
            const float along = sums[1] / (float)a.d * inv;   // mean(g n)
            Vec8 dx;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float nrm = column(x, j) * inv, g = column(dy, j);
                dw.v[j] = fmaf(g, nrm, dw.v[j]);
                dx.v[j] = inv * fmaf(-nrm, along, g * w.v[j]);
                if (a.add) dx.v[j] += column(add, j);
            }
            if (n) store8(a.dx + t * a.ld_dx + c, dx, n, a.wide);
            x = x1;
            dy = dy1;
            t = next;
        }
        if (a.part && n) store8(a.part + (size_t)blockIdx.x * a.d + c, dw, n, a.wide_part);
    } else {
        float* part = a.part ? a.part + (size_t)blockIdx.x * a.d : nullptr;
        const int step = 8 * blockDim.x;
        bool first = true;
        for (uint32_t t = blockIdx.x; t < (uint32_t)a.rows; t += gridDim.x, turn ^= 1) {
            float sums[2] = {0.f, 0.f};
            for (int c = 8 * threadIdx.x; c < a.d; c += step) {
                const int n = columns_at(c, a.d);
                const Vec8 x = load8(a.x + t * a.ld_x + c, n, a.wide), dy = load8(a.dy + t * a.ld_dy + c, n, a.wide);
                const Vec8 w = norm_weight(a.w, c, n, a.wide_w);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    sums[0] = fmaf(x.v[j], x.v[j], sums[0]);
                    sums[1] = fmaf(dy.v[j] * w.v[j], x.v[j], sums[1]);
                }
            }
            cta_sum(sums, scratch[turn]);
            const float inv = 1.f / sqrtf(sums[0] / (float)a.d + a.eps);
            const float along = sums[1] / (float)a.d * inv;
            for (int c = 8 * threadIdx.x; c < a.d; c += step) {
                const int n = columns_at(c, a.d);
                const Vec8 x = load8(a.x + t * a.ld_x + c, n, a.wide), dy = load8(a.dy + t * a.ld_dy + c, n, a.wide);
                const Vec8 w = norm_weight(a.w, c, n, a.wide_w);
                Vec8 dx, add;
                if (a.add) add = load8(a.add + t * a.ld_add + c, n, a.wide);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float nrm = x.v[j] * inv;
                    dx.v[j] = inv * fmaf(-nrm, along, dy.v[j] * w.v[j]);
                    if (a.add) dx.v[j] += add.v[j];
                    if (part && j < n) part[c + j] = fmaf(dy.v[j], nrm, first ? 0.f : part[c + j]);
                }
                store8(a.dx + t * a.ld_dx + c, dx, n, a.wide);
            }
            first = false;
        }
    }
}

// dw = the sum of the CTAs' parts, in a fixed order: 32 columns a CTA, each
// column's parts in 16 runs, which are added up one after the other.
constexpr int kNormRuns = 16;
__global__ void __launch_bounds__(32 * kNormRuns)
rms_norm_dw_kernel(const float* __restrict__ part, int parts, int d, float* __restrict__ dw) {
    pdl_start();
    __shared__ float run[kNormRuns][32];
    const int lane = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const int first = parts * r / kNormRuns, last = parts * (r + 1) / kNormRuns;
    float t = 0.f;
    if (c < d) {
#pragma unroll 8
        for (int p = first; p < last; p++) t += part[(size_t)p * d + c];
    }
    run[r][lane] = t;
    __syncthreads();
    if (r == 0 && c < d) {
#pragma unroll
        for (int i = 1; i < kNormRuns; i++) t += run[i][lane];
        dw[c] = t;
    }
}

}  // namespace qrm
