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
// Memory bounds both from some hundred rows on.  The CTAs walk the rows; one
// holds a row in registers, 8 neighbouring columns to a load, so that each row is
// read once.  Rows come by bulk copies into a ring of `slots` rows in shared
// memory, several ahead of the one that is worked on: a slot is free again once
// all threads have its row in registers, which the row's barrier says.  The wait
// for a copy is bounded; a CTA in which one gave up writes NaN to all its rows in
// the end (ring_walk.h).  A copy
// starts and ends on 16 bytes, so a row that does not is copied with the bytes
// around it and shifted into place on its way to registers; such a row goes out
// by way of shared memory, in words.  Where a CTA has one row, loads of its own
// are sooner there.  Rows that do not fit (more than 16384 columns, 8192 in the
// gradient) are read twice by the same kernels' last form (V = 0).
#pragma once
#include <type_traits>

#include "gemv_tma.cuh"
#include "ring_walk.h"
#include "rows4.cuh"

namespace qrm {

enum NormOut { kNormTyped = 0, kNorm8 = 1, kNorm4 = 2 };

constexpr int kNormSlots = 8;            // most of a ring
constexpr int kNormThreads = 512;   // most of a CTA

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

__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair both(float x) { return pair(x, x); }
// the sum over two packed sums of squares or products
__device__ __forceinline__ float joined(Pair p) {
    const float2 f = unpair(p);
    return f.x + f.y;
}
// eight values as they are stored
template <typename T>
__device__ __forceinline__ Raw8<T> rounded8(const Pairs8& v) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpair(v.p[i]);
        if constexpr (sizeof(T) == 4) {
            r.w[2 * i] = __float_as_uint(f.x);
            r.w[2 * i + 1] = __float_as_uint(f.y);
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __floats2half2_rn(f.x, f.y);
            memcpy(&r.w[i], &h, 4);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
            memcpy(&r.w[i], &h, 4);
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store_raw8(T* p, const Raw8<T>& r, int n, bool wide) {
    if (wide && n == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            reinterpret_cast<uint4*>(p)[i] = make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
    } else {
        T h[8];
        memcpy(h, r.w, sizeof h);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = h[i];
    }
}

// eight columns that this kernel may have written (no read-only path)
template <typename T>
__device__ __forceinline__ Raw8<T> load8_again(const T* p, int n) {
    Raw8<T> r;
    T h[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (sizeof(T) == 4) {
            h[i] = i < n ? *const_cast<const volatile T*>(p + i) : from_f32<T>(0.f);
        } else {
            const unsigned short b = i < n ? *reinterpret_cast<const volatile unsigned short*>(p + i) : 0;
            memcpy(&h[i], &b, 2);
        }
    }
    memcpy(r.w, h, sizeof h);
    return r;
}

// A ring of rows in shared memory: slot i % slots holds the CTA's i-th row of
// each of N arrays (NULL: none), `bytes` of it, with up to 15 bytes in front of it
// and behind it.  (Those bytes share 16 aligned ones with the row's own.)  How it is
// walked: ring_walk.h.
template <int N>
struct RowRing {
    const char* from[N];
    long long pitch[N];   // bytes
    uint32_t at;          // address in shared memory
    uint64_t* full;
    volatile int* given_up;   // [0]: a wait did, [1]: behind how many rows that were loaded
    uint32_t slots, rows;
    int bytes, room;          // room: bytes of a row there
    uint32_t i = 0, parity = 0, here = at;   // of the row that is worked on
    __device__ void init() {
        if (threadIdx.x == 0) {
            for (uint32_t k = 0; k < slots; k++) mbar_init(&full[k], 1);
            given_up[0] = 0;
            given_up[1] = -1;
            fence_barrier_init();
        }
        __syncthreads();
    }
    __device__ uint32_t offset(int j, uint32_t t) const {   // of row t from 16 bytes
        return ((uint32_t)reinterpret_cast<uintptr_t>(from[j]) + t * (uint32_t)pitch[j]) & 15;
    }
    // row t into slot k, by one thread
    __device__ void load(uint32_t k, unsigned long long row) {
        if (row >= rows) return;
        const uint32_t t = (uint32_t)row;
        uint32_t total = 0;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (from[j]) total += (offset(j, t) + bytes + 15) & ~15u;
        mbar_arrive_expect_tx(&full[k], total);
#pragma unroll
        for (int j = 0; j < N; j++)
            if (from[j])
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(at + (k * N + j) * room),
                    "l"(from[j] + (long long)t * pitch[j] - offset(j, t)), "r"((offset(j, t) + bytes + 15) & ~15u), "r"(smem_u32(&full[k]))
                    : "memory");
    }
    __device__ void start() {
        if (threadIdx.x == 0)
            for (uint32_t k = 0, t = blockIdx.x; k < slots && t < rows; k++, t += gridDim.x) load(k, t);
    }
    __device__ bool wait(uint32_t slot, uint32_t phase) {
        if (mbar_try_wait(&full[slot], phase)) return true;
        const uint64_t t0 = global_ns();
        for (;;) {
            for (int k = 0; k < 64; k++)
                if (mbar_try_wait(&full[slot], phase)) return true;
            if (failed() || global_ns() - t0 > kWaitLimitNs) return mbar_try_wait(&full[slot], phase);
        }
    }
    __device__ void drain(uint32_t slot, uint32_t phase) { mbar_wait(&full[slot], phase); }
    __device__ bool lead() const { return threadIdx.x == 0; }
    __device__ void fail() { *given_up = 1; }
    __device__ bool failed() const { return *given_up != 0; }
    __device__ void stop(unsigned long long row) {
        if (given_up[1] < 0) given_up[1] = (int)((min(row, (unsigned long long)rows + gridDim.x - 1) - blockIdx.x) / gridDim.x);
    }
    __device__ void next(uint32_t t) {
        ring_next(*this, t + (unsigned long long)slots * gridDim.x);
        here = i ? here + N * room : at;
    }
    // the n columns at c (the others are 0) of array j's row t; WHOLE: rows start and end on 16 bytes
    template <typename T, bool WHOLE>
    __device__ Raw8<T> row(int j, uint32_t t, int c, int n) const {
        constexpr int W = 2 * (int)sizeof(T);   // words of eight columns
        const uint32_t off = WHOLE ? 0 : offset(j, t), p = here + j * room + c * (int)sizeof(T);
        uint32_t w[W + 4];
#pragma unroll
        for (int k = 0; k < (WHOLE ? W : W + 4); k += 4) {
            w[k] = w[k + 1] = w[k + 2] = w[k + 3] = 0;
            if (n && n * (int)sizeof(T) + (int)off > 4 * k)
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[k]), "=r"(w[k + 1]), "=r"(w[k + 2]), "=r"(w[k + 3])
                             : "r"(p + 4 * k)
                             : "memory");
        }
        if (!WHOLE && off) {   // (the same for all threads)
            if (off & 8) {
#pragma unroll
                for (int k = 0; k < W + 2; k++) w[k] = w[k + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int k = 0; k < W + 1; k++) w[k] = w[k + 1];
            }
            if (off & 2) {
#pragma unroll
                for (int k = 0; k < W; k++) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
            }
        }
        Raw8<T> r;
#pragma unroll
        for (int k = 0; k < W; k++) r.w[k] = w[k];
        if (!WHOLE && n < 8) {
#pragma unroll
            for (int k = 0; k < W; k++) {
                if (sizeof(T) == 4) r.w[k] = k < n ? r.w[k] : 0;
                else r.w[k] = 2 * k + 1 < n ? r.w[k] : 2 * k < n ? r.w[k] & 0xffffu : 0;
            }
        }
        return r;
    }
};

// A row's way out when it does not start on 16 bytes: its columns into shared
// memory, then, behind a barrier, `bytes` of them to p by all threads, in words
// but for the ends.
template <int W>   // words
__device__ __forceinline__ void to_room(uint32_t at, const uint32_t (&w)[W]) {
    if constexpr (W == 2) {
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(w[0]), "r"(w[1]) : "memory");
    } else {
#pragma unroll
        for (int k = 0; k < W; k += 4)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + 4 * k), "r"(w[k]), "r"(w[k + 1]), "r"(w[k + 2]), "r"(w[k + 3])
                         : "memory");
    }
}
__device__ __forceinline__ uint32_t room_word(uint32_t at) {   // four bytes at any address
    uint32_t lo, hi;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(lo) : "r"(at & ~3u) : "memory");
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(hi) : "r"((at & ~3u) + 4) : "memory");
    return __funnelshift_r(lo, hi, 8 * (at & 3));
}
__device__ __forceinline__ void room_to(void* to, uint32_t room, int bytes) {
    char* p = static_cast<char*>(to);
    const int head = min((int)(-reinterpret_cast<intptr_t>(p) & 3), bytes), words = (bytes - head) >> 2, tail = head + 4 * words;
    for (int k = threadIdx.x; k < words; k += blockDim.x) *reinterpret_cast<uint32_t*>(p + head + 4 * k) = room_word(room + head + 4 * k);
    if ((int)threadIdx.x < head) p[threadIdx.x] = (char)room_word(room + threadIdx.x);
    if ((int)threadIdx.x < bytes - tail) p[tail + threadIdx.x] = (char)room_word(room + tail + threadIdx.x);
}

template <typename T>
struct NormArgs {
    const T *x, *add;        // add: NULL, or what is added
    const float* w;          // NULL: 1
    T *sum, *y;              // NULL: not wanted
    uint8_t* codes;
    void* scales;            // f32, or e8m0 bytes
    long long ld_x, ld_add, ld_sum, ld_y, ld_c, ld_s;
    int rows, d;
    int slots, room;             // of the ring (0: rows are loaded where they are needed), bytes of a row in it
    int sum_room, y_room, c_room;   // where in shared memory a row of it is put on its way out, 0: it is written as it is
    float eps, per_d;            // per_d: 1 / d
    bool wide, wide_sum, wide_y, wide_w, wide_c;   // rows start on 16 bytes (wide: those that are read)
};

// s of eight columns as it is stored: x, or x + add rounded
template <typename T>
__device__ __forceinline__ Raw8<T> norm_sum(const NormArgs<T>& a, const Raw8<T>& x, const Raw8<T>& add) {
    if (!a.add) return x;
    Pairs8 v = values8(x), u = values8(add);
#pragma unroll
    for (int i = 0; i < 4; i++) v.p[i] = add2(v.p[i], u.p[i]);
    return rounded8<T>(v);
}
__device__ __forceinline__ Pair squares(const Pairs8& s, Pair total) {
#pragma unroll
    for (int i = 0; i < 4; i++) total = fma2(s.p[i], s.p[i], total);
    return total;
}
__device__ __forceinline__ Pairs8 norm_weight(const float* w, int c, int n, bool wide) {
    Pairs8 r;
    if (w) return values8(load_raw8(w + c, n, wide));
#pragma unroll
    for (int i = 0; i < 4; i++) r.p[i] = both(1.f);
    return r;
}
__device__ __forceinline__ Vec8 weight8(const float* w, int c, int n, bool wide) {
    if (w) return load8(w + c, n, wide);
    Vec8 one;
#pragma unroll
    for (int i = 0; i < 8; i++) one.v[i] = 1.f;
    return one;
}
// y of a thread's 8 V neighbouring columns from c on (of those that do not exist
// s is 0, and so is y) to where it goes.  All 32 lanes take part.
template <typename T, int OUT, int V, bool WHOLE>
__device__ __forceinline__ void norm_out(const NormArgs<T>& a, uint32_t smem, long long t, const Pairs8 (&s)[V], const Pairs8 (&w)[V],
                                         float inv, int c) {
    Pairs8 y[V];   // negated where they are to become 8-bit codes
    const Pair f = both(OUT == kNorm8 ? -inv : inv);
#pragma unroll
    for (int v = 0; v < V; v++)
#pragma unroll
        for (int i = 0; i < 4; i++) y[v].p[i] = mul2(mul2(s[v].p[i], f), w[v].p[i]);
    if (OUT == kNormTyped || a.y) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int n = columns_at(c + 8 * v, a.d);
            Pairs8 z = y[v];
            if (OUT == kNorm8) {
#pragma unroll
                for (int i = 0; i < 4; i++) z.p[i] = negative(z.p[i]);
            }
            if (!WHOLE && a.y_room) to_room(smem + a.y_room + (c + 8 * v) * (int)sizeof(T), rounded8<T>(z).w);
            else if (n) store_raw8(a.y + t * a.ld_y + c + 8 * v, rounded8<T>(z), n, a.wide_y);
        }
    }
    if (OUT == kNormTyped) return;
    float top = 0.f;   // a NaN stays one
#pragma unroll
    for (int v = 0; v < V; v++) top = max_nan(top, amax8(y[v]));
    constexpr int kLanes = (OUT == kNorm8 ? 16 : 4) / V;   // of a block
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool lead = (threadIdx.x & (kLanes - 1)) == 0;
    if (OUT == kNorm8) {
        if (c >= a.d) return;
        const float scale = block_scale(top);
        const Quant q = quant(scale);
        uint2 codes[V];
#pragma unroll
        for (int v = 0; v < V; v++) codes[v] = scale < kFp8Tiny ? codes8_divided(y[v], scale) : codes8(y[v], q);
        uint8_t* to = a.codes + t * a.ld_c + c;
        if (!WHOLE && a.c_room) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                const uint32_t e[2] = {codes[v].x, codes[v].y};
                to_room(smem + a.c_room + c + 8 * v, e);
            }
        } else if (V > 1 && a.wide_c && c + 8 * V <= a.d) {
#pragma unroll
            for (int v = 0; v < V / 2; v++)
                reinterpret_cast<uint4*>(to)[v] = make_uint4(codes[2 * v].x, codes[2 * v].y, codes[2 * v + 1].x, codes[2 * v + 1].y);
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) {
                const int n = columns_at(c + 8 * v, a.d);
                if (n) store_codes8(to + 8 * v, codes[v], n, a.wide_c);
            }
        }
        if (lead) static_cast<float*>(a.scales)[t * a.ld_s + c / kFp8Block] = scale;
    } else {
        if (c / kFp4Block * kFp4Block >= a.d) return;   // (codes past the last column, 0, go up to the block's end)
        const uint32_t scale = fp4_scale(__float_as_uint(top));
        uint32_t codes[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 g = unpair(y[v].p[i]);
                e[2 * i] = g.x;
                e[2 * i + 1] = g.y;
            }
            codes[v] = e2m1x8(e, scale);
        }
        uint8_t* to = a.codes + t * a.ld_c + c / 2;
        if (a.wide_c) {
            if constexpr (V == 4) *reinterpret_cast<uint4*>(to) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            else if constexpr (V == 2) *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
            else *reinterpret_cast<uint32_t*>(to) = codes[0];
        } else {
#pragma unroll
            for (int i = 0; i < 4 * V; i++) to[i] = (uint8_t)(codes[i >> 2] >> (8 * (i & 3)));
        }
        if (lead) static_cast<uint8_t*>(a.scales)[t * a.ld_s + c / kFp4Block] = (uint8_t)scale;
    }
}
// 1 / sqrt(mean + eps), within 2 ulp
__device__ __forceinline__ float norm_factor(float total, float per_d, float eps) { return rsqrtf(fmaf(total, per_d, eps)); }

// Where a wait gave up: the copies land, and all that this CTA has written becomes NaN (out of line: it costs the
// others no registers)
struct RingEnd {
    uint64_t* full;
    uint32_t slots;
    __device__ void drain(uint32_t slot, uint32_t phase) { mbar_wait(&full[slot], phase); }
};
__device__ __forceinline__ void leave_ring(uint64_t* full, int slots, int issued) {
    RingEnd ring{full, (uint32_t)slots};
    if (threadIdx.x == 0) ring_drain(ring, (uint32_t)issued);
    __syncthreads();   // all of it is written
}
template <typename T, int OUT>
__device__ __noinline__ void spoil(const NormArgs<T>& a, uint64_t* full, int issued) {
    leave_ring(full, a.slots, issued);
    const float nan = __uint_as_float(0x7fffffffu);
    for (long long t = blockIdx.x; t < a.rows; t += gridDim.x) {
        for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
            if (a.sum) a.sum[t * a.ld_sum + c] = from_f32<T>(nan);
            if (a.y) a.y[t * a.ld_y + c] = from_f32<T>(nan);
            if (OUT == kNorm8 && c % kFp8Block == 0) static_cast<float*>(a.scales)[t * a.ld_s + c / kFp8Block] = nan;
            if (OUT == kNorm4 && c % kFp4Block == 0) static_cast<uint8_t*>(a.scales)[t * a.ld_s + c / kFp4Block] = 255;
        }
    }
}

// A row of 8 V neighbouring columns a thread (0: of any length, read twice).  sum
// may be x or add, y any of them: a thread has read a column before it writes it,
// and a row is copied ahead of others only.  WHOLE: all rows start and end on 16
// bytes (the code for others costs these a tenth of their time).
//
// 4096 x 7168 bf16 with the residual, the sum written, into 8 bits (206 MB): 38 us,
// 5.3 TB/s (a copy of as many bytes 35), 62 with loads of its own in place of the
// ring, one f32 at a time and 8 columns a thread.  One row of 7168 f32 columns 4.3.
// 4000 x 7001, whose rows start anywhere: 58, and 251 with loads of single values.
template <typename T, int OUT, int V, bool WHOLE>
__global__ void __launch_bounds__(kNormThreads)
rms_norm_kernel(const __grid_constant__ NormArgs<T> a) {
    extern __shared__ __align__(16) char ring_mem[];
    __shared__ uint64_t full[kNormSlots];
    __shared__ int given_up[2];
    __shared__ float scratch[2][1][32];   // two rows' turns
    const uint32_t smem = smem_u32(ring_mem);
    if constexpr (V > 0) {
        const int c = 8 * V * threadIdx.x;
        RowRing<2> ring{{reinterpret_cast<const char*>(a.x), reinterpret_cast<const char*>(a.add)},
                        {a.ld_x * (long long)sizeof(T), a.ld_add * (long long)sizeof(T)}, smem, full, given_up, (uint32_t)a.slots,
                        (uint32_t)a.rows, a.d * (int)sizeof(T), a.room};
        if (a.slots) ring.init();
        pdl_start();
        if (a.slots) ring.start();
        int turn = 0;
        Pairs8 w[V];
#pragma unroll
        for (int i = 0; i < V; i++) w[i] = norm_weight(a.w, c + 8 * i, columns_at(c + 8 * i, a.d), a.wide_w);
        for (uint32_t t = blockIdx.x; t < (uint32_t)a.rows; t += gridDim.x, turn ^= 1) {   // (unsigned, as in combine_rows_kernel)
            Raw8<T> raw[V], more[V];
            Pairs8 s[V];
            if (a.slots) ring_wait(ring);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int at = c + 8 * i, n = columns_at(at, a.d);
                raw[i] = a.slots ? ring.template row<T, WHOLE>(0, t, at, n) : load_raw8(a.x + t * a.ld_x + at, n, a.wide);
                if (a.add) more[i] = a.slots ? ring.template row<T, WHOLE>(1, t, at, n) : load_raw8(a.add + t * a.ld_add + at, n, a.wide);
            }
            Pair part = 0;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int at = c + 8 * i, n = columns_at(at, a.d);
                if (a.add) raw[i] = norm_sum(a, raw[i], more[i]);
                if (!WHOLE && a.sum_room) to_room(smem + a.sum_room + at * (int)sizeof(T), raw[i].w);
                else if (a.sum && n) store_raw8(a.sum + t * a.ld_sum + at, raw[i], n, a.wide_sum);
                s[i] = values8(raw[i]);
                part = squares(s[i], part);
            }
            float total[1] = {joined(part)};
            cta_sum(total, scratch[turn]);   // (one barrier a row: the turns keep a row's sum from the next one's)
            if (a.slots) ring.next(t);
            if (!WHOLE && a.sum_room) room_to(a.sum + t * a.ld_sum, smem + a.sum_room, a.d * (int)sizeof(T));
            norm_out<T, OUT, V, WHOLE>(a, smem, t, s, w, norm_factor(total[0], a.per_d, a.eps), c);
            if (!WHOLE && (a.sum_room | a.y_room | a.c_room)) {
                // What is in shared memory goes out.  It is written again behind the next row's barrier, but for the sum,
                // which is out by this one.
                __syncthreads();
                if (a.y_room) room_to(a.y + t * a.ld_y, smem + a.y_room, a.d * (int)sizeof(T));
                if (a.c_room) room_to(a.codes + t * a.ld_c, smem + a.c_room, a.d);
            }
        }
        if (a.slots && ring.failed()) spoil<T, OUT>(a, full, given_up[1]);   // (what is said before the last row's barrier is seen by all)
    } else {
        pdl_start();
        const int step = 8 * blockDim.x, c0 = 8 * threadIdx.x;
        const long long t = blockIdx.x;
        const T* x = a.x + t * a.ld_x;
        const T* add = a.add ? a.add + t * a.ld_add : nullptr;
        Pair part = 0;
        for (int c = c0; c < a.d; c += step) {
            const int n = columns_at(c, a.d);
            const Raw8<T> raw = load_raw8(x + c, n, a.wide);
            const Raw8<T> s = norm_sum(a, raw, add ? load_raw8(add + c, n, a.wide) : raw);
            if (a.sum) store_raw8(a.sum + t * a.ld_sum + c, s, n, a.wide_sum);
            part = squares(values8(s), part);
        }
        float total[1] = {joined(part)};
        cta_sum(total, scratch[0]);
        const float inv = norm_factor(total[0], a.per_d, a.eps);
        for (int base = 0; base < a.d; base += step) {   // whole warps: a block's lanes meet in norm_out
            const int c = base + c0, n = columns_at(c, a.d);
            Raw8<T> raw;
            if (a.sum) raw = load8_again(a.sum + t * a.ld_sum + c, n);
            else {
                raw = load8_again(x + c, n);
                if (add) raw = norm_sum(a, raw, load8_again(add + c, n));
            }
            const Pairs8 s[1] = {values8(raw)}, w[1] = {norm_weight(a.w, c, n, a.wide_w)};
            norm_out<T, OUT, 1, WHOLE>(a, 0, t, s, w, inv, c);
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
    int slots, room, dx_room;   // as in NormArgs
    float eps, per_d;
    bool wide, wide_dx, wide_w, wide_part;
};

// as the norm's
template <typename T>
__device__ __noinline__ void spoil(const NormGradArgs<T>& a, uint64_t* full, int issued) {
    leave_ring(full, a.slots, issued);
    const float nan = __uint_as_float(0x7fffffffu);
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
        for (long long t = blockIdx.x; t < a.rows; t += gridDim.x) a.dx[t * a.ld_dx + c] = from_f32<T>(nan);
        if (a.part) a.part[(size_t)blockIdx.x * a.d + c] = nan;
    }
}

// A thread keeps its 8 V columns' weights and their sums over the rows in
// registers, so the rows' products for dw are added up without atomics and in a
// fixed order: first a CTA's rows, then the CTAs' parts (rms_norm_dw_kernel).
//
// 4096 x 7168 bf16 with the residual's gradient and dw (235 MB): 49 us, 4.8 TB/s (a
// copy of as many bytes 40), 4 of them for dw.  4000 x 7001: 76, of single values
// 265.  1021 x 2816 f32: 11.5.  Two rows between two barriers and two CTAs an SM were
// no faster.
template <typename T, int V, bool WHOLE>
__global__ void __launch_bounds__(kNormThreads)
rms_norm_grad_kernel(const __grid_constant__ NormGradArgs<T> a) {
    extern __shared__ __align__(16) char ring_mem[];
    __shared__ uint64_t full[kNormSlots];
    __shared__ int given_up[2];
    __shared__ float scratch[2][2][32];   // two rows' turns
    int turn = 0;
    if constexpr (V > 0) {
        const uint32_t smem = smem_u32(ring_mem);
        RowRing<3> ring{{reinterpret_cast<const char*>(a.x), reinterpret_cast<const char*>(a.dy), reinterpret_cast<const char*>(a.add)},
                        {a.ld_x * (long long)sizeof(T), a.ld_dy * (long long)sizeof(T), a.ld_add * (long long)sizeof(T)},
                        smem, full, given_up, (uint32_t)a.slots, (uint32_t)a.rows, a.d * (int)sizeof(T), a.room};
        if (a.slots) ring.init();
        pdl_start();
        if (a.slots) ring.start();
        const int c = 8 * V * threadIdx.x;
        Pairs8 w[V], dw[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            w[i] = norm_weight(a.w, c + 8 * i, columns_at(c + 8 * i, a.d), a.wide_w);
#pragma unroll
            for (int j = 0; j < 4; j++) dw[i].p[j] = 0;
        }
        for (uint32_t t = blockIdx.x; t < (uint32_t)a.rows; t += gridDim.x, turn ^= 1) {   // (unsigned, as in combine_rows_kernel)
            Raw8<T> add[V];
            Pairs8 x[V], dy[V];
            if (a.slots) ring_wait(ring);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int at = c + 8 * i, n = columns_at(at, a.d);
                x[i] = values8(a.slots ? ring.template row<T, WHOLE>(0, t, at, n) : load_raw8(a.x + t * a.ld_x + at, n, a.wide));
                dy[i] = values8(a.slots ? ring.template row<T, WHOLE>(1, t, at, n) : load_raw8(a.dy + t * a.ld_dy + at, n, a.wide));
                if (a.add) add[i] = a.slots ? ring.template row<T, WHOLE>(2, t, at, n) : load_raw8(a.add + t * a.ld_add + at, n, a.wide);
            }
            Pair square = 0, product = 0;
#pragma unroll
            for (int i = 0; i < V; i++) {
                square = squares(x[i], square);
#pragma unroll
                for (int j = 0; j < 4; j++) product = fma2(mul2(dy[i].p[j], w[i].p[j]), x[i].p[j], product);
            }
            float sums[2] = {joined(square), joined(product)};
            cta_sum(sums, scratch[turn]);
            if (a.slots) ring.next(t);
            const float inv = norm_factor(sums[0], a.per_d, a.eps);
            const Pair f = both(inv), minus = both(-(sums[1] * a.per_d * inv));   // - mean(g n)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int at = c + 8 * i, n = columns_at(at, a.d);
                Pairs8 dx;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const Pair nrm = mul2(x[i].p[j], f);
                    dw[i].p[j] = fma2(dy[i].p[j], nrm, dw[i].p[j]);
                    dx.p[j] = mul2(f, fma2(nrm, minus, mul2(dy[i].p[j], w[i].p[j])));
                }
                if (a.add) {
                    const Pairs8 more = values8(add[i]);
#pragma unroll
                    for (int j = 0; j < 4; j++) dx.p[j] = add2(dx.p[j], more.p[j]);
                }
                if (!WHOLE && a.dx_room) to_room(smem + a.dx_room + at * (int)sizeof(T), rounded8<T>(dx).w);
                else if (n) store_raw8(a.dx + t * a.ld_dx + at, rounded8<T>(dx), n, a.wide_dx);
            }
            if (!WHOLE && a.dx_room) {   // (written again behind the next row's barrier)
                __syncthreads();
                room_to(a.dx + t * a.ld_dx, smem + a.dx_room, a.d * (int)sizeof(T));
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int at = c + 8 * i, n = columns_at(at, a.d);
            if (a.part && n) store_raw8(a.part + (size_t)blockIdx.x * a.d + at, rounded8<float>(dw[i]), n, a.wide_part);
        }
        if (a.slots && ring.failed()) spoil(a, full, given_up[1]);   // (as in rms_norm_kernel)
    } else {
        pdl_start();
        float* part = a.part ? a.part + (size_t)blockIdx.x * a.d : nullptr;
        const int step = 8 * blockDim.x;
        bool first = true;
        for (uint32_t t = blockIdx.x; t < (uint32_t)a.rows; t += gridDim.x, turn ^= 1) {
            float sums[2] = {0.f, 0.f};
            for (int c = 8 * threadIdx.x; c < a.d; c += step) {
                const int n = columns_at(c, a.d);
                const Vec8 x = load8(a.x + t * a.ld_x + c, n, a.wide), dy = load8(a.dy + t * a.ld_dy + c, n, a.wide);
                const Vec8 w = weight8(a.w, c, n, a.wide_w);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    sums[0] = fmaf(x.v[j], x.v[j], sums[0]);
                    sums[1] = fmaf(dy.v[j] * w.v[j], x.v[j], sums[1]);
                }
            }
            cta_sum(sums, scratch[turn]);
            const float inv = norm_factor(sums[0], a.per_d, a.eps);
            const float along = sums[1] * a.per_d * inv;
            for (int c = 8 * threadIdx.x; c < a.d; c += step) {
                const int n = columns_at(c, a.d);
                const Vec8 x = load8(a.x + t * a.ld_x + c, n, a.wide), dy = load8(a.dy + t * a.ld_dy + c, n, a.wide);
                const Vec8 w = weight8(a.w, c, n, a.wide_w);
                Vec8 dx, add;
                if (a.add) add = load8(a.add + t * a.ld_add + c, n, a.wide);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float nrm = x.v[j] * inv;
                    dx.v[j] = inv * fmaf(-nrm, along, dy.v[j] * w.v[j]);
                    if (a.add) dx.v[j] += add.v[j];
                    if (part && j < n) part[c + j] = fmaf(dy.v[j], nrm, first ? 0.f : part[c + j]);
                }
                store8(a.dx + t * a.ld_dx + c, dx, n, a.wide_dx);
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
    for (int p = first; c < d && p < last; p += 10) {   // (ten loads on their way: the 148 parts of long rows are ten a run)
        float v[10];
#pragma unroll
        for (int i = 0; i < 10; i++) v[i] = p + i < last ? __ldg(part + (size_t)(p + i) * d + c) : 0.f;
#pragma unroll
        for (int i = 0; i < 10; i++) t += v[i];
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
