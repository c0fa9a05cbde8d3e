// rows4.cuh -- rows in 4-bit microscaled floating point: e2m1 codes, two to a
// byte (the even column in the low four bits), and one e8m0 scale (a power of
// two, byte b stands for 2^(b - 127)) for each 32 columns.
//
//   scale = 2^max(floor(log2 amax) - 2, -127),   code = e2m1(v / scale)
//
// to nearest even, saturating at 6, e2m1's largest number: the block's largest
// magnitude lands in [4, 8), so only what is in (7, 8) of it loses more than a
// rounding.  Both steps are exact but for that one rounding: the exponent is
// read off the f32 number's bits, and the quotient by a power of two is a
// product.  A NaN or an infinity makes the block's scale 255, which stands for
// NaN: the whole block does then (its codes are 0), and its neighbours are
// untouched.
//
// A row of codes takes whole blocks (16 bytes each); the codes past its last
// column are 0.
#pragma once
#include "rows.cuh"

namespace qrm {

constexpr int kFp4Block = 32;

// the scale's byte by the bits of the block's largest magnitude (bits of f32
// magnitudes are in the order of their values, NaN above all)
__device__ __forceinline__ uint32_t fp4_scale(uint32_t amax) {
    const uint32_t e = amax >> 23;
    return e == 255 ? 255 : e > 2 ? e - 2 : 0;
}
// what values are multiplied with for their codes
__device__ __forceinline__ float fp4_inverse(uint32_t scale) { return __uint_as_float((254u - min(scale, 254u)) << 23); }
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// eight codes of a block with this scale, the first value's in the lowest bits
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8], uint32_t scale) {
    const float inverse = fp4_inverse(scale);
    uint32_t r;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(r)
        : "f"(v[0] * inverse), "f"(v[1] * inverse), "f"(v[2] * inverse), "f"(v[3] * inverse), "f"(v[4] * inverse),
          "f"(v[5] * inverse), "f"(v[6] * inverse), "f"(v[7] * inverse));
    return scale == 255 ? 0 : r;
}

// A thread's 16 columns of a row (a block is two neighbouring threads'), in
// 4 bits.  All 32 lanes take part.
struct Fp4Half {
    uint2 codes;
    uint32_t scale;
};
__device__ __forceinline__ Fp4Half fp4_half(const float (&lo)[8], const float (&hi)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, max(magnitude(lo[i]), magnitude(hi[i])));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    Fp4Half r;
    r.scale = fp4_scale(m);
    r.codes = make_uint2(e2m1x8(lo, r.scale), e2m1x8(hi, r.scale));
    return r;
}
// 16 columns' codes at p; `wide`: p is on an 8-byte boundary
__device__ __forceinline__ void store_fp4_half(uint8_t* __restrict__ p, uint2 c, bool wide) {
    if (wide) {
        *reinterpret_cast<uint2*>(p) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
}
template <typename T>
__device__ __forceinline__ Fp4Half quantize4_16(const T* __restrict__ x, int n, bool wide) {
    const Vec8 a = load8(x, min(n, 8), wide), b = load8(x + 8, max(n - 8, 0), wide);
    return fp4_half(a.v, b.v);
}

// rows[pos[a]] = x[t] in 4 bits: a token's row is quantised once for all its
// slots, as gather_rows_fp8_kernel does in 8 bits.  Memory bounds both kernels:
// 1024 rows of 7168 bf16 columns to 8 places each (46 MB) 9.3 us, 4.9 TB/s; below,
// 4096 x 4096 bf16 (42 MB) 8.8 us, 4.8 TB/s, cold.  A thread takes half a block, so
// that its loads and stores are 16 and 8 bytes and a block's largest magnitude
// needs one exchange.
template <typename T>
__global__ void __launch_bounds__(256)
gather_rows_fp4_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ pos, int k, int d,
                       uint32_t n_rows, uint8_t* __restrict__ codes, long long ld_c, uint8_t* __restrict__ scales,
                       long long ld_s, bool wide_x, bool wide_c) {
    pdl_start();
    const int t = blockIdx.x, c = (blockIdx.y * blockDim.x + threadIdx.x) * 16;
    pos += (size_t)t * k;
    const Fp4Half q = quantize4_16(x + t * ld_x + c, columns_at(c, d, 16), wide_x);
    if (c / kFp4Block * kFp4Block >= d) return;   // past the row's last block
    const bool lead = (threadIdx.x & 1) == 0;
#pragma unroll 4
    for (int j = 0; j < k; j++) {
        const uint32_t p = pos[j];
        if (p >= n_rows) continue;
        store_fp4_half(codes + p * ld_c + c / 2, q.codes, wide_c);
        if (lead) scales[p * ld_s + c / kFp4Block] = (uint8_t)q.scale;
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
quantize_fp4_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ n_dev, int cols,
                    uint8_t* __restrict__ codes, long long ld_c, uint8_t* __restrict__ scales, long long ld_s, bool wide_x,
                    bool wide_c) {
    pdl_start();
    const long long t = blockIdx.x;
    if (n_dev && t >= *n_dev) return;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 16;
    const Fp4Half q = quantize4_16(x + t * ld_x + c, columns_at(c, cols, 16), wide_x);
    if (c / kFp4Block * kFp4Block >= cols) return;
    store_fp4_half(codes + t * ld_c + c / 2, q.codes, wide_c);
    if ((threadIdx.x & 1) == 0) scales[t * ld_s + c / kFp4Block] = (uint8_t)q.scale;
}

}  // namespace qrm
