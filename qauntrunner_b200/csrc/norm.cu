// norm.cu -- entry points of the root-mean-square norm and its gradient
// (kernels: norm.cuh).  Stateless, as those of rows.cu.
#include <algorithm>
#include <cmath>

#include "norm.cuh"
#include "rows_host.h"

using namespace qrm;

namespace {

int64_t chunks_of(int64_t d) { return (d + 7) / 8; }
int whole_warps(int64_t threads) { return (int)((threads + 31) / 32 * 32); }

int check_eps(const char* what, float eps) {
    return eps >= 0.f && std::isfinite(eps) ? QRM_OK : failf(QRM_E_INVALID, "%s: eps %g", what, (double)eps);
}

// Slots of a ring of rows, `bytes` each, that fit beside the other CTAs of the
// SM and `other` bytes of the CTA's own.  None where fewer than two fit, or where
// a CTA has one row only that its threads can load in wide pieces: it is there
// sooner (4.3 us in place of 5.1 for one row of 7168 f32 columns).
constexpr int kRingRoom = 200 * 1024;   // of an SM's 227 KB
int ring_slots(int64_t bytes, int64_t other, int ctas_an_sm, int64_t rows_a_cta, bool wide) {
    const int64_t fit = std::min<int64_t>((kRingRoom / ctas_an_sm - other) / bytes, kNormSlots);
    return fit < (wide ? 2 : 1) || (wide && rows_a_cta < 2) ? 0 : (int)std::min(fit, rows_a_cta);
}
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
template <typename A>
cudaError_t launch_ring(void (*kernel)(A), int64_t ctas, int threads, size_t smem, cudaStream_t s, const A& a) {
    if (smem > 46 * 1024) {   // a launch has 48 KB without asking, the kernel's own included
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingRoom);
        if (e != cudaSuccess) return e;
    }
    return launch_ahead(kernel, dim3((unsigned)ctas), threads, smem, s, a);
}

template <typename T, int OUT>
cudaError_t launch(NormArgs<T>& a, int sms, cudaStream_t s) {
    const int64_t chunks = chunks_of(a.d);
    if (chunks > 4 * kNormThreads) return launch_ahead(rms_norm_kernel<T, OUT, 0, false>, dim3((unsigned)a.rows), kNormThreads, 0, s, a);
    const int v = chunks <= 256 ? 1 : chunks <= 2 * kNormThreads ? 2 : 4, threads = whole_warps((chunks + v - 1) / v);
    const int an_sm = std::max(1, std::min(8, 1024 / threads));
    const int64_t ctas = std::min<int64_t>(a.rows, (int64_t)sms * an_sm);
    // rows that start elsewhere than on 16 bytes: with the bytes around them, and by way of shared memory out again
    const bool wide = a.wide && a.d * sizeof(T) % 16 == 0;
    a.room = (int)up16(a.d * sizeof(T) + (wide ? 0 : 30));
    const int64_t bytes = 2 * a.room, out = up16((int64_t)8 * v * threads * sizeof(T) + 16);   // (threads write whole chunks, words are read in twos)
    const bool by_sum = a.sum && !a.wide_sum, by_y = a.y && !a.wide_y, by_c = OUT == kNorm8 && !a.wide_c;
    const int64_t other = out * (by_sum + by_y + by_c);
    a.slots = ring_slots(bytes, other + 16, an_sm, (a.rows + ctas - 1) / ctas, wide && !other);
    size_t smem = 0;
    if (a.slots) {
        smem = a.slots * bytes + 16;   // (a row's last load may reach 16 bytes past it)
        for (int* room : {by_sum ? &a.sum_room : nullptr, by_y ? &a.y_room : nullptr, by_c ? &a.c_room : nullptr})
            if (room) {
                *room = (int)smem;
                smem += out;
            }
    }
    const bool whole = wide && !other;
    return launch_ring(v == 1   ? whole ? rms_norm_kernel<T, OUT, 1, true> : rms_norm_kernel<T, OUT, 1, false>
                       : v == 2 ? whole ? rms_norm_kernel<T, OUT, 2, true> : rms_norm_kernel<T, OUT, 2, false>
                                : rms_norm_kernel<T, OUT, 4, false>,
                       ctas, threads, smem, s, a);
}

int norm(const char* what, int out, int type, const void* x, int64_t ld_x, const void* add, int64_t ld_add, int64_t rows,
         int64_t d, const float* w, float eps, void* sum, int64_t ld_sum, void* y, int64_t ld_y, uint8_t* codes,
         int64_t ld_codes, void* scales, int64_t ld_scales, void* stream) {
    TRY(check_rows(what, type, rows, d));
    TRY(check_eps(what, eps));
    if (rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "x", x, &ld_x, d, b));
    if (add) TRY(check_array(what, "add", add, &ld_add, d, b));
    if (sum) TRY(check_array(what, "sum", sum, &ld_sum, d, b));
    if (y || out == kNormTyped) TRY(check_array(what, "y", y, &ld_y, d, b));
    if (out == kNorm8) {
        TRY(check_array(what, "codes", codes, &ld_codes, d, 1));
        TRY(check_array(what, "scales", scales, &ld_scales, blocks_of(d), 4));
    } else if (out == kNorm4) {
        TRY(check_array(what, "codes", codes, &ld_codes, 16 * blocks4_of(d), 1));
        TRY(check_array(what, "scales", scales, &ld_scales, blocks4_of(d), 1));
    }
    if (w) TRY(check_ints(what, "w", w));
    int device, sms;
    TRY(current_device(&device, &sms));
    const bool wide = wide_rows(x, ld_x, b) && (!add || wide_rows(add, ld_add, b));
    cudaError_t e;
    const cudaStream_t s = (cudaStream_t)stream;
    BY_TYPE(type, {
        NormArgs<V> a{(const V*)x, (const V*)add, w, (V*)sum, (V*)y, codes, scales, ld_x, ld_add, ld_sum, ld_y,
                      ld_codes, ld_scales, (int)rows, (int)d, 0, 0, 0, 0, 0, eps, 1.f / (float)d, wide, wide_rows(sum, ld_sum, b),
                      wide_rows(y, ld_y, b), aligned(w, 16), wide_codes16(codes, ld_codes)};
        e = out == kNormTyped ? launch<V, kNormTyped>(a, sms, s) : out == kNorm8 ? launch<V, kNorm8>(a, sms, s)
                                                                                 : launch<V, kNorm4>(a, sms, s);
    });
    return done(what, e);
}

// The gradient's columns a thread (chunks of 8; 0: the form that reads rows
// twice), its CTAs, and so many parts of dw: about 700 threads an SM.  With 512
// (or 1024) and 16 columns a thread from 1024 on, 4096 x 2816 bf16 takes 29 (21)
// us in place of 21, 4096 x 7168 48 (52) in place of 48, 1021 x 2816 f32 17 (11)
// in place of 11.  Other widths were not measured; from 2817 to 4096 columns a CTA
// has 384 to 512 threads, and an SM one of them.  (148 SMs, a number of its own, so
// that the room for the parts needs no device.)
int grad_chunks(int64_t d) { return chunks_of(d) <= 512 ? 1 : chunks_of(d) <= 2 * kNormThreads ? 2 : 0; }
int grad_threads(int64_t d) { return grad_chunks(d) ? whole_warps((chunks_of(d) + grad_chunks(d) - 1) / grad_chunks(d)) : kNormThreads; }
int grad_ctas_an_sm(int64_t d) { return std::max(1, std::min(4, 704 / grad_threads(d))); }
int64_t grad_ctas(int64_t rows, int64_t d) { return std::min<int64_t>(rows, 148 * grad_ctas_an_sm(d)); }

}  // namespace

extern "C" int qrm_rms_norm(int type, const void* x_dev, int64_t ld_x, const void* add_dev, int64_t ld_add, int64_t rows,
                            int64_t d, const float* w_dev, float eps, void* sum_dev, int64_t ld_sum, void* y_dev,
                            int64_t ld_y, void* stream) {
    return norm("qrm_rms_norm", kNormTyped, type, x_dev, ld_x, add_dev, ld_add, rows, d, w_dev, eps, sum_dev, ld_sum, y_dev,
                ld_y, nullptr, 0, nullptr, 0, stream);
}

extern "C" int qrm_rms_norm_fp8(int type, const void* x_dev, int64_t ld_x, const void* add_dev, int64_t ld_add, int64_t rows,
                                int64_t d, const float* w_dev, float eps, void* sum_dev, int64_t ld_sum, void* y_dev,
                                int64_t ld_y, uint8_t* codes_dev, int64_t ld_codes, float* scales_dev, int64_t ld_scales,
                                void* stream) {
    return norm("qrm_rms_norm_fp8", kNorm8, type, x_dev, ld_x, add_dev, ld_add, rows, d, w_dev, eps, sum_dev, ld_sum, y_dev,
                ld_y, codes_dev, ld_codes, scales_dev, ld_scales, stream);
}

extern "C" int qrm_rms_norm_fp4(int type, const void* x_dev, int64_t ld_x, const void* add_dev, int64_t ld_add, int64_t rows,
                                int64_t d, const float* w_dev, float eps, void* sum_dev, int64_t ld_sum, void* y_dev,
                                int64_t ld_y, uint8_t* codes_dev, int64_t ld_codes, uint8_t* scales_dev, int64_t ld_scales,
                                void* stream) {
    return norm("qrm_rms_norm_fp4", kNorm4, type, x_dev, ld_x, add_dev, ld_add, rows, d, w_dev, eps, sum_dev, ld_sum, y_dev,
                ld_y, codes_dev, ld_codes, scales_dev, ld_scales, stream);
}

extern "C" int64_t qrm_rms_norm_grad_work(int64_t rows, int64_t d) {
    if (rows <= 1 || rows > INT_MAX || d <= 0 || d > kMaxCols) return 0;
    return grad_ctas(rows, d) * d;
}

extern "C" int qrm_rms_norm_grad(int type, const void* dy_dev, int64_t ld_dy, const void* x_dev, int64_t ld_x, int64_t rows,
                                 int64_t d, const float* w_dev, float eps, const void* add_dev, int64_t ld_add, void* dx_dev,
                                 int64_t ld_dx, float* dw_dev, float* work_dev, void* stream) {
    const char* what = "qrm_rms_norm_grad";
    TRY(check_rows(what, type, rows, d));
    TRY(check_eps(what, eps));
    const int b = type_bytes(type);
    if (dw_dev) TRY(check_ints(what, "dw", dw_dev));
    const cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {   // a sum of nothing
        if (!dw_dev) return QRM_OK;
        int device, sms;
        TRY(current_device(&device, &sms));
        return done(what, launch_ahead(rms_norm_dw_kernel, dim3((unsigned)((d + 31) / 32)), 32 * kNormRuns, 0, s, dw_dev, 0, (int)d, dw_dev));
    }
    TRY(check_array(what, "dy", dy_dev, &ld_dy, d, b));
    TRY(check_array(what, "x", x_dev, &ld_x, d, b));
    if (add_dev) TRY(check_array(what, "add", add_dev, &ld_add, d, b));
    TRY(check_array(what, "dx", dx_dev, &ld_dx, d, b));
    if (w_dev) TRY(check_ints(what, "w", w_dev));
    const int64_t ctas = grad_ctas(rows, d);
    if (dw_dev && ctas > 1) TRY(check_ints(what, "work", work_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    const bool wide = wide_rows(dy_dev, ld_dy, b) && wide_rows(x_dev, ld_x, b) && (!add_dev || wide_rows(add_dev, ld_add, b));
    const bool wide_dx = wide_rows(dx_dev, ld_dx, b);
    float* part = !dw_dev ? nullptr : ctas > 1 ? work_dev : dw_dev;
    const int threads = grad_threads(d);
    const bool whole = wide && d * b % 16 == 0;
    const int64_t room = up16(d * b + (whole ? 0 : 30)), out = wide_dx ? 0 : up16((int64_t)8 * grad_chunks(d) * threads * b + 16);
    const int slots = grad_chunks(d) ? ring_slots(3 * room, out + 16, grad_ctas_an_sm(d), (rows + ctas - 1) / ctas, whole && wide_dx) : 0;
    const int64_t ring = slots ? 3 * room * slots + 16 : 0;
    cudaError_t e;
    BY_TYPE(type, {
        const NormGradArgs<V> a{(const V*)dy_dev, (const V*)x_dev, (const V*)add_dev, w_dev, (V*)dx_dev, part, ld_dy, ld_x,
                                ld_add, ld_dx, (int)rows, (int)d, slots, (int)room, slots && !wide_dx ? (int)ring : 0, eps,
                                1.f / (float)d, wide, wide_dx, aligned(w_dev, 16), aligned(part, 16) && d % 4 == 0};
        e = launch_ring(grad_chunks(d) == 1   ? whole && wide_dx ? rms_norm_grad_kernel<V, 1, true> : rms_norm_grad_kernel<V, 1, false>
                        : grad_chunks(d) == 2 ? whole && wide_dx ? rms_norm_grad_kernel<V, 2, true> : rms_norm_grad_kernel<V, 2, false>
                                              : rms_norm_grad_kernel<V, 0, false>,
                        ctas, threads, slots ? ring + out : 0, s, a);
    });
    if (e == cudaSuccess && dw_dev && ctas > 1)
        e = launch_ahead(rms_norm_dw_kernel, dim3((unsigned)((d + 31) / 32)), 32 * kNormRuns, 0, s, work_dev, (int)ctas, (int)d, dw_dev);
    return done(what, e);
}
