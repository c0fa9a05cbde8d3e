// rows.cu -- entry points of the token-row operators (kernels: rows.cuh).
// Stateless: they run on the calling thread's current device and keep nothing.
#include <algorithm>
#include <climits>

#include "host_util.h"
#include "rows4.cuh"
#include "rows_host.h"

namespace qrm {
namespace {

// The CTAs that fit on the SMs at once, for kernels that walk the rows.
int walkers(int64_t rows, unsigned pieces, int sms, int resident) {
    return (int)std::min<int64_t>(rows, std::max<int64_t>(1, (int64_t)sms * resident / pieces));
}

// Columns to threads, `each` of them in one, in whole blocks of 128; at most
// 256 threads a CTA, spread evenly over the pieces that a row is cut into
// (7168 columns: 4 x 224 threads of 8, 2 x 224 threads of 16).
struct Cut {
    int threads;
    dim3 grid;
};
Cut cut_columns(int64_t rows, int64_t cols, int each) {
    const int64_t lanes = (cols + kFp8Block - 1) / kFp8Block * (kFp8Block / each);
    const int64_t pieces = (lanes + 255) / 256;
    const int64_t threads = ((lanes + pieces - 1) / pieces + 31) / 32 * 32;
    return {(int)threads, dim3((unsigned)rows, (unsigned)pieces)};
}

}  // namespace
}  // namespace qrm

using namespace qrm;

extern "C" int qrm_sort_tokens(const int32_t* topk_idx_dev, int64_t T, int k, int first, int n_experts,
                               int32_t* perm_dev, int32_t* pos_dev, int32_t* offsets_dev, void* stream) {
    const char* what = "qrm_sort_tokens";
    TRY(check_tokens(what, T, k, 0));
    if (n_experts <= 0) return failf(QRM_E_INVALID, "%s: %d experts", what, n_experts);
    if (n_experts > kSortMaxExperts)
        return failf(QRM_E_CAPACITY, "%s: %d experts, at most %d", what, n_experts, kSortMaxExperts);
    if (first < 0 || first > INT_MAX - n_experts) return failf(QRM_E_INVALID, "%s: first expert %d", what, first);
    TRY(check_ints(what, "offsets", offsets_dev));
    if (T > 0) {
        TRY(check_ints(what, "topk_idx", topk_idx_dev));
        TRY(check_ints(what, "perm", perm_dev));
        TRY(check_ints(what, "pos", pos_dev));
    }
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    const int64_t n = T * k;
    const bool many = n > 4096;
    const int warps = (int)std::min<int64_t>(32, std::max<int64_t>(8, (n + 255) / 256 * 8));
    cudaLaunchConfig_t cfg = {};
    int bits = 1;
    while (n_experts >> bits) bits++;   // an expert outside is all ones, which no expert is in this many bits
    cfg.gridDim = dim3(many ? kSortCluster : 1);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = sizeof(int32_t) * (size_t)(2 + warps) * n_experts;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cfg.gridDim.x;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // as in launch_ahead
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    auto kernel = many ? sort_tokens_kernel<kSortCluster> : sort_tokens_kernel<1>;
    e = cudaSuccess;
    // a launch has 48 KB without asking, the kernel's own warp sums included
    if (cfg.dynamicSmemBytes + kSortOwnSmem > 48 * 1024)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)(sizeof(int32_t) * 34 * kSortMaxExperts));
    if (e == cudaSuccess)
        e = cudaLaunchKernelEx(&cfg, kernel, topk_idx_dev, (long long)n, first, n_experts, bits, perm_dev, pos_dev, offsets_dev);
    return done(what, e);
}

extern "C" int qrm_gather_rows(int type, const void* x_dev, int64_t ld_x, const int32_t* pos_dev, int64_t T, int k,
                               int64_t d, void* rows_dev, int64_t n_rows, int64_t ld_rows, void* stream) {
    const char* what = "qrm_gather_rows";
    TRY(check_rows(what, type, T, d));
    TRY(check_tokens(what, T, k, n_rows));
    if (T == 0 || n_rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "x", x_dev, &ld_x, d, b));
    TRY(check_array(what, "rows", rows_dev, &ld_rows, d, b));
    TRY(check_ints(what, "pos", pos_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    const Cut c = cut_columns(T, d, 8);
    const bool wide = wide_rows(x_dev, ld_x, b) && wide_rows(rows_dev, ld_rows, b);
    BY_TYPE(type, e = launch_ahead(gather_rows_kernel<V>, c.grid, c.threads, 0, (cudaStream_t)stream, (const V*)x_dev, ld_x, pos_dev, k, (int)d, (uint32_t)n_rows, (V*)rows_dev, ld_rows, wide));
    return done(what, e);
}

extern "C" int qrm_gather_rows_fp8(int type, const void* x_dev, int64_t ld_x, const int32_t* pos_dev, int64_t T, int k,
                                   int64_t d, uint8_t* codes_dev, int64_t n_rows, int64_t ld_codes, float* scales_dev,
                                   int64_t ld_scales, void* stream) {
    const char* what = "qrm_gather_rows_fp8";
    TRY(check_rows(what, type, T, d));
    TRY(check_tokens(what, T, k, n_rows));
    if (T == 0 || n_rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "x", x_dev, &ld_x, d, b));
    TRY(check_array(what, "codes", codes_dev, &ld_codes, d, 1));
    TRY(check_array(what, "scales", scales_dev, &ld_scales, blocks_of(d), 4));
    TRY(check_ints(what, "pos", pos_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    const Cut c = cut_columns(T, d, 16);
    BY_TYPE(type, e = launch_ahead(gather_rows_fp8_kernel<V>, c.grid, c.threads, 0, (cudaStream_t)stream, (const V*)x_dev, ld_x, pos_dev, k, (int)d, (uint32_t)n_rows, codes_dev, ld_codes, scales_dev,
                      ld_scales, wide_rows(x_dev, ld_x, b), wide_codes16(codes_dev, ld_codes)));
    return done(what, e);
}

extern "C" int qrm_combine_rows(int type, const void* rows_dev, int64_t n_rows, int64_t ld_rows, const int32_t* pos_dev,
                                const float* w_dev, int64_t T, int k, int64_t d, const void* add_dev, int64_t ld_add,
                                void* out_dev, int64_t ld_out, void* stream) {
    const char* what = "qrm_combine_rows";
    TRY(check_rows(what, type, T, d));
    TRY(check_tokens(what, T, k, n_rows));
    if (T == 0) return QRM_OK;
    const int b = type_bytes(type);
    if (n_rows > 0) TRY(check_array(what, "rows", rows_dev, &ld_rows, d, b));
    if (add_dev) TRY(check_array(what, "add", add_dev, &ld_add, d, b));
    TRY(check_array(what, "out", out_dev, &ld_out, d, b));
    TRY(check_ints(what, "pos", pos_dev));
    if (w_dev) TRY(check_ints(what, "w", w_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    Cut c = cut_columns(T, d, 8);
    c.grid.x = walkers(T, c.grid.y, sms, 4 * 256 / c.threads);
    const bool wide = wide_rows(rows_dev, ld_rows, b) && wide_rows(out_dev, ld_out, b) &&
                      (!add_dev || wide_rows(add_dev, ld_add, b));
    BY_TYPE(type, e = launch_ahead(combine_rows_kernel<V>, c.grid, c.threads, 0, (cudaStream_t)stream, (const V*)rows_dev, ld_rows, (uint32_t)n_rows, pos_dev, w_dev, (uint32_t)T, k, (int)d, (const V*)add_dev, ld_add,
                      (V*)out_dev, ld_out, wide));
    return done(what, e);
}

// drows in the activations' type, or (codes, scales) in 8 bits
static int combine_grad(const char* what, int type, const void* dout_dev, int64_t ld_dout, const void* rows_dev,
                        int64_t n_rows, int64_t ld_rows, const int32_t* pos_dev, const float* w_dev, int64_t T, int k,
                        int64_t d, void* drows_dev, uint8_t* codes_dev, int64_t ld_d, float* scales_dev,
                        int64_t ld_scales, float* dw_dev, bool fp8, void* stream) {
    TRY(check_rows(what, type, T, d));
    TRY(check_tokens(what, T, k, n_rows));
    if (T == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "dout", dout_dev, &ld_dout, d, b));
    TRY(check_ints(what, "pos", pos_dev));
    if (n_rows > 0) {
        if (dw_dev) TRY(check_array(what, "rows", rows_dev, &ld_rows, d, b));
        if (fp8) {
            TRY(check_array(what, "codes", codes_dev, &ld_d, d, 1));
            TRY(check_array(what, "scales", scales_dev, &ld_scales, blocks_of(d), 4));
        } else {
            TRY(check_array(what, "drows", drows_dev, &ld_d, d, b));
        }
    }
    if (w_dev) TRY(check_ints(what, "w", w_dev));
    if (dw_dev) TRY(check_ints(what, "dw", dw_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    // one CTA per token, dout's columns in shared memory
    const size_t smem = sizeof(float) * blocks_of(std::min<int64_t>(d, kGradCols)) * kFp8Block;   // 32 KB at most
    const bool wide = wide_rows(dout_dev, ld_dout, b) && (!dw_dev || wide_rows(rows_dev, ld_rows, b));
    const bool wide_d = fp8 ? wide_codes(codes_dev, ld_d) : wide_rows(drows_dev, ld_d, b);
    const bool fast = wide && wide_d && d % 8 == 0;
    const cudaStream_t s = (cudaStream_t)stream;
#define QRM_GRAD(FP8, FAST)                                                                                             \
    BY_TYPE(type, e = launch_ahead(combine_grad_kernel<V, FP8, FAST>, dim3((unsigned)T), 256, smem, s, \
                      (const V*)dout_dev, ld_dout, (const V*)rows_dev, ld_rows, (uint32_t)n_rows, pos_dev, w_dev, k, (int)d, \
                      (V*)drows_dev, codes_dev, ld_d, scales_dev, ld_scales, dw_dev, wide, wide_d))
    if (fp8 && fast) QRM_GRAD(true, true);
    else if (fp8) QRM_GRAD(true, false);
    else if (fast) QRM_GRAD(false, true);
    else QRM_GRAD(false, false);
#undef QRM_GRAD
    return done(what, e);
}

extern "C" int qrm_combine_rows_grad(int type, const void* dout_dev, int64_t ld_dout, const void* rows_dev,
                                     int64_t n_rows, int64_t ld_rows, const int32_t* pos_dev, const float* w_dev,
                                     int64_t T, int k, int64_t d, void* drows_dev, int64_t ld_drows, float* dw_dev,
                                     void* stream) {
    return combine_grad("qrm_combine_rows_grad", type, dout_dev, ld_dout, rows_dev, n_rows, ld_rows, pos_dev, w_dev, T,
                        k, d, drows_dev, nullptr, ld_drows, nullptr, 0, dw_dev, false, stream);
}

extern "C" int qrm_combine_rows_grad_fp8(int type, const void* dout_dev, int64_t ld_dout, const void* rows_dev,
                                         int64_t n_rows, int64_t ld_rows, const int32_t* pos_dev, const float* w_dev,
                                         int64_t T, int k, int64_t d, uint8_t* codes_dev, int64_t ld_codes,
                                         float* scales_dev, int64_t ld_scales, float* dw_dev, void* stream) {
    return combine_grad("qrm_combine_rows_grad_fp8", type, dout_dev, ld_dout, rows_dev, n_rows, ld_rows, pos_dev, w_dev,
                        T, k, d, nullptr, codes_dev, ld_codes, scales_dev, ld_scales, dw_dev, true, stream);
}

extern "C" int qrm_quantize_fp8(int type, const void* x_dev, int64_t ld_x, int64_t rows, int64_t cols,
                                const int32_t* n_rows_dev, uint8_t* codes_dev, int64_t ld_codes, float* scales_dev,
                                int64_t ld_scales, void* stream) {
    const char* what = "qrm_quantize_fp8";
    TRY(check_rows(what, type, rows, cols));
    if (rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "x", x_dev, &ld_x, cols, b));
    TRY(check_array(what, "codes", codes_dev, &ld_codes, cols, 1));
    TRY(check_array(what, "scales", scales_dev, &ld_scales, blocks_of(cols), 4));
    if (n_rows_dev) TRY(check_ints(what, "n_rows", n_rows_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    const Cut c = cut_columns(rows, cols, 16);
    BY_TYPE(type, e = launch_ahead(quantize_fp8_kernel<V>, c.grid, c.threads, 0, (cudaStream_t)stream, (const V*)x_dev, ld_x, n_rows_dev, (int)cols, codes_dev, ld_codes, scales_dev, ld_scales,
                      wide_rows(x_dev, ld_x, b), wide_codes16(codes_dev, ld_codes)));
    return done(what, e);
}

extern "C" int qrm_quantize_fp8_weights(int type, const void* w_dev, int groups, int64_t rows, int64_t cols,
                                        uint8_t* codes_dev, float* scales_dev, void* stream) {
    const char* what = "qrm_quantize_fp8_weights";
    TRY(check_rows(what, type, rows, cols));
    if (groups <= 0 || groups > 65535 || rows <= 0 || blocks_of(rows) > 65535)
        return failf(QRM_E_INVALID, "%s: %d matrices of %lld rows", what, groups, (long long)rows);
    const int b = type_bytes(type);
    int64_t ld = 0, lds = 0, ldc = 0;
    TRY(check_array(what, "w", w_dev, &ld, cols, b));
    TRY(check_array(what, "codes", codes_dev, &ldc, cols, 1));
    TRY(check_array(what, "scales", scales_dev, &lds, blocks_of(cols), 4));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    const dim3 grid((unsigned)blocks_of(cols), (unsigned)blocks_of(rows), (unsigned)groups);
    const bool wide = wide_rows(w_dev, cols, b) && wide_codes(codes_dev, cols);
    BY_TYPE(type, e = launch_ahead(quantize_fp8_weights_kernel<V>, grid, 256, 0, (cudaStream_t)stream, (const V*)w_dev, (int)rows, (int)cols,
                                                                                         codes_dev, scales_dev, wide));
    return done(what, e);
}

// 4-bit rows: whole blocks of 16 bytes, and a byte for each block's scale
static int check_rows4(const char* what, uint8_t* codes, int64_t* ld_codes, uint8_t* scales, int64_t* ld_scales, int64_t cols) {
    TRY(check_array(what, "codes", codes, ld_codes, 16 * blocks4_of(cols), 1));
    return check_array(what, "scales", scales, ld_scales, blocks4_of(cols), 1);
}

extern "C" int qrm_gather_rows_fp4(int type, const void* x_dev, int64_t ld_x, const int32_t* pos_dev, int64_t T, int k,
                                   int64_t d, uint8_t* codes_dev, int64_t n_rows, int64_t ld_codes, uint8_t* scales_dev,
                                   int64_t ld_scales, void* stream) {
    const char* what = "qrm_gather_rows_fp4";
    TRY(check_rows(what, type, T, d));
    TRY(check_tokens(what, T, k, n_rows));
    if (T == 0 || n_rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "x", x_dev, &ld_x, d, b));
    TRY(check_rows4(what, codes_dev, &ld_codes, scales_dev, &ld_scales, d));
    TRY(check_ints(what, "pos", pos_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    const Cut c = cut_columns(T, d, 16);
    BY_TYPE(type, e = launch_ahead(gather_rows_fp4_kernel<V>, c.grid, c.threads, 0, (cudaStream_t)stream, (const V*)x_dev, ld_x, pos_dev, k, (int)d, (uint32_t)n_rows, codes_dev, ld_codes, scales_dev,
                      ld_scales, wide_rows(x_dev, ld_x, b), wide_codes(codes_dev, ld_codes)));
    return done(what, e);
}

extern "C" int qrm_quantize_fp4(int type, const void* x_dev, int64_t ld_x, int64_t rows, int64_t cols,
                                const int32_t* n_rows_dev, uint8_t* codes_dev, int64_t ld_codes, uint8_t* scales_dev,
                                int64_t ld_scales, void* stream) {
    const char* what = "qrm_quantize_fp4";
    TRY(check_rows(what, type, rows, cols));
    if (rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "x", x_dev, &ld_x, cols, b));
    TRY(check_rows4(what, codes_dev, &ld_codes, scales_dev, &ld_scales, cols));
    if (n_rows_dev) TRY(check_ints(what, "n_rows", n_rows_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    const Cut c = cut_columns(rows, cols, 16);
    BY_TYPE(type, e = launch_ahead(quantize_fp4_kernel<V>, c.grid, c.threads, 0, (cudaStream_t)stream, (const V*)x_dev, ld_x, n_rows_dev, (int)cols, codes_dev, ld_codes, scales_dev, ld_scales,
                      wide_rows(x_dev, ld_x, b), wide_codes(codes_dev, ld_codes)));
    return done(what, e);
}

static int check_limit(const char* what, float limit) {
    return limit >= 0.f ? QRM_OK : failf(QRM_E_INVALID, "%s: limit %g", what, (double)limit);
}

extern "C" int qrm_swiglu_fp8(int type, const void* gu_dev, int64_t ld_gu, int64_t rows, int64_t f,
                              const int32_t* n_rows_dev, float limit, uint8_t* codes_dev, int64_t ld_codes,
                              float* scales_dev, int64_t ld_scales, void* stream) {
    const char* what = "qrm_swiglu_fp8";
    TRY(check_rows(what, type, rows, f));
    TRY(check_limit(what, limit));
    if (rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "gu", gu_dev, &ld_gu, 2 * f, b));
    TRY(check_array(what, "codes", codes_dev, &ld_codes, f, 1));
    TRY(check_array(what, "scales", scales_dev, &ld_scales, blocks_of(f), 4));
    if (n_rows_dev) TRY(check_ints(what, "n_rows", n_rows_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    Cut c = cut_columns(rows, f, 8);
    c.grid.x = walkers(rows, c.grid.y, sms, 6 * 256 / c.threads);
    const bool wide = wide_rows(gu_dev, ld_gu, b) && f * b % 16 == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    const bool wide_c = wide_codes(codes_dev, ld_codes);
    if (limit > 0.f)
        BY_TYPE(type, e = launch_ahead(swiglu_fp8_kernel<V, true>, c.grid, c.threads, 0, s, (const V*)gu_dev, ld_gu, (int)rows, n_rows_dev, (int)f,
                          limit, codes_dev, ld_codes, scales_dev, ld_scales, wide, wide_c));
    else
        BY_TYPE(type, e = launch_ahead(swiglu_fp8_kernel<V, false>, c.grid, c.threads, 0, s, (const V*)gu_dev, ld_gu, (int)rows, n_rows_dev, (int)f,
                          limit, codes_dev, ld_codes, scales_dev, ld_scales, wide, wide_c));
    return done(what, e);
}

extern "C" int qrm_swiglu_fp8_grad(int type, const void* gu_dev, int64_t ld_gu, const void* dh_dev, int64_t ld_dh,
                                   int64_t rows, int64_t f, const int32_t* n_rows_dev, float limit, uint8_t* codes_dev,
                                   int64_t ld_codes, float* scales_dev, int64_t ld_scales, void* stream) {
    const char* what = "qrm_swiglu_fp8_grad";
    TRY(check_rows(what, type, rows, f));
    TRY(check_limit(what, limit));
    if (f % kFp8Block)
        return failf(QRM_E_INVALID, "%s: %lld columns are no whole blocks of %d, so one block would hold both halves",
                     what, (long long)f, kFp8Block);
    if (rows == 0) return QRM_OK;
    const int b = type_bytes(type);
    TRY(check_array(what, "gu", gu_dev, &ld_gu, 2 * f, b));
    TRY(check_array(what, "dh", dh_dev, &ld_dh, f, b));
    TRY(check_array(what, "codes", codes_dev, &ld_codes, 2 * f, 1));
    TRY(check_array(what, "scales", scales_dev, &ld_scales, blocks_of(2 * f), 4));
    if (n_rows_dev) TRY(check_ints(what, "n_rows", n_rows_dev));
    int device, sms;
    TRY(current_device(&device, &sms));
    cudaError_t e;
    Cut c = cut_columns(rows, f, 8);
    c.grid.x = walkers(rows, c.grid.y, sms, 4 * 256 / c.threads);
    const bool wide = wide_rows(gu_dev, ld_gu, b) && wide_rows(dh_dev, ld_dh, b);
    const cudaStream_t s = (cudaStream_t)stream;
    const bool wide_c = wide_codes(codes_dev, ld_codes);
    if (limit > 0.f)
        BY_TYPE(type, e = launch_ahead(swiglu_fp8_grad_kernel<V, true>, c.grid, c.threads, 0, s, (const V*)gu_dev, ld_gu, (const V*)dh_dev, ld_dh, (int)rows, n_rows_dev, (int)f, limit, codes_dev, ld_codes,
                          scales_dev, ld_scales, wide, wide_c));
    else
        BY_TYPE(type, e = launch_ahead(swiglu_fp8_grad_kernel<V, false>, c.grid, c.threads, 0, s, (const V*)gu_dev, ld_gu, (const V*)dh_dev, ld_dh, (int)rows, n_rows_dev, (int)f, limit, codes_dev, ld_codes,
                          scales_dev, ld_scales, wide, wide_c));
    return done(what, e);
}
