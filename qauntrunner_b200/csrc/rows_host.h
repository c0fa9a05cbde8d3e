// rows_host.h -- what the units of token-row operators (rows.cu, norm.cu) share
// on the host: checks of their arguments, the choice by activation type.
#pragma once
#include <climits>

#include "host_util.h"
#include "rows4.cuh"

namespace qrm {
namespace {

bool wide_rows(const void* p, int64_t ld, int bytes) { return aligned(p, 16) && ld * bytes % 16 == 0; }
bool wide_codes(const void* p, int64_t ld) { return aligned(p, 8) && ld % 8 == 0; }
bool wide_codes16(const void* p, int64_t ld) { return aligned(p, 16) && ld % 16 == 0; }

constexpr int64_t kMaxCols = 1 << 24;   // columns of a row (a grid's y holds its pieces)

int check_rows(const char* what, int type, int64_t rows, int64_t cols) {
    if (!type_bytes(type)) return failf(QRM_E_FORMAT, "%s: type %d is not F32, F16 or BF16", what, type);
    if (rows < 0 || rows > (int64_t)INT_MAX) return failf(QRM_E_INVALID, "%s: %lld rows", what, (long long)rows);
    if (cols <= 0 || cols > kMaxCols) return failf(QRM_E_INVALID, "%s: %lld columns", what, (long long)cols);
    return QRM_OK;
}
int check_tokens(const char* what, int64_t T, int k, int64_t n_rows) {
    if (T < 0 || k <= 0 || T > INT_MAX / (int64_t)k)
        return failf(QRM_E_INVALID, "%s: %lld tokens x %d slots", what, (long long)T, k);
    if (n_rows < 0 || n_rows > (int64_t)INT_MAX) return failf(QRM_E_INVALID, "%s: %lld rows", what, (long long)n_rows);
    return QRM_OK;
}
// an array of values of `bytes` bytes each, in rows `ld` apart (0: dense)
int check_array(const char* what, const char* name, const void* p, int64_t* ld, int64_t cols, int bytes) {
    if (!p) return failf(QRM_E_INVALID, "%s: %s is NULL", what, name);
    if (!aligned(p, bytes)) return failf(QRM_E_INVALID, "%s: %s is not aligned to its %d-byte values", what, name, bytes);
    if (!pitch_ok(ld, cols))
        return failf(QRM_E_INVALID, "%s: pitch %lld of %s is below its %lld columns", what, (long long)*ld, name,
                     (long long)cols);
    return QRM_OK;
}
int check_ints(const char* what, const char* name, const void* p) {
    if (!p) return failf(QRM_E_INVALID, "%s: %s is NULL", what, name);
    if (!aligned(p, 4)) return failf(QRM_E_INVALID, "%s: %s is not aligned to 4 bytes", what, name);
    return QRM_OK;
}

#define TRY(expr)            \
    do {                     \
        int r_ = (expr);     \
        if (r_) return r_;   \
    } while (0)

// the statement with V = float, __half or __nv_bfloat16, by the activation type
#define BY_TYPE(type, ...)                                  \
    do {                                                    \
        if ((type) == QRM_F32) { using V = float; __VA_ARGS__; } \
        else if ((type) == QRM_F16) { using V = __half; __VA_ARGS__; } \
        else { using V = __nv_bfloat16; __VA_ARGS__; }      \
    } while (0)

int done(const char* what, cudaError_t e) {
    return e == cudaSuccess ? QRM_OK : failf(QRM_E_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

int64_t blocks_of(int64_t cols) { return (cols + kFp8Block - 1) / kFp8Block; }
int64_t blocks4_of(int64_t cols) { return (cols + kFp4Block - 1) / kFp4Block; }

}  // namespace
}  // namespace qrm
