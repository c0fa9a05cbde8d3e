// fp8.cu -- matrices in 8-bit floating point with a scale for each 128 x 128
// block, resident in HBM, and their products (kernels: fp8.cuh).
#include <stdlib.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <new>

#include "fp8.cuh"
#include "host_util.h"
#include "umma_host.h"

using namespace qrm;

struct qrm_fp8 {
    int device = 0, sms = 0, groups = 0;
    int form = -1;                           // QRM_FP8_PAIR: 1 wherever it can / 0 never rows of x on the MMA's M side
    int64_t rows = 0, cols = 0, pitch = 0;   // of one matrix; pitch: bytes of a stored row
    uint8_t* codes = nullptr;                // [groups][rows][pitch]; the other arrays are in the same allocation
    float* scales = nullptr;                 // [groups][row blocks][column blocks]
    float* part = nullptr;                   // partial tiles of the CTAs
    int32_t* arrivals = nullptr;
    int32_t* err = nullptr;
    // the stored codes in boxes of 128 x 128, and, for a pair's CTA, of half a block of outputs: 64 outputs of
    // the product x 128 contracted, 64 of the transposed product x 128
    CUtensorMap map, pair_map, pair_map_t;
};

namespace {

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

void release(qrm_fp8* m) {
    if (!m) return;
    DeviceGuard here;
    here.enter(m->device);
    cudaDeviceSynchronize();
    cudaFree(m->codes);
    delete m;
}

// waits for what any stream still writes at p, when that is on another device
cudaError_t await_source(const void* p, int device) {
    cudaPointerAttributes at{};
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();   // the copy will say what is wrong with it
        return cudaSuccess;
    }
    if (at.type != cudaMemoryTypeDevice || at.device == device) return cudaSuccess;
    DeviceGuard there;
    const cudaError_t e = there.enter(at.device);
    return e == cudaSuccess ? cudaDeviceSynchronize() : e;
}

// 8-bit tensor of up to three dimensions, innermost first, as a TMA map; what
// lies outside reads as zero
bool encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint32_t step[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kSmemMost = 227 * 1024;
int stage_bytes(int x_rows) { return kFp8Tile + x_rows * 128; }
int stages_for(int groups, int x_rows) {
    return std::min(kFp8MaxStages, (kSmemMost - 1024 - fp8_stage_off(groups)) / stage_bytes(x_rows));
}
size_t smem_for(int groups, int x_rows) {
    return 1024 + (size_t)fp8_stage_off(groups) + (size_t)stages_for(groups, x_rows) * stage_bytes(x_rows);
}

size_t pair_smem(int groups) { return 1024 + (size_t)fp8_pair_stage_off(groups) + (size_t)kFp8PairStages * kFp8PairStage; }

int create(int device, int groups, int64_t rows, int64_t cols, const void* codes, size_t code_bytes, const float* scales,
           size_t scale_bytes, cudaMemcpyKind kind, qrm_fp8** out) {
    const char* what = "qrm_fp8_create";
    if (!out) return failf(QRM_E_INVALID, "%s: out is NULL", what);
    *out = nullptr;
    if (!codes || !scales) return failf(QRM_E_INVALID, "%s: NULL argument", what);
    if (groups <= 0 || rows <= 0 || cols <= 0 || rows > (1 << 24) || cols > (1 << 24))
        return failf(QRM_E_INVALID, "%s: %d matrices of %lld x %lld", what, groups, (long long)rows, (long long)cols);
    if (groups > kFp8MaxGroups) return failf(QRM_E_CAPACITY, "%s: %d matrices, at most %d", what, groups, kFp8MaxGroups);
    const int64_t nb = (int64_t)groups * blocks_of(rows) * blocks_of(cols);
    if (code_bytes != (size_t)(groups * rows * cols))
        return failf(QRM_E_SIZE, "%s: %zu bytes of codes, %d x %lld x %lld = %lld", what, code_bytes, groups,
                     (long long)rows, (long long)cols, (long long)(groups * rows * cols));
    if (scale_bytes != (size_t)nb * sizeof(float))
        return failf(QRM_E_SIZE, "%s: %zu bytes of scales, one f32 for each of %lld blocks is %lld", what, scale_bytes,
                     (long long)nb, (long long)nb * 4);
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) return failf(QRM_E_CUDA, "%s: no CUDA device", what);
    if (device < 0 || device >= count) return failf(QRM_E_INVALID, "%s: device %d out of range", what, device);
    int sms;
    DeviceGuard here;
    if (here.enter(device) != cudaSuccess) return failf(QRM_E_CUDA, "%s: device %d", what, device);
    if (int rc = current_device(&device, &sms)) return rc;
    if (const char* e = getenv("QRM_WAIT_LIMIT_US"))
        if (set_wait_limit_here((uint64_t)std::max(1LL, atoll(e)) * 1000ull) != cudaSuccess)
            return failf(QRM_E_CUDA, "%s: wait limit", what);
    qrm_fp8* m = new (std::nothrow) qrm_fp8();
    if (!m) return failf(QRM_E_NOMEM, "%s: host memory", what);
    auto bail = [&](int rc) {
        release(m);
        return rc;
    };
    if (const char* e = getenv("QRM_FP8_PAIR")) m->form = atoi(e) != 0;
    m->device = device;
    m->sms = sms;
    m->groups = groups;
    m->rows = rows;
    m->cols = cols;
    m->pitch = (cols + 15) / 16 * 16;
    // one allocation: codes, scales, partial tiles, arrivals, error flags
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t codes_at = up((size_t)groups * rows * m->pitch), scales_at = codes_at + up(scale_bytes);
    const size_t part_at = scales_at + up(sizeof(float) * (size_t)sms * 2 * kFp8MaxRows * 128);
    const size_t counts = sizeof(int32_t) * ((size_t)sms * kFp8EpiWarps + 1);
    if (cudaMalloc(&m->codes, part_at + counts) != cudaSuccess) {
        cudaGetLastError();
        return bail(failf(QRM_E_NOMEM, "%s: cannot allocate %zu bytes", what, part_at + counts));
    }
    m->scales = reinterpret_cast<float*>(m->codes + codes_at);
    m->part = reinterpret_cast<float*>(m->codes + scales_at);
    m->arrivals = reinterpret_cast<int32_t*>(m->codes + part_at);
    m->err = m->arrivals + (size_t)sms * kFp8EpiWarps;
    // device sources: what any stream still writes there is awaited, as in qrm_upload_expert_device, and on their own
    // device if that is another one
    cudaError_t e = cudaDeviceSynchronize();
    if (kind == cudaMemcpyDeviceToDevice) {
        if (e == cudaSuccess) e = await_source(codes, device);
        if (e == cudaSuccess) e = await_source(scales, device);
    }
    if (e == cudaSuccess) e = cudaMemcpy2D(m->codes, m->pitch, codes, cols, cols, (size_t)groups * rows, kind);
    if (e == cudaSuccess) e = cudaMemcpy(m->scales, scales, scale_bytes, kind);
    if (e == cudaSuccess) e = cudaMemset(m->arrivals, 0, counts);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fp8_stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(fp8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pair_smem(kFp8MaxGroups));
    cudaFuncAttributes pair{};
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&pair, fp8_pair_kernel);
    if (e != cudaSuccess) return bail(failf(QRM_E_CUDA, "%s: %s", what, cudaGetErrorString(e)));
    if (pair.numRegs * kFp8Warps * 32 < kFp8PairRegs)
        return bail(failf(QRM_E_CUDA, "%s: built with %d registers a thread, too few for its split", what, pair.numRegs));
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)groups};
    const cuuint64_t strides[2] = {(cuuint64_t)m->pitch, (cuuint64_t)(m->pitch * rows)};
    const cuuint32_t box[3] = {128, 128, 1};
    const cuuint32_t pair_box[3] = {128, 64, 1}, pair_box_t[3] = {64, 128, 1};
    if (!encode(&m->map, m->codes, 3, dims, strides, box) || !encode(&m->pair_map, m->codes, 3, dims, strides, pair_box) ||
        !encode(&m->pair_map_t, m->codes, 3, dims, strides, pair_box_t, CU_TENSOR_MAP_SWIZZLE_64B))
        return bail(failf(QRM_E_CUDA, "%s: tensor map", what));
    *out = m;
    return QRM_OK;
}

// Which kernel a product takes, by an estimate of what both would cost with all
// T rows held and spread evenly over the groups: where offsets leave many of
// them out (another rank's slots), it takes the large-group kernel too early, as
// 16 rows each counted as 128 at 32 x 4096 x 7168 would take 222 us in place of
// 179; a caller that knows how many are held passes that as T.  Measured (us; weights on the MMA's M
// side / rows of x on it), outputs x contracted:
//   1 x 4096 x 7168:  1 row 15 / 30, 64 rows 21 / 30, 256 rows 30 / 31, 512 rows 38 / 32
//   1 x 28672 x 4096: 1 row 32 / 42, 64 rows 39 / 38, 128 rows 46 / 39, 256 rows 78 / 40, 4096 rows 877 / 425
//   1 x 4096 x 28672: 1 row 30 / 95, 128 rows 46 / 96, 512 rows 128 / 99
//   1 x 1024 x 2816:  1 row 12 / 16, 64 rows 18 / 16, 512 rows 19 / 18
//   8 x 5632 x 1024:  1 row each 14 / 17, 64 rows each 24 / 23, 256 rows each 41 / 31
//   32 x 4096 x 7168: 16 rows each 179 / 222, 64 rows each 204 / 233, 128 rows each 304 / 252, 256 rows each 572 / 324
// The first shares all blocks out to all SMs: a block costs it 0.3 us and 2 ns
// a row, a tile that several SMs share 50 ns a row more in the end.  The second
// does whole tiles of 256 rows x 256 outputs in waves over the pairs of SMs, a
// block in 0.42 us, or 0.55 when most pairs are at work.  The worst choice
// among 90 measured sizes, all of even groups with every row held, takes 1.2
// times as long as the other kernel.
bool pair_is_faster(int64_t T, int groups, int64_t M, int64_t mb, int64_t kb, int sms) {
    const double used = (double)std::min<int64_t>(T, groups), rows = T / used;   // groups with rows, rows of each
    const double blocks = std::ceil(rows / kFp8MaxRows), in_tile = rows / blocks, tiles = used * mb * blocks;
    const double even = tiles * kb / sms;
    double busy, shared = 0;   // blocks of the busiest CTA
    if (tiles > sms) {
        busy = std::min(std::ceil(tiles / sms) * kb, even + 16);
    } else {
        const double each = std::max(1.0, std::floor(sms / tiles));
        busy = std::min(kb / each, even + 8);
        if (each > 1) shared = 8;
    }
    const double one = 5 + (0.30 + 0.0021 * in_tile) * (busy + shared) + (tiles <= sms ? 0.05 * in_tile : 0);
    const double pairs = used * ((M + 255) / 256) * std::ceil(rows / 256), room = sms / 2;
    const double two = 4 + (pairs > room / 2 ? 0.55 : 0.42) * std::ceil(pairs / room) * kb;
    return two < one;
}

int product(const char* what, qrm_fp8* m, bool back, const void* x, int64_t ld_x, const float* xs, int64_t ld_xs,
            const int32_t* offsets, int64_t T, int type, void* out, int64_t ld_out, void* stream) {
    if (!m) return failf(QRM_E_INVALID, "%s: NULL matrix", what);
    const int64_t in = back ? m->rows : m->cols, M = back ? m->cols : m->rows;
    const int b = type_bytes(type);
    if (!b) return failf(QRM_E_FORMAT, "%s: type %d is not F32, F16 or BF16", what, type);
    if (T < 0 || T > INT_MAX) return failf(QRM_E_INVALID, "%s: %lld rows", what, (long long)T);
    const int64_t mb = blocks_of(M), kb = blocks_of(in);
    // (at most one partly filled tile for each group)
    if ((T / kFp8MaxRows + m->groups) * mb > INT_MAX)
        return failf(QRM_E_CAPACITY, "%s: %lld rows in %d groups are too many tiles", what, (long long)T, m->groups);
    if (T == 0) return QRM_OK;
    if (!x || !xs || !out) return failf(QRM_E_INVALID, "%s: NULL argument", what);
    if (!offsets && m->groups > 1) return failf(QRM_E_INVALID, "%s: %d matrices need offsets", what, m->groups);
    if (!pitch_ok(&ld_x, in) || !pitch_ok(&ld_xs, kb) || !pitch_ok(&ld_out, M))
        return failf(QRM_E_INVALID, "%s: a pitch is below its row (x %lld, scales %lld, out %lld)", what, (long long)ld_x,
                     (long long)ld_xs, (long long)ld_out);
    if (!aligned(x, 16) || ld_x % 16)
        return failf(QRM_E_INVALID, "%s: rows of codes must start on 16 bytes (pitch %lld)", what, (long long)ld_x);
    if (!aligned(xs, 4) || !aligned(out, b) || (offsets && !aligned(offsets, 4)))
        return failf(QRM_E_INVALID, "%s: a pointer is not aligned to its values", what);
    DeviceGuard here;
    cudaError_t e = here.enter(m->device);
    if (e != cudaSuccess) return failf(QRM_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
    CUtensorMap x_map;
    const cuuint64_t dims[2] = {(cuuint64_t)in, (cuuint64_t)T};
    const cuuint64_t strides[1] = {(cuuint64_t)ld_x};
    const int wkb = (int)blocks_of(m->cols), wnb = (int)blocks_of(m->rows);
    Fp8Params p{};
    p.w_scales = m->scales;
    p.x_scales = xs;
    p.offsets = offsets;
    p.out = out;
    p.part = m->part;
    p.arrivals = m->arrivals;
    p.err = m->err;
    p.ld_xs = ld_xs;
    p.ld_out = ld_out;
    p.T = (int)T;
    p.groups = m->groups;
    p.M = (int)M;
    p.mb = (int)mb;
    p.kb = (int)kb;
    p.s_group = wnb * wkb;
    p.s_m = back ? 1 : wkb;
    p.s_k = back ? wkb : 1;
    p.back = back;
    p.type = type;
    // the kernel for large groups writes rows that start on 16 bytes
    const bool pair = aligned(out, 16) && ld_out * b % 16 == 0 &&
                      (m->form >= 0 ? m->form : pair_is_faster(T, m->groups, M, mb, kb, m->sms));
    const cuuint32_t box[2] = {128, pair ? 128u : 16u};
    if (!encode(&x_map, x, 2, dims, strides, box)) return failf(QRM_E_CUDA, "%s: tensor map", what);
    if (pair) {
        const int wide_out = aligned(out, 32) && ld_out * b % 32 == 0, wide_xs = aligned(xs, 16) && ld_xs % 4 == 0;
        e = launch_ahead(fp8_pair_kernel, dim3(m->sms / 2 * 2), kFp8Warps * 32, pair_smem(m->groups), (cudaStream_t)stream,
                         back ? m->pair_map_t : m->pair_map, x_map, p, wide_out, wide_xs);
        return e == cudaSuccess ? QRM_OK : failf(QRM_E_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
    }
    const int x_rows = (int)std::min<int64_t>(kFp8MaxRows, (T + 15) / 16 * 16);
    e = launch_ahead(fp8_stream_kernel, dim3(m->sms), kFp8Warps * 32, smem_for(m->groups, x_rows), (cudaStream_t)stream, m->map,
                     x_map, p, stages_for(m->groups, x_rows), x_rows);
    return e == cudaSuccess ? QRM_OK : failf(QRM_E_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" int qrm_fp8_create(int device, int groups, int64_t rows, int64_t cols, const void* codes, size_t code_bytes,
                              const float* scales, size_t scale_bytes, qrm_fp8** out) {
    return create(device, groups, rows, cols, codes, code_bytes, scales, scale_bytes, cudaMemcpyHostToDevice, out);
}

extern "C" int qrm_fp8_create_device(int device, int groups, int64_t rows, int64_t cols, const void* codes_dev,
                                     size_t code_bytes, const float* scales_dev, size_t scale_bytes, qrm_fp8** out) {
    return create(device, groups, rows, cols, codes_dev, code_bytes, scales_dev, scale_bytes, cudaMemcpyDeviceToDevice, out);
}

extern "C" void qrm_fp8_destroy(qrm_fp8* m) { release(m); }

extern "C" int qrm_fp8_product(qrm_fp8* m, const void* x_codes_dev, int64_t ld_x, const float* x_scales_dev,
                               int64_t ld_xs, const int32_t* offsets_dev, int64_t T, int type, void* y_dev, int64_t ld_y,
                               void* stream) {
    return product("qrm_fp8_product", m, false, x_codes_dev, ld_x, x_scales_dev, ld_xs, offsets_dev, T, type, y_dev, ld_y,
                   stream);
}

extern "C" int qrm_fp8_product_t(qrm_fp8* m, const void* y_codes_dev, int64_t ld_y, const float* y_scales_dev,
                                 int64_t ld_ys, const int32_t* offsets_dev, int64_t T, int type, void* x_dev,
                                 int64_t ld_x, void* stream) {
    return product("qrm_fp8_product_t", m, true, y_codes_dev, ld_y, y_scales_dev, ld_ys, offsets_dev, T, type, x_dev, ld_x,
                   stream);
}

extern "C" int qrm_fp8_sync(qrm_fp8* m) {
    if (!m) return failf(QRM_E_INVALID, "qrm_fp8_sync: NULL matrix");
    DeviceGuard here;
    cudaError_t e = here.enter(m->device);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    int32_t err = 0;
    if (e == cudaSuccess) e = cudaMemcpy(&err, m->err, sizeof err, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && err) {
        // a product that gave up may have left counts behind
        e = cudaMemset(m->arrivals, 0, sizeof(int32_t) * (size_t)m->sms * kFp8EpiWarps);
        if (e == cudaSuccess) e = cudaMemset(m->err, 0, sizeof err);
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
    }
    if (e != cudaSuccess) return failf(QRM_E_CUDA, "qrm_fp8_sync: %s", cudaGetErrorString(e));
    if (err & ERR_TIMEOUT) return failf(QRM_E_TIMEOUT, "qrm_fp8_sync: a device wait timed out");
    if (err) return failf(QRM_E_INVALID, "qrm_fp8_sync: offsets do not ascend within the rows (flags 0x%x)", err);
    return QRM_OK;
}
