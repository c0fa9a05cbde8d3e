// fp4.cu -- matrices in 4-bit microscaled floating point, resident in HBM, and
// their products (kernels: fp4.cuh).
#include <stdlib.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <new>

#include "fp4.cuh"
#include "matrix_host.h"

using namespace qrm;

struct qrm_fp4 {
    int device = 0, sms = 0, groups = 0;
    int form = -1;                       // QRM_FP4_PAIR: 1 always / 0 never rows of x on the MMA's M side
    int64_t rows = 0, cols = 0;
    int units = 0, gated_units = 0;      // of 128 rows; of 64 features, if there are two halves
    int steps = 0;                       // of 256 columns
    uint8_t* codes = nullptr;            // [groups][rows][whole blocks of 16 bytes]; the other arrays are in the same allocation
    uint8_t* scales = nullptr;           // [groups][units][steps][2][512]
    uint8_t* gated_scales = nullptr;     // [groups][gated_units][steps][2][512]
    int32_t* err = nullptr;
    // codes in boxes of 256 columns x 128 rows (gated: 64 features, in turns of 16); scales in boxes of a unit's for one stage
    CUtensorMap map, gated_map, scales_map, gated_scales_map;
};

namespace {

int64_t blocks_of(int64_t n) { return (n + kFp4Block - 1) / kFp4Block; }

void release(qrm_fp4* m) {
    if (!m) return;
    DeviceGuard here;
    here.enter(m->device);
    cudaDeviceSynchronize();
    cudaFree(m->codes);
    delete m;
}

size_t pair_smem(int groups) { return 1024 + (size_t)fp4_pair_stage_off(groups) + (size_t)kFp4PairStages * kFp4PairStage + 8 * kFp4PairOut; }
size_t tail_smem(int groups, int stages) { return 1024 + (size_t)fp4_pair_stage_off(groups) + (size_t)stages * kFp4TailStage + kFp4TailRoom; }
constexpr int kSmemStatic = 512;   // more than the kernels' own
int tail_stages(int groups) { return tail_smem(groups, kFp4TailStages) <= kSmemMost - kSmemStatic ? kFp4TailStages : kFp4TailStages - 1; }

template <int MODE>
cudaError_t prepare_kernels() {
    cudaError_t e = cudaFuncSetAttribute(fp4_split_kernel<MODE, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fp4_split_kernel<MODE, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(fp4_pair_kernel<MODE, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pair_smem(kFp4MaxGroups));
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(fp4_pair_kernel<MODE, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost - kSmemStatic);
    return e;
}
// registers a thread that the pair kernels were built with: their split may not pass what a launch has
template <int MODE>
bool enough_regs() {
    cudaFuncAttributes pair{}, tails{};
    return cudaFuncGetAttributes(&pair, fp4_pair_kernel<MODE, false>) == cudaSuccess && pair.numRegs * kFp4PairThreads >= kFp4PairRegs &&
           cudaFuncGetAttributes(&tails, fp4_pair_kernel<MODE, true>) == cudaSuccess && tails.numRegs * kFp4PairThreads >= kFp4PairRegs;
}

int create(int device, int groups, int64_t rows, int64_t cols, const void* codes, size_t code_bytes, const void* scales,
           size_t scale_bytes, cudaMemcpyKind kind, qrm_fp4** out) {
    const char* what = "qrm_fp4_create";
    if (!out) return failf(QRM_E_INVALID, "%s: out is NULL", what);
    *out = nullptr;
    if (!codes || !scales) return failf(QRM_E_INVALID, "%s: NULL argument", what);
    if (groups <= 0 || rows <= 0 || cols <= 0 || rows > (1 << 22) || cols > (1 << 24))
        return failf(QRM_E_INVALID, "%s: %d matrices of %lld x %lld", what, groups, (long long)rows, (long long)cols);
    if (groups > kFp4MaxGroups) return failf(QRM_E_CAPACITY, "%s: %d matrices, at most %d", what, groups, kFp4MaxGroups);
    const int64_t blocks = blocks_of(cols), all = groups * rows;
    if (code_bytes != (size_t)(all * blocks * 16))
        return failf(QRM_E_SIZE, "%s: %zu bytes of codes, %d x %lld rows of %lld blocks of 16 is %lld", what, code_bytes, groups,
                     (long long)rows, (long long)blocks, (long long)(all * blocks * 16));
    if (scale_bytes != (size_t)(all * blocks))
        return failf(QRM_E_SIZE, "%s: %zu bytes of scales, one for each of %lld blocks", what, scale_bytes, (long long)(all * blocks));
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
    qrm_fp4* m = new (std::nothrow) qrm_fp4();
    if (!m) return failf(QRM_E_NOMEM, "%s: host memory", what);
    auto bail = [&](int rc) {
        release(m);
        return rc;
    };
    if (const char* e = getenv("QRM_FP4_PAIR")) m->form = atoi(e) != 0;
    m->device = device;
    m->sms = sms;
    m->groups = groups;
    m->rows = rows;
    m->cols = cols;
    m->units = (int)((rows + 127) / 128);
    m->steps = (int)((cols + kFp4Step - 1) / kFp4Step);
    const int f = rows % 2 ? 0 : (int)(rows / 2);
    m->gated_units = (f + 63) / 64;
    // one allocation: codes, scales in both orders, the error flags
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t stage = (size_t)m->steps * kFp4Scales, pitch = (size_t)blocks * 16;
    // (the gated map's last sixteen features may reach 15 rows past the last matrix)
    const size_t scales_at = up(code_bytes + 16 * pitch), gated_at = scales_at + (size_t)groups * m->units * stage;
    const size_t err_at = gated_at + (size_t)groups * m->gated_units * stage;
    uint8_t* staged = nullptr;   // the scales as they came, until they are in units
    if (cudaMalloc(&m->codes, err_at + 256) != cudaSuccess || cudaMalloc(&staged, scale_bytes) != cudaSuccess) {
        cudaGetLastError();
        return bail(failf(QRM_E_NOMEM, "%s: cannot allocate %zu bytes", what, err_at + 256 + scale_bytes));
    }
    m->scales = m->codes + scales_at;
    m->gated_scales = m->codes + gated_at;
    m->err = reinterpret_cast<int32_t*>(m->codes + err_at);
    // device sources: what any stream still writes there is awaited, on their own device if that is another one
    cudaError_t e = cudaDeviceSynchronize();
    if (kind == cudaMemcpyDeviceToDevice) {
        if (e == cudaSuccess) e = await_source(codes, device);
        if (e == cudaSuccess) e = await_source(scales, device);
    }
    if (e == cudaSuccess) e = cudaMemcpy(m->codes, codes, code_bytes, kind);
    if (e == cudaSuccess) e = cudaMemcpy(staged, scales, scale_bytes, kind);
    if (e == cudaSuccess) e = cudaMemset(m->err, 0, sizeof(int32_t));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e == cudaSuccess && cols % kFp4Block)
        e = launch_ahead(fp4_clear_tail_kernel, dim3((unsigned)((all + 255) / 256)), 256, 0, nullptr, m->codes, all, (int)cols, (int)pitch);
    if (e == cudaSuccess)
        e = launch_ahead(fp4_scale_units_kernel, dim3(2 * m->steps, m->units, groups), 128, 0, nullptr, staged, (int)rows, (int)blocks,
                         0, m->units, m->steps, reinterpret_cast<uint32_t*>(m->scales));
    if (e == cudaSuccess && f)
        e = launch_ahead(fp4_scale_units_kernel, dim3(2 * m->steps, m->gated_units, groups), 128, 0, nullptr, staged, (int)rows,
                         (int)blocks, f, m->gated_units, m->steps, reinterpret_cast<uint32_t*>(m->gated_scales));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    cudaFree(staged);
    if (e == cudaSuccess) e = prepare_kernels<kFp4Plain>();
    if (e == cudaSuccess) e = prepare_kernels<kFp4Gated>();
    if (e == cudaSuccess) e = prepare_kernels<kFp4GatedRows>();
    if (e != cudaSuccess) return bail(failf(QRM_E_CUDA, "%s: %s", what, cudaGetErrorString(e)));
    if (!enough_regs<kFp4Plain>() || !enough_regs<kFp4Gated>() || !enough_regs<kFp4GatedRows>())
        return bail(failf(QRM_E_CUDA, "%s: built with too few registers a thread for their split", what));
    const cuuint64_t dims[3] = {(cuuint64_t)pitch, (cuuint64_t)rows, (cuuint64_t)groups};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch, (cuuint64_t)(pitch * rows)};
    const cuuint32_t box[3] = {128, 128, 1}, gated_box[5] = {128, 16, 2, 4, 1}, unit_box[2] = {256, kFp4Scales / 256};
    const cuuint64_t by_gate[5] = {(cuuint64_t)pitch, 16, 2, (cuuint64_t)(f + 15) / 16, (cuuint64_t)groups};
    const cuuint64_t by_gate_strides[4] = {(cuuint64_t)pitch, (cuuint64_t)(pitch * f), (cuuint64_t)(pitch * 16), (cuuint64_t)(pitch * rows)};
    const cuuint64_t unit_strides[1] = {256};
    const cuuint64_t unit_dims[2] = {256, (cuuint64_t)groups * m->units * stage / 256};
    const cuuint64_t gated_dims[2] = {256, (cuuint64_t)groups * m->gated_units * stage / 256};
    if (!encode(&m->map, m->codes, 3, dims, strides, box) || (f && !encode(&m->gated_map, m->codes, 5, by_gate, by_gate_strides, gated_box)) ||
        !encode(&m->scales_map, m->scales, 2, unit_dims, unit_strides, unit_box, CU_TENSOR_MAP_SWIZZLE_NONE) ||
        (f && !encode(&m->gated_scales_map, m->gated_scales, 2, gated_dims, unit_strides, unit_box, CU_TENSOR_MAP_SWIZZLE_NONE)))
        return bail(failf(QRM_E_CUDA, "%s: tensor map", what));
    *out = m;
    return QRM_OK;
}

// Which kernel a product takes, by an estimate of what both would cost with all
// T rows held and spread evenly over the groups: a call that passes room for more
// rows than its groups have is judged by the room, which the host knows, not by
// the offsets.  Measured (us, graphs of ten calls in bursts, matrices that no cache
// holds; weights / rows of x on the MMA's M side), outputs x contracted:
//   1 x 4096 x 7168:   1 row 8.4 / 15.4, 16 rows 9.7 / 15.2, 64 rows 13.1 / 15.8, 128 rows 14.7 / 16.2, 256 rows 15.4 / 16.6
//   1 x 28672 x 4096:  1 row 12.9 / 26.4, 32 rows 16.4 / 20.7, 64 rows 19.9 / 20.7, 128 rows 27.6 / 21.7
//   1 x 1024 x 2816:   1 row 5.5 / 8.3, 32 rows 7.7 / 8.8, 64 rows 10.0 / 9.2
//   1 x 7168 x 2048:   16 rows 6.8 / 8.8, 32 rows 8.0 / 9.0, 64 rows 10.4 / 9.0
//   8 x 5632 x 1024:   8 rows each 10.6 / 12.5, 16 rows each 12.3 / 13.1, 32 rows each 14.9 / 13.7
//   32 x 4096 x 7168:  2 rows each 73 / 90, 16 rows each 87 / 100, 32 rows each 101 / 102, 64 rows each 112 / 105
//   32 x 7168 x 2048:  4 rows each 48 / 53, 16 rows each 59 / 57, 64 rows each 79 / 60
// (Grouped, under sustained load: 32 x 4096 x 7168 75 / 105, 89 / 117, 104 / 120,
// 119 / 123; 32 x 7168 x 2048 48 / 63, 59 / 68, 79 / 72.)  The first takes what
// reading the weights takes, and something for each row of a tile and all tiles'
// rows; the second a time for each stage of whole tiles of 256 rows x 256 outputs,
// in waves over the pairs of SMs, longer where most pairs are at work.  The worst
// choice among these sizes takes 1.08 times as long as the other kernel in bursts
// and 1.09 times under load (256 rows through 4096 x 7168, both).
bool pair_is_faster(int64_t T, int64_t used, int64_t tiles_across, int steps, int tile_rows, int sms) {
    const double rows = (double)T / used, row_tiles = std::ceil(rows / tile_rows), tiles = used * tiles_across * row_tiles;
    const double read = (double)used * tiles_across * steps * 34816 / 6.4e6;   // us, of a stage's 256 x 256 codes and scales
    const double one = 4 + read * (1 + (row_tiles - 1) / 2) + std::min<double>(rows, tile_rows) * (0.07 + 0.0004 * tiles);
    const double pairs = sms / 2, wide = used * tiles_across * std::ceil(rows / 256);
    const double two = 5.5 + std::ceil(wide / pairs) * steps * (wide <= pairs / 2 ? 0.3 : 0.45);
    return two < one;
}

template <int MODE>
cudaError_t launch(const qrm_fp4* m, const CUtensorMap& x_map, const CUtensorMap& few_map, const Fp4Params& p, bool pair, int wide_out, int64_t T, cudaStream_t s) {
    const CUtensorMap& w_map = MODE == kFp4Plain ? m->map : m->gated_map;
    if (pair) {
        // Tails (a sixth more shared memory a stage, smaller pieces on the way out) where groups are likely to have one and a
        // tile has stages enough.  With and without, us in bursts, the mean of three draws of uneven groups: 32 x 4096 x 7168,
        // 8192 rows 142 / 148, 9000 rows 149 / 164, 12000 rows 188 / 202; 32 x 7168 x 2048, 8192 rows 85 / 87; 64 x 4096 x 2048,
        // 20000 rows 113 / 120; 20 x 3584 x 2816, 7000 rows 50.1 / 50.0; 8 x 5632 x 2048, 2560 rows 26.1 / 25.7; where the rule
        // takes none, 8 x 5632 x 1024, 512 rows 15.2 / 13.8, 20 x f 1536 x 6144 gated, 2559 rows 54.9 / 52.9.  A single draw may go the other way, since what counts is whether the tiles saved are a wave over the pairs: the worst one seen
        // took 1.08 times as long with tails (7000 rows over 20 x 3584 x 2816).
        const bool tails = m->groups > 1 && T > (int64_t)128 * m->groups && p.steps >= 8;
        const int stages = tails ? tail_stages(m->groups) : kFp4PairStages;
        return launch_ahead(tails ? fp4_pair_kernel<MODE, true> : fp4_pair_kernel<MODE, false>, dim3(m->sms / 2 * 2), kFp4PairThreads,
                            tails ? tail_smem(m->groups, stages) : pair_smem(m->groups), s, w_map,
                            MODE == kFp4Plain ? m->scales_map : m->gated_scales_map, x_map, few_map, p, wide_out, stages);
    }
    const int64_t across = p.across;
    const int64_t used = std::min<int64_t>(T, m->groups), per = (T / used + p.tile_rows - 1) / p.tile_rows;
    const int64_t tiles = used * per * across;
    int ranks = 1;
    while (ranks < 8 && tiles * ranks * 2 <= 2 * m->sms && p.steps >= 4 * ranks) ranks *= 2;
    const int64_t ctas = (int64_t)p.row_tiles * across * ranks;
    // two CTAs on an SM, 1 KB of it kept for each: of one launch, or the next one's first
    const int stages = std::min(kFp4MaxStages, (kSmemMost / 2 - 512 - 1024 - kFp4Header) / fp4_stage_bytes(p.tile_rows));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kFp4Threads);
    cfg.dynamicSmemBytes = 1024 + kFp4Header + (size_t)stages * fp4_stage_bytes(p.tile_rows);
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // as in launch_ahead
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, p.groups > 1 ? fp4_split_kernel<MODE, true> : fp4_split_kernel<MODE, false>, w_map, few_map, p, stages);
}

constexpr int64_t kMostRows = INT_MAX - 1023;   // the end of the last one's tile fits in 32 bits

int product(const char* what, int mode, qrm_fp4* m, const void* x, int64_t ld_x, const uint8_t* xs, int64_t ld_xs,
            const int32_t* offsets, int64_t T, float limit, int type, void* out, int64_t ld_out, uint8_t* out_scales,
            int64_t ld_os, void* stream) {
    if (!m) return failf(QRM_E_INVALID, "%s: NULL matrix", what);
    if (mode != kFp4Plain && m->rows % 2) return failf(QRM_E_INVALID, "%s: %lld rows are no two halves", what, (long long)m->rows);
    const int64_t M = mode == kFp4Plain ? m->rows : m->rows / 2, blocks = blocks_of(m->cols);
    const int b = mode == kFp4GatedRows ? 1 : type_bytes(type);
    if (!b) return failf(QRM_E_FORMAT, "%s: type %d is not F32, F16 or BF16", what, type);
    if (!(limit >= 0.f)) return failf(QRM_E_INVALID, "%s: limit %g", what, (double)limit);
    if (T < 0 || T > kMostRows) return failf(QRM_E_INVALID, "%s: %lld rows", what, (long long)T);
    // rows of x in a tile of the kernel with weights on the M side: a third more than a group has on average, so that most
    // groups take one tile and a stage stays small
    const int64_t used = std::max<int64_t>(1, std::min<int64_t>(T, m->groups)), each = (T + used - 1) / used;
    const int tile_rows = (int)std::max<int64_t>(16, std::min<int64_t>(kFp4Rows, ((m->groups > 1 ? each * 4 / 3 : each) + 15) / 16 * 16));
    const int64_t across = (M + 127) / 128, row_tiles = T / tile_rows + used;
    if (row_tiles * across > INT_MAX / 8)
        return failf(QRM_E_CAPACITY, "%s: %lld rows in %d groups are too many tiles", what, (long long)T, m->groups);
    if (T == 0) return QRM_OK;
    if (!x || !xs || !out) return failf(QRM_E_INVALID, "%s: NULL argument", what);
    if (!offsets && m->groups > 1) return failf(QRM_E_INVALID, "%s: %d matrices need offsets", what, m->groups);
    const int64_t out_cols = mode == kFp4GatedRows ? 16 * blocks_of(M) : M;
    if (!pitch_ok(&ld_x, 16 * blocks) || !pitch_ok(&ld_xs, blocks) || !pitch_ok(&ld_out, out_cols))
        return failf(QRM_E_INVALID, "%s: a pitch is below its row (x %lld, scales %lld, out %lld)", what, (long long)ld_x,
                     (long long)ld_xs, (long long)ld_out);
    if (!aligned(x, 16) || ld_x % 16)
        return failf(QRM_E_INVALID, "%s: rows of codes must start on 16 bytes (pitch %lld)", what, (long long)ld_x);
    if (!aligned(out, b) || (offsets && !aligned(offsets, 4)))
        return failf(QRM_E_INVALID, "%s: a pointer is not aligned to its values", what);
    if (mode == kFp4GatedRows) {
        if (!out_scales) return failf(QRM_E_INVALID, "%s: NULL argument", what);
        if (!pitch_ok(&ld_os, blocks_of(M)))
            return failf(QRM_E_INVALID, "%s: a pitch is below its row (scales %lld)", what, (long long)ld_os);
        if (!aligned(out, 16) || ld_out % 16)
            return failf(QRM_E_INVALID, "%s: rows of codes must start on 16 bytes (pitch %lld)", what, (long long)ld_out);
    }
    DeviceGuard here;
    cudaError_t e = here.enter(m->device);
    if (e != cudaSuccess) return failf(QRM_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
    const bool pair = m->form >= 0 ? m->form : pair_is_faster(T, used, mode == kFp4Plain ? (M + 255) / 256 : across, m->steps, tile_rows, m->sms);
    const int wide_out = aligned(out, 16) && ld_out * b % 16 == 0;
    CUtensorMap x_map, few_map;   // in boxes of 128 rows; of half a tail's, or (weights on the M side) of 16
    const cuuint64_t dims[2] = {(cuuint64_t)(16 * blocks), (cuuint64_t)T};
    const cuuint64_t strides[1] = {(cuuint64_t)ld_x};
    const cuuint32_t box[2] = {128, 128}, few[2] = {128, pair ? kFp4TailRows / 2u : 16u};
    if ((pair && !encode(&x_map, x, 2, dims, strides, box)) || !encode(&few_map, x, 2, dims, strides, few)) return failf(QRM_E_CUDA, "%s: tensor map", what);
    Fp4Params p{};
    p.w_scales = mode == kFp4Plain ? m->scales : m->gated_scales;
    p.x_scales = xs;
    p.offsets = offsets;
    p.out = out;
    p.out_scales = out_scales;
    p.err = m->err;
    p.ld_xs = ld_xs;
    p.ld_out = ld_out;
    p.ld_os = ld_os;
    p.limit = limit > 0.f ? limit : INFINITY;
    p.T = (int)T;
    p.groups = m->groups;
    p.M = (int)M;
    p.units = mode == kFp4Plain ? m->units : m->gated_units;
    p.steps = m->steps;
    p.blocks = (int)blocks;
    p.type = type;
    p.tile_rows = tile_rows;
    p.across = (int)(mode == kFp4Plain ? (M + 255) / 256 : across);
    p.row_tiles = (int)(m->groups > 1 ? row_tiles : (T + tile_rows - 1) / tile_rows);
    p.wide_xs = aligned(xs, 16) && ld_xs % 16 == 0 ? 2 : aligned(xs, 8) && ld_xs % 8 == 0 ? 1 : 0;
    const cudaStream_t s = (cudaStream_t)stream;
    e = mode == kFp4Plain   ? launch<kFp4Plain>(m, x_map, few_map, p, pair, wide_out, T, s)
        : mode == kFp4Gated ? launch<kFp4Gated>(m, x_map, few_map, p, pair, wide_out, T, s)
                            : launch<kFp4GatedRows>(m, x_map, few_map, p, pair, wide_out, T, s);
    return e == cudaSuccess ? QRM_OK : failf(QRM_E_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" int qrm_fp4_create(int device, int groups, int64_t rows, int64_t cols, const void* codes, size_t code_bytes,
                              const void* scales, size_t scale_bytes, qrm_fp4** out) {
    return create(device, groups, rows, cols, codes, code_bytes, scales, scale_bytes, cudaMemcpyHostToDevice, out);
}

extern "C" int qrm_fp4_create_device(int device, int groups, int64_t rows, int64_t cols, const void* codes_dev,
                                     size_t code_bytes, const void* scales_dev, size_t scale_bytes, qrm_fp4** out) {
    return create(device, groups, rows, cols, codes_dev, code_bytes, scales_dev, scale_bytes, cudaMemcpyDeviceToDevice, out);
}

extern "C" void qrm_fp4_destroy(qrm_fp4* m) { release(m); }

extern "C" int qrm_fp4_product(qrm_fp4* m, const void* x_codes_dev, int64_t ld_x, const uint8_t* x_scales_dev,
                               int64_t ld_xs, const int32_t* offsets_dev, int64_t T, int type, void* y_dev, int64_t ld_y,
                               void* stream) {
    return product("qrm_fp4_product", kFp4Plain, m, x_codes_dev, ld_x, x_scales_dev, ld_xs, offsets_dev, T, 0.f, type, y_dev,
                   ld_y, nullptr, 0, stream);
}

extern "C" int qrm_fp4_swiglu(qrm_fp4* m, const void* x_codes_dev, int64_t ld_x, const uint8_t* x_scales_dev,
                              int64_t ld_xs, const int32_t* offsets_dev, int64_t T, float limit, int type, void* h_dev,
                              int64_t ld_h, void* stream) {
    return product("qrm_fp4_swiglu", kFp4Gated, m, x_codes_dev, ld_x, x_scales_dev, ld_xs, offsets_dev, T, limit, type, h_dev,
                   ld_h, nullptr, 0, stream);
}

extern "C" int qrm_fp4_swiglu_fp4(qrm_fp4* m, const void* x_codes_dev, int64_t ld_x, const uint8_t* x_scales_dev,
                                  int64_t ld_xs, const int32_t* offsets_dev, int64_t T, float limit, uint8_t* codes_dev,
                                  int64_t ld_codes, uint8_t* scales_dev, int64_t ld_scales, void* stream) {
    return product("qrm_fp4_swiglu_fp4", kFp4GatedRows, m, x_codes_dev, ld_x, x_scales_dev, ld_xs, offsets_dev, T, limit,
                   QRM_F32, codes_dev, ld_codes, scales_dev, ld_scales, stream);
}

extern "C" int qrm_fp4_sync(qrm_fp4* m) {
    if (!m) return failf(QRM_E_INVALID, "qrm_fp4_sync: NULL matrix");
    DeviceGuard here;
    cudaError_t e = here.enter(m->device);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    int32_t err = 0;
    if (e == cudaSuccess) e = cudaMemcpy(&err, m->err, sizeof err, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && err) {
        e = cudaMemset(m->err, 0, sizeof err);
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
    }
    if (e != cudaSuccess) return failf(QRM_E_CUDA, "qrm_fp4_sync: %s", cudaGetErrorString(e));
    if (err & ERR_TIMEOUT) return failf(QRM_E_TIMEOUT, "qrm_fp4_sync: a device wait timed out");
    if (err) return failf(QRM_E_INVALID, "qrm_fp4_sync: offsets do not ascend within the rows (flags 0x%x)", err);
    return QRM_OK;
}
