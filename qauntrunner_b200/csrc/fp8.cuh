// fp8.cuh -- product of 8-bit rows with 8-bit matrices that carry a scale for
// each block of 128: dense, or grouped (rows of group g times matrix g).
//
//   y[t][m] = sum_b sx[t][b] sw[m/128][b] * sum_{c in block b} qx[t][c] qw[m][c]
//
// with blocks of 128 along the contracted dimension.  The inner sums are
// tcgen05.mma (kind::f8f6f4, e4m3 x e4m3) into f32 tensor memory, a fresh
// accumulator per block; the outer sum is one f32 FMA per value and block in
// the epilogue warps' registers.  The transposed product (the input gradient,
// y = W^T x) reads the same stored matrix: its tiles enter the MMA with M as
// their contiguous dimension instead of K, and the scales' two block indices
// change places.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "gemv_imma.cuh"
#include "umma_ptx.cuh"

namespace qrm {

constexpr int kFp8MaxGroups = 1024;

struct Fp8Params {
    const float* w_scales;    // [groups][ceil(N/128)][ceil(K/128)]
    const float* x_scales;    // [T][ld_xs]
    const int32_t* offsets;   // [groups+1] rows of each group, or NULL (one group)
    void* out;                // [T][ld_out]
    float* part;              // partial tiles: [CTA][2][rows of x in a tile][128]
    int32_t* arrivals;        // [CTA][warps]
    int32_t* err;
    long long ld_xs, ld_out;
    int T, groups;
    int M;                    // length of an output row
    int mb, kb;               // blocks of 128 in it, and of the contracted dimension
    int s_group, s_m, s_k;    // strides of w_scales: matrix, block of M, contracted block
    int back;                 // the transposed product
    int type;                 // of out
};

// Shared-memory matrix descriptor of an operand whose M (or N) dimension is
// contiguous, 128-byte swizzle: 128 values of M a row, 8 contracted rows a
// swizzle atom of 1024 bytes (stride byte offset between the atoms), one atom
// wide (`wide_stride` apart when there are several).
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t wide_stride) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(wide_stride >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor of kind::f8f6f4: f32 accumulators, e4m3 A and B,
// M = 128; a_mn / b_mn: the operand is contiguous along M / N, not K.
__device__ __forceinline__ uint32_t umma_idesc_e4m3(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
// D[tmem] (+)= A[smem] * B[smem]^T over 32 contracted values
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
// 16 / 32 columns of this warp's 32 tensor-memory lanes; the wait is part of
// the statement, so nothing that uses the registers can move before it
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void store_typed(void* out, long long i, float v, int type) {
    if (type == 0) reinterpret_cast<float*>(out)[i] = v;
    else if (type == 1) reinterpret_cast<__half*>(out)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// ------------------------------------------------------------ weights on the MMA's M side
// A tile is 128 outputs (one block row of the matrix, the MMA's M) x up to 128
// rows of x (its N, rounded up to 16 only), so a group of a few rows costs
// about what its weights cost to read: this form is for memory-bound sizes.
//
// All tiles' blocks, one after the other, are cut into as many equal runs as
// there are CTAs (one per SM), wherever that falls inside a tile: one token
// through one matrix still reads it with every SM.  A CTA that did only part
// of a tile's blocks leaves its f32 sums in the workspace, and the last one to
// arrive adds the parts up in the CTAs' order, so that the result does not
// depend on who was last.  Nobody waits.
//
// Warps: 0 loads tiles (TMA), 1 issues the MMAs, 2 brings the scales (their
// product sx sw for each row of x and block), 4-11 add up: lane quarter
// (warp & 3) x 64 of the tile's rows of x.
constexpr int kFp8Warps = 12;
constexpr int kFp8EpiWarp0 = 4;
constexpr int kFp8EpiWarps = 8;
constexpr int kFp8Tile = 128 * 128;     // bytes of a weight tile
constexpr int kFp8MaxRows = 128;        // rows of x in a tile
constexpr int kFp8Acc = 4;              // accumulators in tensor memory
constexpr int kFp8ScaleRing = 16;
constexpr int kFp8MaxStages = 12;
constexpr int kFp8ScaleOff = 1024;                                       // after the barriers
constexpr int kFp8TableOff = kFp8ScaleOff + kFp8ScaleRing * kFp8MaxRows * 4;
__host__ __device__ inline int fp8_stage_off(int groups) { return (kFp8TableOff + 12 * (groups + 1) + 1023) / 1024 * 1024; }

// What a CTA does: blocks [q, q_end) of the sequence (tile, block).
struct Fp8Piece {
    int tile;        // number of the tile
    int k0, k1;      // its blocks of this CTA
    int group, m;    // matrix, block of 128 outputs
    int pos, n;      // first row of x, rows
};

struct Fp8Plan {
    const int32_t* first_tile;   // [groups+1]
    const int32_t* start;        // [groups] first row of x
    const int32_t* rows;         // [groups]
    int groups, mb, kb;
    long long total;             // blocks of all tiles
    int ctas;                    // that share them, at most `total`
    __device__ long long cut(int c) const { return total * c / ctas; }
    // the CTA whose run holds block q
    __device__ int owner(long long q) const { return (int)(((q + 1) * ctas - 1) / total); }
    __device__ Fp8Piece piece(long long q, long long q_end) const {
        Fp8Piece r;
        r.tile = (int)(q / kb);
        r.k0 = (int)(q - (long long)r.tile * kb);
        const long long left = q_end - q;
        r.k1 = left < kb - r.k0 ? r.k0 + (int)left : kb;
        int lo = 0, hi = groups;   // the last group with first_tile <= tile has rows
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first_tile[mid] <= r.tile) lo = mid;
            else hi = mid;
        }
        r.group = lo;
        const int blocks = (rows[lo] + kFp8MaxRows - 1) / kFp8MaxRows;
        const int per = ((rows[lo] + blocks - 1) / blocks + 15) & ~15;
        const int in = r.tile - first_tile[lo];
        r.m = in / blocks;
        const int at = (in - r.m * blocks) * per;
        r.pos = start[lo] + at;
        r.n = min(per, rows[lo] - at);
        return r;
    }
};

// The groups' tables in shared memory, by one warp; the caller synchronises.
// Offsets that do not ascend within [0, T] make a group empty and raise an
// error: no row outside x or out is ever touched.
__device__ inline void fp8_tables(const Fp8Params& p, int32_t* first_tile, int32_t* start, int32_t* rows, bool report) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    bool bad = false;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + lane;
        int a = 0, b = 0;
        if (g < p.groups) {
            a = p.offsets ? p.offsets[g] : 0;
            b = p.offsets ? p.offsets[g + 1] : p.T;
            if (a < 0 || b < a || b > p.T) {
                bad = true;
                a = b = 0;
            }
        }
        const int tiles = (b - a + kFp8MaxRows - 1) / kFp8MaxRows * p.mb;
        int scan = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (g < p.groups) {
            first_tile[g] = before + scan - tiles;
            start[g] = a;
            rows[g] = b - a;
        }
        before += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (lane == 0) first_tile[p.groups] = before;
    if (__any_sync(0xffffffffu, bad) && report && lane == 0) atomicOr(p.err, (int)ERR_BOUNDS);
}

__global__ void __launch_bounds__(kFp8Warps * 32, 1)
fp8_stream_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, Fp8Params p,
                  int stages, int x_rows /* room for rows of x in a stage */) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm);          // [stages]
    uint64_t* empty = full + kFp8MaxStages;
    uint64_t* acc_full = empty + kFp8MaxStages;                // [kFp8Acc]
    uint64_t* acc_empty = acc_full + kFp8Acc;
    uint64_t* sc_full = acc_empty + kFp8Acc;                   // [kFp8ScaleRing]
    uint64_t* sc_empty = sc_full + kFp8ScaleRing;
    uint64_t* done_bar = sc_empty + kFp8ScaleRing;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + 768);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + 776);
    float* sc_ring = reinterpret_cast<float*>(sm + kFp8ScaleOff);
    int32_t* first_tile = reinterpret_cast<int32_t*>(sm + kFp8TableOff);
    int32_t* start = first_tile + p.groups + 1;
    int32_t* rows = start + p.groups + 1;
    const int stage_off = fp8_stage_off(p.groups), stage_bytes = kFp8Tile + x_rows * 128;
    uint8_t* ring = sm + stage_off;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < kFp8Acc; i++) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], kFp8EpiWarps);
        }
        for (int i = 0; i < kFp8ScaleRing; i++) {
            mbar_init(&sc_full[i], 1);
            mbar_init(&sc_empty[i], kFp8EpiWarps);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 512);
    if (warp == 2) fp8_tables(p, first_tile, start, rows, blockIdx.x == 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    Fp8Plan plan{first_tile, start, rows, p.groups, p.mb, p.kb, (long long)first_tile[p.groups] * p.kb, 0};
    plan.ctas = (int)min((long long)gridDim.x, plan.total);   // each has a block at least
    const bool idle = (int)blockIdx.x >= plan.ctas;
    const long long q0 = idle ? 0 : plan.cut(blockIdx.x), q1 = idle ? 0 : plan.cut(blockIdx.x + 1);

    if (warp == 0) {
        // ------------------------------------------------ tiles
        bool ok = true;
        uint32_t i = 0;
        for (long long q = q0; q < q1 && ok;) {
            const Fp8Piece t = plan.piece(q, q1);
            const int boxes = (t.n + 15) >> 4;
            for (int kb = t.k0; kb < t.k1; kb++, i++) {
                const int s = i % stages;
                if (i >= (uint32_t)stages) {
                    const bool w = lane == 0 ? mbar_wait_abort(&empty[s], ((i / stages) & 1u) ^ 1u, abort_flag) : true;
                    if (!__shfl_sync(0xffffffffu, (int)w, 0)) { ok = false; break; }
                }
                uint8_t* st = ring + (size_t)s * stage_bytes;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&full[s], (uint32_t)(kFp8Tile + boxes * 2048));
                    if (p.back) tma_load_3d(st, &w_map, t.m * 128, kb * 128, t.group, &full[s]);
                    else tma_load_3d(st, &w_map, kb * 128, t.m * 128, t.group, &full[s]);
                }
                __syncwarp();
                if (lane < boxes) tma_load_2d(st + kFp8Tile + lane * 2048, &x_map, kb * 128, t.pos + 16 * lane, &full[s]);
            }
            q += t.k1 - t.k0;
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            atomicOr(p.err, (int)ERR_TIMEOUT);
            // copies already issued must land before the CTA exits
            for (uint32_t j = i > (uint32_t)stages ? i - stages : 0; j < i; j++) mbar_wait(&full[j % stages], (j / stages) & 1u);
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMAs (one thread)
        if (lane == 0) {
            bool ok = true;
            uint32_t i = 0;
            for (long long q = q0; q < q1 && ok;) {
                const Fp8Piece t = plan.piece(q, q1);
                const uint32_t idesc = umma_idesc_e4m3((t.n + 15) & ~15, p.back, false);
                for (int kb = t.k0; kb < t.k1; kb++, i++) {
                    const int s = i % stages, b = i % kFp8Acc;
                    if ((i >= kFp8Acc && !mbar_wait_abort(&acc_empty[b], ((i / kFp8Acc) & 1u) ^ 1u, abort_flag)) ||
                        !mbar_wait_abort(&full[s], (i / stages) & 1u, abort_flag)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t a = smem_u32(ring + (size_t)s * stage_bytes), x = a + kFp8Tile;
#pragma unroll
                    for (int c = 0; c < 4; c++)   // 32 contracted values: 32 bytes along K, or 32 rows of 128 bytes
                        umma_f8(tmem + 128 * b, p.back ? sw128_desc_mn(a + 4096 * c, kFp8Tile) : sw128_desc(a + 32 * c),
                                sw128_desc(x + 32 * c), idesc, c ? 1u : 0u);
                    umma_commit(&empty[s]);
                    umma_commit(&acc_full[b]);
                }
                q += t.k1 - t.k0;
            }
            if (!ok) {
                *abort_flag = 1;
                atomicOr(p.err, (int)ERR_TIMEOUT);
            }
            // every MMA of this CTA has completed before tensor memory is released
            umma_commit(done_bar);
            mbar_wait(done_bar, 0u);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------ scales, four blocks' loads at a time
        bool ok = true;
        uint32_t i = 0;
        for (long long q = q0; q < q1 && ok;) {
            const Fp8Piece t = plan.piece(q, q1);
            const float* ws = p.w_scales + (long long)t.group * p.s_group + (long long)t.m * p.s_m;
            const float* xs = p.x_scales + (long long)t.pos * p.ld_xs;
            for (int k4 = t.k0; k4 < t.k1 && ok; k4 += 4) {
                float v[4][4], w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int kb = k4 + j;
                    w[j] = kb < t.k1 ? __ldg(ws + (long long)kb * p.s_k) : 0.f;
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        v[j][r] = kb < t.k1 && lane + 32 * r < t.n ? __ldg(xs + (lane + 32 * r) * p.ld_xs + kb) : 0.f;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (k4 + j >= t.k1) break;
                    const int s = i % kFp8ScaleRing;
                    if (i >= kFp8ScaleRing &&
                        !warp_wait(&sc_empty[s], ((i / kFp8ScaleRing) & 1u) ^ 1u, abort_flag, p.err)) { ok = false; break; }
#pragma unroll
                    for (int r = 0; r < 4; r++) sc_ring[s * kFp8MaxRows + lane + 32 * r] = v[j][r] * w[j];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[s]);
                    i++;
                }
            }
            q += t.k1 - t.k0;
        }
    } else if (warp >= kFp8EpiWarp0) {
        // ------------------------------------------------ sums over the blocks
        const int e = warp - kFp8EpiWarp0, c0 = 64 * (e >> 2);   // first row of x of this warp in a tile
        const int lane_row = 32 * (warp & 3) + lane;             // output inside the tile
        const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + c0;
        bool ok = true;
        uint32_t i = 0;
        for (long long q = q0; q < q1 && ok;) {
            const Fp8Piece t = plan.piece(q, q1);
            const int n = t.n - c0;   // rows of x of this warp (none: it only keeps the hand-overs going)
            float2 acc[32];
#pragma unroll
            for (int c = 0; c < 32; c++) acc[c] = make_float2(0.f, 0.f);
            for (int kb = t.k0; kb < t.k1; kb++, i++) {
                const int b = i % kFp8Acc, s = i % kFp8ScaleRing;
                if (!warp_wait(&acc_full[b], (i / kFp8Acc) & 1u, abort_flag, p.err) ||
                    !warp_wait(&sc_full[s], (i / kFp8ScaleRing) & 1u, abort_flag, p.err)) { ok = false; break; }
                tc_fence_after();
                const float4* sc = reinterpret_cast<const float4*>(sc_ring + s * kFp8MaxRows + c0);
                if (n > 32) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float v[32];
                        tmem_ld32(taddr + 128 * b + 32 * h, v);
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            const float4 w = sc[8 * h + c];
                            acc[16 * h + 2 * c] = ffma2(make_float2(v[4 * c], v[4 * c + 1]), make_float2(w.x, w.y), acc[16 * h + 2 * c]);
                            acc[16 * h + 2 * c + 1] = ffma2(make_float2(v[4 * c + 2], v[4 * c + 3]), make_float2(w.z, w.w), acc[16 * h + 2 * c + 1]);
                        }
                    }
                } else if (n > 0) {
                    float v[32];
                    if (n > 16) {
                        tmem_ld32(taddr + 128 * b, v);
                    } else {
                        float u[16];
                        tmem_ld16(taddr + 128 * b, u);
#pragma unroll
                        for (int c = 0; c < 16; c++) {
                            v[c] = u[c];
                            v[16 + c] = 0.f;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        const float4 w = sc[c];
                        acc[2 * c] = ffma2(make_float2(v[4 * c], v[4 * c + 1]), make_float2(w.x, w.y), acc[2 * c]);
                        acc[2 * c + 1] = ffma2(make_float2(v[4 * c + 2], v[4 * c + 3]), make_float2(w.z, w.w), acc[2 * c + 1]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&acc_empty[b]);
                    mbar_arrive(&sc_empty[s]);
                }
            }
            if (!ok) break;
            const bool whole = t.k0 == 0 && t.k1 == p.kb;
            bool mine = true;   // this warp writes the tile's sums out
            if (!whole && n > 0) {
                const long long tq = (long long)t.tile * p.kb;
                const int c_first = plan.owner(tq), c_last = plan.owner(tq + p.kb - 1);
                // slot 0: the CTA did not begin the tile; slot 1: it began and left it
                const size_t slot = (size_t)x_rows * 128;
                float* to = p.part + ((size_t)blockIdx.x * 2 + (t.k0 == 0 ? 1 : 0)) * slot + (size_t)c0 * 128 + lane_row;
#pragma unroll
                for (int c = 0; c < 64; c++)
                    if (c < n) __stcg(to + c * 128, c & 1 ? acc[c >> 1].y : acc[c >> 1].x);
                __threadfence();
                __syncwarp();
                int arrived = 0;
                if (lane == 0) arrived = atomicAdd(&p.arrivals[c_first * kFp8EpiWarps + e], 1);
                arrived = __shfl_sync(0xffffffffu, arrived, 0);
                mine = arrived == c_last - c_first;
                if (mine) {
                    if (lane == 0) p.arrivals[c_first * kFp8EpiWarps + e] = 0;   // as the next launch finds it
                    __threadfence();
#pragma unroll
                    for (int c = 0; c < 32; c++) acc[c] = make_float2(0.f, 0.f);
                    for (int k = c_first; k <= c_last; k++) {
                        const float* from = p.part + ((size_t)k * 2 + (k == c_first ? 1 : 0)) * slot + (size_t)c0 * 128 + lane_row;
#pragma unroll
                        for (int c = 0; c < 64; c++)
                            if (c < n) {
                                const float v = __ldcg(from + c * 128);
                                if (c & 1) acc[c >> 1].y += v;
                                else acc[c >> 1].x += v;
                            }
                    }
                }
            }
            const int m = t.m * 128 + lane_row;
            if (mine && m < p.M) {
                const long long o = (long long)(t.pos + c0) * p.ld_out + m;
#pragma unroll
                for (int c = 0; c < 64; c++)
                    if (c < n) store_typed(p.out, o + c * p.ld_out, c & 1 ? acc[c >> 1].y : acc[c >> 1].x, p.type);
            }
            __syncwarp();
            q += t.k1 - t.k0;
        }
    }
    // ---------------- teardown: every role is done (or gave up); free tensor memory
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

}  // namespace qrm
