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

// ------------------------------------------------------------ waits
// A ready barrier costs one try_wait and a vote; the bounded loop is out of
// line.  (The single-lane waits with an integer division for the ring's slot
// that this kernel began with cost some 300 cycles each, ready or not, and
// were what bounded it: 710 TFLOP/s at 4096 x 28672 x 4096.)
struct Fp8Ctl {
    volatile int* abort_flag;
    int32_t* err;
};
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
    const uint64_t t0 = global_ns(), lim = wait_limit_ns();
    bool ok = false;
    for (;;) {
        for (int i = 0; i < 8 && !ok; i++) ok = bar_try(bar, parity);
        if (ok || *abort_flag || global_ns() - t0 > lim) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && (threadIdx.x & 31) == 0) {
        *abort_flag = 1;
        atomicOr(err, (int)ERR_TIMEOUT);
    }
    return ok;
}
// all lanes; false for all of them when the wait gave up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const Fp8Ctl& c) {
    if (__all_sync(0xffffffffu, bar_try(bar, parity))) return true;
    return bar_wait_slow(bar, parity, c.abort_flag, c.err);
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
// position in a ring: slot and the parity of its current phase
struct Ring {
    uint32_t i = 0, phase = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++i == n) {
            i = 0;
            phase ^= 1;
        }
    }
};

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
constexpr int kFp8ScaleRing = 4;        // slots of four blocks' scales
constexpr int kFp8MaxStages = 12;
constexpr int kFp8ScaleOff = 1024;                                       // after the barriers
constexpr int kFp8ScaleSlot = 4 * kFp8MaxRows;                           // floats
constexpr int kFp8TableOff = kFp8ScaleOff + kFp8ScaleRing * kFp8ScaleSlot * 4;
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
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm);
    uint64_t* full = bars;                                     // [stages] tiles are there
    uint64_t* done = full + kFp8MaxStages;                     // [stages] their MMAs are done
    uint64_t* acc_empty = done + kFp8MaxStages;                // [kFp8Acc]
    uint64_t* sc_full = acc_empty + kFp8Acc;                   // [kFp8ScaleRing]
    uint64_t* sc_empty = sc_full + kFp8ScaleRing;
    uint64_t* done_bar = sc_empty + kFp8ScaleRing;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + 768);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + 776);
    float* sc_ring = reinterpret_cast<float*>(sm + kFp8ScaleOff);
    int32_t* first_tile = reinterpret_cast<int32_t*>(sm + kFp8TableOff);
    int32_t* start = first_tile + p.groups + 1;
    int32_t* rows = start + p.groups + 1;
    const uint32_t stage_bytes = kFp8Tile + x_rows * 128;
    uint8_t* ring = sm + fp8_stage_off(p.groups);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&done[i], 1);
        }
        for (int i = 0; i < kFp8Acc; i++) mbar_init(&acc_empty[i], kFp8EpiWarps);
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
    const Fp8Ctl ctl{abort_flag, p.err};
    const uint32_t full0 = smem_u32(full), done0 = smem_u32(done), acc_empty0 = smem_u32(acc_empty);
    const uint32_t sc_full0 = smem_u32(sc_full), sc_empty0 = smem_u32(sc_empty);
    Fp8Plan plan{first_tile, start, rows, p.groups, p.mb, p.kb, (long long)first_tile[p.groups] * p.kb, 0};
    plan.ctas = (int)min((long long)gridDim.x, plan.total);   // each has a block at least
    const bool idle = (int)blockIdx.x >= plan.ctas;
    const long long q0 = idle ? 0 : plan.cut(blockIdx.x), q1 = idle ? 0 : plan.cut(blockIdx.x + 1);

    if (warp == 0) {
        // ------------------------------------------------ tiles
        bool ok = true;
        Ring r;
        uint32_t issued = 0;
        for (long long q = q0; q < q1 && ok;) {
            const Fp8Piece t = plan.piece(q, q1);
            const int boxes = (t.n + 15) >> 4;
            for (int kb = t.k0; kb < t.k1; kb++) {
                if (!bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                uint8_t* st = ring + r.i * stage_bytes;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&full[r.i], (uint32_t)(kFp8Tile + boxes * 2048));
                    if (p.back) tma_load_3d(st, &w_map, t.m * 128, kb * 128, t.group, &full[r.i]);
                    else tma_load_3d(st, &w_map, kb * 128, t.m * 128, t.group, &full[r.i]);
                    for (int b = 0; b < boxes; b++)
                        tma_load_2d(st + kFp8Tile + b * 2048, &x_map, kb * 128, t.pos + 16 * b, &full[r.i]);
                }
                __syncwarp();
                r.next(stages);
                issued++;
            }
            q += t.k1 - t.k0;
        }
        if (!ok && lane == 0)   // copies already issued must land before the CTA exits
            for (uint32_t j = issued > (uint32_t)stages ? issued - stages : 0; j < issued; j++)
                mbar_wait(&full[j % stages], (j / stages) & 1u);
    } else if (warp == 1) {
        // ------------------------------------------------ MMAs (one thread issues)
        bool ok = true;
        Ring r, a;
        // 32 contracted values are 32 bytes along K, or 32 rows of 128 bytes
        const uint32_t ring0 = smem_u32(ring), step = p.back ? 4096 >> 4 : 32 >> 4;
        const uint64_t w_desc = p.back ? sw128_desc_mn(ring0, kFp8Tile) : sw128_desc(ring0), x_desc = sw128_desc(ring0 + kFp8Tile);
        for (long long q = q0; q < q1 && ok;) {
            const Fp8Piece t = plan.piece(q, q1);
            const uint32_t idesc = umma_idesc_e4m3((t.n + 15) & ~15, p.back, false);
            for (int kb = t.k0; kb < t.k1; kb++) {
                if (!bar_wait(acc_empty0 + 8 * a.i, a.phase ^ 1u, ctl) || !bar_wait(full0 + 8 * r.i, r.phase, ctl)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t at = r.i * stage_bytes >> 4, d = tmem + 128 * a.i;
                    umma_f8(d, w_desc + at, x_desc + at, idesc, 0u);
                    umma_f8(d, w_desc + at + step, x_desc + at + 2, idesc, 1u);
                    umma_f8(d, w_desc + at + 2 * step, x_desc + at + 4, idesc, 1u);
                    umma_f8(d, w_desc + at + 3 * step, x_desc + at + 6, idesc, 1u);
                    umma_commit(&done[r.i]);
                }
                __syncwarp();
                r.next(stages);
                a.next(kFp8Acc);
            }
            q += t.k1 - t.k0;
        }
        // every MMA of this CTA has completed before tensor memory is released
        if (elect_one()) {
            umma_commit(done_bar);
            mbar_wait(done_bar, 0u);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------ scales, four blocks at a time
        bool ok = true;
        Ring r;
        for (long long q = q0; q < q1 && ok;) {
            const Fp8Piece t = plan.piece(q, q1);
            const float* ws = p.w_scales + (long long)t.group * p.s_group + (long long)t.m * p.s_m;
            const float* xs = p.x_scales + (long long)t.pos * p.ld_xs;
            for (int k4 = t.k0; k4 < t.k1; k4 += 4) {
                float v[4][4], w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int kb = k4 + j;
                    w[j] = kb < t.k1 ? __ldg(ws + (long long)kb * p.s_k) : 0.f;
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        v[j][c] = kb < t.k1 && lane + 32 * c < t.n ? __ldg(xs + (lane + 32 * c) * p.ld_xs + kb) : 0.f;
                }
                if (!bar_wait(sc_empty0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        sc_ring[r.i * kFp8ScaleSlot + j * kFp8MaxRows + lane + 32 * c] = v[j][c] * w[j];
                __syncwarp();
                if (lane == 0) bar_arrive(sc_full0 + 8 * r.i);
                r.next(kFp8ScaleRing);
            }
            q += t.k1 - t.k0;
        }
    } else if (warp >= kFp8EpiWarp0) {
        // ------------------------------------------------ sums over the blocks
        const int e = warp - kFp8EpiWarp0, c0 = 64 * (e >> 2);   // first row of x of this warp in a tile
        const int lane_row = 32 * (warp & 3) + lane;             // output inside the tile
        const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + c0;
        bool ok = true;
        Ring r, a, sr;
        for (long long q = q0; q < q1 && ok;) {
            const Fp8Piece t = plan.piece(q, q1);
            const int n = t.n - c0;   // rows of x of this warp (none: it only keeps the hand-overs going)
            float2 acc[32];
#pragma unroll
            for (int c = 0; c < 32; c++) acc[c] = make_float2(0.f, 0.f);
            for (int kb = t.k0; kb < t.k1; kb++) {
                const int j = (kb - t.k0) & 3;
                if ((j == 0 && !bar_wait(sc_full0 + 8 * sr.i, sr.phase, ctl)) || !bar_wait(done0 + 8 * r.i, r.phase, ctl)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float4* sc = reinterpret_cast<const float4*>(sc_ring + sr.i * kFp8ScaleSlot + j * kFp8MaxRows + c0);
                const uint32_t from = taddr + 128 * a.i;
                if (n > 32) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float v[32];
                        tmem_ld32(from + 32 * h, v);
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            const float4 w = sc[8 * h + c];
                            acc[16 * h + 2 * c] = ffma2(make_float2(v[4 * c], v[4 * c + 1]), make_float2(w.x, w.y), acc[16 * h + 2 * c]);
                            acc[16 * h + 2 * c + 1] = ffma2(make_float2(v[4 * c + 2], v[4 * c + 3]), make_float2(w.z, w.w), acc[16 * h + 2 * c + 1]);
                        }
                    }
                } else if (n > 16) {
                    float v[32];
                    tmem_ld32(from, v);
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        const float4 w = sc[c];
                        acc[2 * c] = ffma2(make_float2(v[4 * c], v[4 * c + 1]), make_float2(w.x, w.y), acc[2 * c]);
                        acc[2 * c + 1] = ffma2(make_float2(v[4 * c + 2], v[4 * c + 3]), make_float2(w.z, w.w), acc[2 * c + 1]);
                    }
                } else if (n > 0) {
                    float v[16];
                    tmem_ld16(from, v);
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const float4 w = sc[c];
                        acc[2 * c] = ffma2(make_float2(v[4 * c], v[4 * c + 1]), make_float2(w.x, w.y), acc[2 * c]);
                        acc[2 * c + 1] = ffma2(make_float2(v[4 * c + 2], v[4 * c + 3]), make_float2(w.z, w.w), acc[2 * c + 1]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                const bool last = j == 3 || kb + 1 == t.k1;   // of the scales' slot
                if (lane == 0) {
                    bar_arrive(acc_empty0 + 8 * a.i);
                    if (last) bar_arrive(sc_empty0 + 8 * sr.i);
                }
                r.next(stages);
                a.next(kFp8Acc);
                if (last) sr.next(kFp8ScaleRing);
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
