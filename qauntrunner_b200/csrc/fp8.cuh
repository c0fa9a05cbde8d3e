// fp8.cuh -- product of 8-bit rows with 8-bit matrices that carry a scale for
// each block of 128: dense, or grouped (rows of group g times matrix g).
//
//   y[t][m] = sum_b sx[t][b] sw[m/128][b] * sum_{c in block b} qx[t][c] qw[m][c]
//
// with blocks of 128 along the contracted dimension.  The inner sums are
// tcgen05.mma (kind::f8f6f4, e4m3 x e4m3) into f32 tensor memory, a fresh
// accumulator per block; the outer sum is one f32 FMA per value and block in
// the epilogue warps' registers.  Its factor sx sw is formed first, in f32: it
// loses bits below 2^-126, which only results below some 1e-29 show, and is
// infinite from 2^128 on (two factors, one after the other, would cost the
// large-group kernel's sums another operation a value).  The transposed product (the input gradient,
// y = W^T x) reads the same stored matrix: its tiles enter the MMA with M as
// their contiguous dimension instead of K, and the scales' two block indices
// change places.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "gemv_imma.cuh"
#include "pair_drain.h"
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
// The same with the 64-byte swizzle: 64 values a row, atoms of 512 bytes.
__device__ __forceinline__ uint64_t sw64_desc_mn(uint32_t saddr, uint32_t wide_stride) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(wide_stride >> 4) << 16) | ((uint64_t)(512 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)4 << 61);
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
__device__ __forceinline__ void tmem_ld16_now(uint32_t taddr, float* v) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
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

template <typename T> __device__ __forceinline__ T round_to(float v);
template <> __device__ __forceinline__ float round_to<float>(float v) { return v; }
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
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
__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
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
// the last `stages` of a CTA's own copies have landed (out of line: it runs only when a wait gave up)
__device__ __noinline__ void drain_own(uint64_t* full, uint32_t issued, uint32_t stages) {
    for (uint32_t j = issued > stages ? issued - stages : 0; j < issued; j++) mbar_wait(&full[j % stages], (j / stages) & 1u);
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
// All tiles' blocks, one after the other, are cut into runs for one CTA on each
// SM, inside a tile where that pays (fp8_share_out): one token through one
// matrix still reads it with every SM.  A CTA that did only part of a tile's
// blocks leaves its f32 sums in the workspace, and the last one to arrive adds
// the parts up in the CTAs' order, so that the result does not depend on who
// was last.  Nobody waits.
//
// 512 rows over 32 matrices of 4096 x 7168 (940 MB): 163 us, 5.8 TB/s.  One row
// through one such matrix: 12 us, latencies.
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
constexpr int kFp8MinRun = 4;           // blocks a CTA has at least
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
    bool whole;                  // no tile is shared
    __device__ long long cut(int c) const { return whole ? total / kb * c / ctas * kb : total * c / ctas; }
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

// How `tiles` tiles of kb blocks are shared out.  Parts of a tile have to be
// announced and added up, which costs about 6 us (16 blocks), 3 of them for the
// second part where a CTA has parts of two.  So
// - with fewer tiles than CTAs, each tile gets the same whole number of CTAs,
//   unless that gives the busiest CTA 8 blocks more than an even share (one
//   row through 4096 x 7168: 11.4 us in place of 14.9);
// - with more, CTAs take whole tiles, unless that is 16 blocks more;
// - otherwise all blocks in equal runs, kFp8MinRun at least.
__device__ inline void fp8_share_out(Fp8Plan& plan, int tiles, int kb, int ctas) {
    plan.total = (long long)tiles * kb;
    plan.whole = false;
    const long long even = (plan.total + ctas - 1) / ctas;
    if (tiles > 0 && tiles <= ctas) {
        const int each = max(1, min(ctas / tiles, kb / kFp8MinRun));
        if ((kb + each - 1) / each <= even + 8) {
            plan.ctas = tiles * each;
            return;
        }
    } else if (tiles > ctas && (long long)((tiles + ctas - 1) / ctas) * kb <= even + 16) {
        plan.ctas = ctas;
        plan.whole = true;
        return;
    }
    plan.ctas = (int)min((long long)ctas, (plan.total + kFp8MinRun - 1) / kFp8MinRun);
}

// The groups' tables in shared memory, by one warp; the caller synchronises.
// Offsets that do not ascend within [0, T] make a group empty and raise an
// error, and so does a start below any offset before it: no row outside x or
// out is ever touched, and none belongs to two groups (whose CTAs would both
// write it, and whose tiles together could be more than a count of them holds).
// tile_rows rows of x a tile, `across` tiles along the outputs.
__device__ inline void fp8_tables(const Fp8Params& p, int32_t* first_tile, int32_t* start, int32_t* rows, int tile_rows,
                                  int across, bool report) {
    const int lane = threadIdx.x & 31;
    int before = 0, top = 0;   // tiles, largest offset so far
    bool bad = false;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + lane;
        int a = 0, b = 0;
        if (g < p.groups) {
            a = p.offsets ? p.offsets[g] : 0;
            b = p.offsets ? p.offsets[g + 1] : p.T;
        }
        int most = a;   // of the offsets up to this one
        if (p.groups > 1) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) most = max(most, __shfl_up_sync(0xffffffffu, most, o));   // (lanes below o get their own)
            most = max(most, top);
            top = __shfl_sync(0xffffffffu, most, 31);
        }
        if (a < most || a < 0 || b < a || b > p.T) {
            bad |= g < p.groups;
            a = b = 0;
        }
        const int tiles = (b - a + tile_rows - 1) / tile_rows * across;
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

// f(0) ... f(n - 1), n <= 64, by constant indices (the columns are registers),
// 16 at a time: what is not needed is jumped over.  This code runs once or
// twice in a launch, cold, and straight through all 64 it took 2.5 us for one.
template <typename F>
__device__ __forceinline__ void for_columns(int n, F f) {
#pragma unroll
    for (int h = 0; h < 4; h++) {
        if (n <= 16 * h) return;
#pragma unroll
        for (int c = 0; c < 16; c++)
            if (16 * h + c < n) f(16 * h + c);
    }
}
template <typename T>
__device__ __forceinline__ void store_columns_as(T* to, long long ld, const float2 (&acc)[32], int n) {
    for_columns(n, [&](int c) { to[c * ld] = round_to<T>(c & 1 ? acc[c >> 1].y : acc[c >> 1].x); });
}
// a warp's sums to out: lane_row is the output inside the tile, c0 the first of the n rows of x
__device__ __forceinline__ void store_columns(const Fp8Params& p, const float2 (&acc)[32], const Fp8Piece& t, int c0, int n,
                                              int lane_row) {
    const int m = t.m * 128 + lane_row;
    if (m >= p.M) return;
    const long long o = (long long)(t.pos + c0) * p.ld_out + m;
    if (p.type == 0) store_columns_as(reinterpret_cast<float*>(p.out) + o, p.ld_out, acc, n);
    else if (p.type == 1) store_columns_as(reinterpret_cast<__half*>(p.out) + o, p.ld_out, acc, n);
    else store_columns_as(reinterpret_cast<__nv_bfloat16*>(p.out) + o, p.ld_out, acc, n);
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
    volatile uint32_t* issued = reinterpret_cast<volatile uint32_t*>(sm + 780);   // stages, once their warp is through
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
    pdl_start();   // nothing before this reads or writes global memory
    if (warp == 2) fp8_tables(p, first_tile, start, rows, kFp8MaxRows, p.mb, blockIdx.x == 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Fp8Ctl ctl{abort_flag, p.err};
    const uint32_t full0 = smem_u32(full), done0 = smem_u32(done), acc_empty0 = smem_u32(acc_empty);
    const uint32_t sc_full0 = smem_u32(sc_full), sc_empty0 = smem_u32(sc_empty);
    Fp8Plan plan{first_tile, start, rows, p.groups, p.mb, p.kb};
    fp8_share_out(plan, first_tile[p.groups], p.kb, gridDim.x);
    const bool idle = (int)blockIdx.x >= plan.ctas;
    const long long q0 = idle ? 0 : plan.cut(blockIdx.x), q1 = idle ? 0 : plan.cut(blockIdx.x + 1);

    if (warp == 0) {
        // ------------------------------------------------ tiles
        bool ok = true;
        Ring r;
        uint32_t n_issued = 0;
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
                n_issued++;
            }
            q += t.k1 - t.k0;
        }
        if (lane == 0) *issued = n_issued;
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
        const size_t slot = (size_t)x_rows * 128;   // floats of a part
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
                    tmem_ld16_now(from, v);
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
            if (t.k0 == 0 && t.k1 == p.kb) {
                store_columns(p, acc, t, c0, n, lane_row);
            } else {
                // slot 0: the CTA did not begin the tile; slot 1: it began and left it
                float* to = p.part + ((size_t)blockIdx.x * 2 + (t.k0 == 0 ? 1 : 0)) * slot + (size_t)c0 * 128 + lane_row;
                for_columns(n, [&](int c) { __stcg(to + c * 128, c & 1 ? acc[c >> 1].y : acc[c >> 1].x); });
            }
            q += t.k1 - t.k0;
        }
        // Parts of tiles: the CTA's first and its last piece, if they are.  Both
        // are announced here, when their stores have long landed, and not
        // between the pieces, where the fence stopped the sums for 1.5 us.
        __threadfence();
        __syncwarp();
#pragma unroll 1
        for (int w = 0; w < 2 && ok && q0 < q1; w++) {
            const int last_tile = (int)((q1 - 1) / p.kb);
            if (w == 1 && (long long)last_tile * p.kb <= q0) break;   // one piece only
            const Fp8Piece t = plan.piece(w == 0 ? q0 : (long long)last_tile * p.kb, q1);
            const int n = t.n - c0;
            if ((t.k0 == 0 && t.k1 == p.kb) || n <= 0) continue;
            const long long tq = (long long)t.tile * p.kb;
            const int c_first = plan.owner(tq), c_last = plan.owner(tq + p.kb - 1);
            int arrived = 0;
            if (lane == 0) arrived = atomicAdd(&p.arrivals[c_first * kFp8EpiWarps + e], 1);
            arrived = __shfl_sync(0xffffffffu, arrived, 0);
            if (arrived != c_last - c_first) continue;
            // the last to arrive adds the parts up, in the CTAs' order
            if (lane == 0) p.arrivals[c_first * kFp8EpiWarps + e] = 0;   // as the next launch finds it
            __threadfence();
            float2 acc[32];
#pragma unroll
            for (int c = 0; c < 32; c++) acc[c] = make_float2(0.f, 0.f);
            const float* from = p.part + (size_t)c0 * 128 + lane_row;
#pragma unroll 1
            for (int k = c_first; k <= c_last; k += 4) {   // of up to 16 columns, four parts' loads in flight
                const float* part[4];
#pragma unroll
                for (int u = 0; u < 4; u++) part[u] = from + ((size_t)min(k + u, c_last) * 2 + (k + u == c_first ? 1 : 0)) * slot;
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    if (n <= 16 * h) break;
                    float v[4][16];
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int c = 0; c < 16; c++)
                            v[u][c] = 16 * h + c < n && k + u <= c_last ? __ldcg(part[u] + (16 * h + c) * 128) : 0.f;
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            acc[8 * h + c].x += v[u][2 * c];
                            acc[8 * h + c].y += v[u][2 * c + 1];
                        }
                }
            }
            store_columns(p, acc, t, c0, n, lane_row);
        }
    }
    // ---------------- teardown: every role is done (or gave up); free tensor memory
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // a role that gave up may have left copies that nothing waited for: they land before the CTA exits
    if (threadIdx.x == 0 && *abort_flag) drain_own(full, *issued, stages);
    if (warp == 1) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------ rows of x on the MMA's M side
// For groups of many rows, which the tensor cores bound.  A pair of SMs
// (cta_group::2) shares a tile of 256 rows of x times 256 outputs: each CTA
// loads 128 rows of x and 128 outputs' weights for a block (32 KB) and the MMA
// reads both halves of the weights, so a block costs each SM 64 bytes of L2
// traffic a cycle at the full MMA rate, half of what a tile of its own would
// cost.  A thread of the epilogue owns one row of x and 128 outputs (128 f32 in
// registers): the two scales are one product for all 128.
//
// What bounds it is the way around an accumulator: MMAs, hand-over, the
// epilogue's loads out of tensor memory, hand-over back.  So the tile's two
// blocks of 128 outputs have MMAs, accumulators (two each) and epilogue warps
// of their own, and take turns on the tensor cores.  4096 rows, 28672 x 4096:
// 427 us, 2.25 PFLOP/s, tensor pipe 62 % active; 497 us under sustained load
// (power cap, 1.5 GHz).
//
// Warps: 0 loads tiles, 1 issues the MMAs (in the pair's first CTA), 2 brings
// the scales, 4-11 add up: lane quarter (warp & 3), outputs 128 (warp >= 8).
constexpr int kFp8PairStages = 6;
constexpr int kFp8PairStage = 2 * kFp8Tile;   // rows of x, weights
constexpr int kFp8PairAcc = 2;                // accumulators of 128 columns for each block of outputs
constexpr int kFp8PairScaleSlot = 4 * 2 * 128;
constexpr int kFp8PairScaleRing = 3;
// registers a thread after the split: the loading, issuing and scaling warps
// give up what the sums need.  The sum may not pass what the launch has (168 a
// thread; qrm_fp8_create checks it), or the split would wait for ever.
constexpr int kFp8PairRegsFew = 72, kFp8PairRegsMany = 216;
constexpr int kFp8PairRegs = 128 * kFp8PairRegsFew + 256 * kFp8PairRegsMany;
static_assert(kFp8PairRegs <= kFp8Warps * 32 * 168, "register split");
constexpr int kFp8PairTableOff = kFp8ScaleOff + kFp8PairScaleRing * kFp8PairScaleSlot * 4;
__host__ __device__ inline int fp8_pair_stage_off(int groups) {
    return (kFp8PairTableOff + 12 * (groups + 1) + 1023) / 1024 * 1024;
}
__device__ __forceinline__ uint32_t map_to_rank0(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
// (What it hands over was read from tensor memory and is ordered by the
// tcgen05 fence before it; with cluster scope here a full memory barrier came
// with every block: 1010 us in place of 560 at 4096 x 28672 x 4096, then.)
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// loads of a pair's CTA that complete on a barrier of its first CTA
__device__ __forceinline__ void tma_pair_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_pair_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrives on the barrier at `bar`'s offset in both CTAs once the MMAs are done
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// a word of the peer's shared memory, at the same place as ours; the cluster barrier after it makes it visible
__device__ __forceinline__ void store_peer(uint32_t* p, uint32_t rank, uint32_t v) {
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n st.shared::cluster.u32 [a], %2;\n}\n" ::"r"(smem_u32(p)),
        "r"(rank), "r"(v)
        : "memory");
}
// the first CTA's barriers, as drain_pair moves them on
struct PairBars {
    uint64_t* full;
    __device__ void expect(uint32_t slot) { mbar_arrive_expect_tx(&full[slot], kFp8PairStage); }
    __device__ void complete(uint32_t slot) {
        asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[slot])),
                     "r"((uint32_t)kFp8PairStage)
                     : "memory");
    }
    __device__ void wait(uint32_t slot, uint32_t parity) { mbar_wait(&full[slot], parity); }
};

struct Fp8PairTile {
    int group, n;    // matrix, first output
    int pos, rows;   // first row of x of the tile, rows of the group from there on
};

// 128 outputs of one row that starts on 16 bytes, or on 32 (`wide`): a warp
// writes 32 rows at once, so what counts is how few stores a row takes (32 bytes
// a store: 495 us in place of 531 at 4096 x 28672 x 4096 in bf16, 542 in place
// of 621 in f32, 420 in place of 435 for 8192 rows over 32 x 4096 x 7168, each
// under sustained load).  One value at a time took some 20 us
// a tile: where the rows of out do not start on 16 bytes, the other kernel
// runs, whose warps write neighbouring outputs.
template <typename T>
__device__ __forceinline__ void store_row(T* out, int left, const float2 (&acc)[64], bool wide) {
    constexpr int V = 32 / sizeof(T);   // values of one store
#pragma unroll
    for (int c = 0; c < 128 / V; c++) {
        if (V * c + V <= left) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if constexpr (sizeof(T) == 4) {
                    const float2 v = acc[4 * c + i / 2];
                    w[i] = __float_as_uint(i & 1 ? v.y : v.x);
                } else {
                    const T h[2] = {round_to<T>(acc[8 * c + i].x), round_to<T>(acc[8 * c + i].y)};
                    memcpy(&w[i], h, 4);
                }
            }
            if (wide) {
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + V * c), "r"(w[0]), "r"(w[1]),
                             "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                             : "memory");
            } else {
                uint4* to = reinterpret_cast<uint4*>(out + V * c);
                to[0] = make_uint4(w[0], w[1], w[2], w[3]);
                to[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
        } else {   // the last few
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                const float2 v = acc[V / 2 * c + i];
                if (V * c + 2 * i < left) out[V * c + 2 * i] = round_to<T>(v.x);
                if (V * c + 2 * i + 1 < left) out[V * c + 2 * i + 1] = round_to<T>(v.y);
            }
        }
        asm volatile("" ::: "memory");   // one store's registers at a time
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFp8Warps * 32, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, Fp8Params p,
                int wide_out, int wide_xs) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm);
    uint64_t* full = bars;                            // first CTA: both CTAs' tiles are there
    uint64_t* done = full + kFp8PairStages;           // both: the stage's MMAs are done
    uint64_t* done_first = done + kFp8PairStages;     // both: those of its first block of outputs
    uint64_t* acc_empty = done_first + kFp8PairStages;   // first CTA: both epilogues have read; [block of outputs][acc]
    uint64_t* sc_full = acc_empty + 2 * kFp8PairAcc;
    uint64_t* sc_empty = sc_full + kFp8PairScaleRing;
    uint64_t* done_bar = sc_empty + kFp8PairScaleRing;
    uint64_t* left_bar = done_bar + 1;                // both, when the first CTA gave up: its commits are through
    // (not in the dynamic part, whose addresses would take registers through the sums)
    __shared__ volatile int given_up;
    __shared__ volatile uint32_t from_peer, issued;   // issued: stages, once their warp is through
    volatile int* abort_flag = &given_up;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + 776);
    float* sc_ring = reinterpret_cast<float*>(sm + kFp8ScaleOff);
    int32_t* first_tile = reinterpret_cast<int32_t*>(sm + kFp8PairTableOff);
    int32_t* start = first_tile + p.groups + 1;
    int32_t* rows = start + p.groups + 1;
    uint8_t* ring = sm + fp8_pair_stage_off(p.groups);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;   // in the pair: the cluster is two CTAs along x
    if (threadIdx.x == 0) {
        for (int i = 0; i < kFp8PairStages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&done[i], 1);
            mbar_init(&done_first[i], 1);
        }
        for (int i = 0; i < 2 * kFp8PairAcc; i++) mbar_init(&acc_empty[i], kFp8EpiWarps);
        for (int i = 0; i < kFp8PairScaleRing; i++) {
            mbar_init(&sc_full[i], 1);
            mbar_init(&sc_empty[i], kFp8EpiWarps);
        }
        mbar_init(done_bar, 1);
        mbar_init(left_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pdl_start();   // nothing before this reads or writes global memory
    if (warp == 2) fp8_tables(p, first_tile, start, rows, 256, (p.M + 255) / 256, blockIdx.x == 0);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers are ready
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Fp8Ctl ctl{abort_flag, p.err};
    const uint32_t done0 = smem_u32(done), sc_full0 = smem_u32(sc_full), sc_empty0 = smem_u32(sc_empty);
    const int tiles = first_tile[p.groups], pairs = gridDim.x >> 1, KB = p.kb;

    // tile number -> what this CTA does of it; the tiles of one block of
    // outputs follow each other, so its weights come from HBM once
    auto tile_at = [&](int i) {
        int lo = 0, hi = p.groups;   // the last group with first_tile <= i has rows
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first_tile[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int blocks = (rows[lo] + 255) >> 8, in = i - first_tile[lo];
        const int n = in / blocks, at = (in - n * blocks) * 256 + 128 * (int)rank;
        return Fp8PairTile{lo, n * 256, start[lo] + at, rows[lo] - at};
    };

    if (warp < kFp8EpiWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp8PairRegsFew));
        if (warp == 0) {
            // -------------------------------------------- tiles
            bool ok = true;
            Ring r;
            uint32_t n_issued = 0;
            const uint32_t full0 = map_to_rank0(smem_u32(full)), ring0 = smem_u32(ring);
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
                const Fp8PairTile t = tile_at(i);
                const int n = t.n + 64 * (int)rank;   // half of each block of outputs
                for (int kb = 0; kb < KB; kb++) {
                    if (!bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                    if (elect_one()) {
                        const uint32_t st = ring0 + r.i * kFp8PairStage, bar = full0 + 8 * r.i;
                        if (rank == 0) mbar_arrive_expect_tx(&full[r.i], 2 * kFp8PairStage);
                        // (no rows for this CTA: from past the end, which is zeros and no traffic)
                        tma_pair_2d(st, &x_map, kb * 128, t.rows > 0 ? t.pos : p.T, bar);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t to = st + kFp8Tile + h * (kFp8Tile / 2);
                            if (p.back) tma_pair_3d(to, &w_map, n + 128 * h, kb * 128, t.group, bar);
                            else tma_pair_3d(to, &w_map, kb * 128, n + 128 * h, t.group, bar);
                        }
                    }
                    __syncwarp();
                    r.next(kFp8PairStages);
                    n_issued++;
                }
            }
            if (lane == 0) issued = n_issued;
        } else if (warp == 1 && rank == 0) {
            // -------------------------------------------- MMAs (one thread issues for both CTAs)
            bool ok = true;
            Ring r, a;
            const uint32_t full0 = smem_u32(full), acc_empty0 = smem_u32(acc_empty), ring0 = smem_u32(ring);
            const uint32_t done_first0 = smem_u32(done_first);
            // (along N: rows of 64 values, half of a block of outputs, 32 of them contracted by one MMA)
            const uint32_t step = p.back ? 2048 >> 4 : 32 >> 4;
            const uint64_t x_desc = sw128_desc(ring0);
            const uint64_t w_desc = p.back ? sw64_desc_mn(ring0 + kFp8Tile, kFp8Tile / 2) : sw128_desc(ring0 + kFp8Tile);
            const uint32_t idesc = (umma_idesc_e4m3(128, false, p.back) & ~(0x1Fu << 24)) | ((uint32_t)(256 >> 4) << 24);
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
                for (int kb = 0; kb < KB; kb++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (!bar_wait(acc_empty0 + 8 * (kFp8PairAcc * h + a.i), a.phase ^ 1u, ctl) ||
                            (h == 0 && !bar_wait(full0 + 8 * r.i, r.phase, ctl))) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t at = r.i * (kFp8PairStage >> 4), d = tmem + 128 * (kFp8PairAcc * h + a.i);
                            const uint64_t xd = x_desc + at, wd = w_desc + at + h * (kFp8Tile / 2 >> 4);
                            umma_f8_pair(d, xd, wd, idesc, 0u);
                            umma_f8_pair(d, xd + 2, wd + step, idesc, 1u);
                            umma_f8_pair(d, xd + 4, wd + 2 * step, idesc, 1u);
                            umma_f8_pair(d, xd + 6, wd + 3 * step, idesc, 1u);
                            umma_commit_pair((h == 0 ? done_first0 : done0) + 8 * r.i);
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    r.next(kFp8PairStages);
                    a.next(kFp8PairAcc);
                }
            }
            // every MMA has completed before tensor memory is released
            if (elect_one()) {
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(done_bar)) : "memory");
                mbar_wait(done_bar, 0u);
            }
            __syncwarp();
        } else if (warp == 2) {
            // -------------------------------------------- scales: sx sw of 128 rows x two blocks of outputs
            bool ok = true;
            Ring r;
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
                const Fp8PairTile t = tile_at(i);
                const int m = t.n >> 7, m1 = min(m + 1, p.mb - 1);   // an absent second block is not stored
                const float* ws = p.w_scales + (long long)t.group * p.s_group;
                const float* xs = p.x_scales + (long long)t.pos * p.ld_xs;
                for (int k4 = 0; k4 < KB; k4 += 4) {
                    float v[4][4], w[4][2];   // [row lane + 32 c][block j]
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int kb = k4 + j;
                        w[j][0] = kb < KB ? __ldg(ws + (long long)m * p.s_m + (long long)kb * p.s_k) : 0.f;
                        w[j][1] = kb < KB ? __ldg(ws + (long long)m1 * p.s_m + (long long)kb * p.s_k) : 0.f;
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const bool in = lane + 32 * c < t.rows;
                        const float* from = xs + (long long)(lane + 32 * c) * p.ld_xs + k4;
                        if (wide_xs && k4 + 4 <= KB) {
                            const float4 f = in ? __ldg(reinterpret_cast<const float4*>(from)) : make_float4(0.f, 0.f, 0.f, 0.f);
                            v[c][0] = f.x; v[c][1] = f.y; v[c][2] = f.z; v[c][3] = f.w;
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; j++) v[c][j] = in && k4 + j < KB ? __ldg(from + j) : 0.f;
                        }
                    }
                    if (!bar_wait(sc_empty0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                    float* to = sc_ring + r.i * kFp8PairScaleSlot + lane;
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            to[j * 256 + 32 * c] = v[c][j] * w[j][0];
                            to[j * 256 + 128 + 32 * c] = v[c][j] * w[j][1];
                        }
                    __syncwarp();
                    if (lane == 0) bar_arrive(sc_full0 + 8 * r.i);
                    r.next(kFp8PairScaleRing);
                }
            }
        }
    } else {
        // ------------------------------------------------ sums over the blocks
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp8PairRegsMany));   // 428 us in place of 452
        const int half = (warp - kFp8EpiWarp0) >> 2, row = 32 * (warp & 3) + lane;   // block of outputs, row of x in the tile
        const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128 * kFp8PairAcc * half;
        const uint32_t acc_empty0 = map_to_rank0(smem_u32(acc_empty + kFp8PairAcc * half));
        const uint32_t ready0 = half ? done0 : smem_u32(done_first);
        bool ok = true;
        Ring r, a, sr;
        for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
            const Fp8PairTile t = tile_at(i);
            float2 acc[64];
#pragma unroll
            for (int c = 0; c < 64; c++) acc[c] = make_float2(0.f, 0.f);
            for (int kb = 0; kb < KB; kb++) {
                const int j = kb & 3;
                if ((j == 0 && !bar_wait(sc_full0 + 8 * sr.i, sr.phase, ctl)) || !bar_wait(ready0 + 8 * r.i, r.phase, ctl)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float f = sc_ring[sr.i * kFp8PairScaleSlot + j * 256 + 128 * half + row];
                const float2 f2 = make_float2(f, f);
                const uint32_t from = taddr + 128 * a.i;
                // (16 columns at a time: with the next load issued before a load's sums, or 32 and 64 at a time, it was
                // 430 to 527 us in place of 428 at 4096 x 28672 x 4096: the scheduler's other warp fills the gaps)
#pragma unroll
                for (int h = 0; h < 8; h++) {
                    float v[16];
                    tmem_ld16_now(from + 16 * h, v);
                    if (h == 7) {   // all of it is in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive_cluster(acc_empty0 + 8 * a.i);
                    }
#pragma unroll
                    for (int c = 0; c < 8; c++) acc[8 * h + c] = ffma2(make_float2(v[2 * c], v[2 * c + 1]), f2, acc[8 * h + c]);
                }
                if (j == 3 || kb + 1 == KB) {
                    if (lane == 0) bar_arrive(sc_empty0 + 8 * sr.i);
                    sr.next(kFp8PairScaleRing);
                }
                r.next(kFp8PairStages);
                a.next(kFp8PairAcc);
            }
            if (!ok) break;
            if (row < t.rows) {
                const long long o = (long long)(t.pos + row) * p.ld_out + t.n + 128 * half;
                const int left = p.M - t.n - 128 * half;
                if (p.type == 0) store_row(reinterpret_cast<float*>(p.out) + o, left, acc, wide_out);
                else if (p.type == 1) store_row(reinterpret_cast<__half*>(p.out) + o, left, acc, wide_out);
                else store_row(reinterpret_cast<__nv_bfloat16*>(p.out) + o, left, acc, wide_out);
            }
            __syncwarp();
        }
    }
    // ---------------- teardown: every role of both CTAs is done (or gave up); free tensor memory
    tc_fence_before();
    __syncthreads();
    // Copies that nothing waited for are left only where the MMAs did not run to their end, and then the first CTA's
    // flag is set.  It learns how many stages the other has issued, which learns whether to stay.
    if (threadIdx.x == 0) store_peer(const_cast<uint32_t*>(&from_peer), rank ^ 1, rank == 0 ? (uint32_t)given_up : issued);
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    if (rank == 0 ? given_up != 0 : from_peer != 0) {
        if (rank == 0 && threadIdx.x == 0) {
            PairBars bars{full};
            drain_pair(issued, from_peer, kFp8PairStages, bars);
        }
        if (warp == 1) {
            if (rank == 0 && elect_one()) umma_commit_pair(smem_u32(left_bar));
            __syncwarp();
            if (lane == 0) mbar_wait(left_bar, 0u);
        }
        __syncwarp();
        cluster_sync_all();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace qrm
