// fp4.cuh -- product of 4-bit microscaled rows with 4-bit microscaled matrices,
// dense or grouped (rows of group g times matrix g), and the gated product of
// gate and up with SwiGLU behind it.
//
//   y[t][m] = sum_b 2^(sx[t][b] + sw[m][b] - 254) sum_{c in block b} qx[t][c] qw[m][c]
//   h[t][j] = silu(y[t][j]) y[t][f + j]                       (gated; a matrix of 2 f rows)
//
// with blocks of 32 along the contracted dimension, e2m1 codes and e8m0 scales.
// All of it is tcgen05.mma kind::mxf4, which takes the scales from tensor memory
// and multiplies by them on its way: 64 contracted values, two blocks, an
// instruction.  Products of two codes and their sums by powers of two are exact
// as far as f32 goes, and nothing is left for the epilogue but the output.
//
// Scales enter tensor memory in units of 512 bytes for 128 rows x 128 contracted
// values: row r's four bytes at 16 (r % 32) + 4 (r / 32), which tcgen05.cp
// spreads over four columns.  A matrix's are laid out that way when it is made;
// those of x stay as they are and are brought into that order on their way to
// shared memory, because a group may start at any row.  For the gated product
// the matrix's rows enter the MMA in turns of 16: 16 of gate, the same 16 of up,
// so that both halves of a feature are in the same 32 lanes of tensor memory (or
// the same 32 columns), and its scales are kept in that order as well.
#pragma once
#include "pair_drain.h"
#include "rows4.cuh"
#include "umma_sync.cuh"

namespace qrm {

constexpr int kFp4MaxGroups = 1024;
constexpr int kFp4Step = 256;                // contracted values of a stage: 128 bytes of a row
constexpr int kFp4Tile = 128 * 128;          // bytes of 128 rows of codes in a stage
constexpr int kFp4Scales = 1024;             // bytes of their scales

enum Fp4Mode { kFp4Plain = 0, kFp4Gated = 1, kFp4GatedRows = 2 };   // y; h; h in 4-bit rows

struct Fp4Params {
    const uint8_t* w_scales;   // [groups][units][steps][2][512]
    const uint8_t* x_scales;   // [T][ld_xs]
    const int32_t* offsets;    // [groups+1] rows of each group, or NULL (one group)
    void* out;                 // [T][ld_out], or codes (ld_out in bytes)
    uint8_t* out_scales;       // [T][ld_os]
    int32_t* err;
    long long ld_xs, ld_out, ld_os;
    float limit;               // infinite: none
    int T, groups;
    int M;                     // outputs (gated: f)
    int units;                 // of 128 rows in w_scales, of one matrix (gated: 64 features)
    int steps;                 // stages of the contracted dimension
    int blocks;                // of 32 in it
    int type;                  // of out
    int row_tiles;             // room for tiles of rows in the grid (weights on the M side)
    int wide_xs;               // rows of scales start on 16 bytes: 2, on 8: 1
};

// Instruction descriptor of kind::mxf4: f32 accumulators, e2m1 A and B, e8m0
// scales, of which bytes `part` and `part` + 1 of each word are used (0 or 2).
__device__ __forceinline__ constexpr uint32_t umma_idesc_mxf4(int m, int n, int part) {
    return ((uint32_t)part << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) |
           ((uint32_t)part << 29);
}
// Descriptor of a unit of scales in shared memory for tcgen05.cp: 32 rows of 16
// bytes one after the other, no swizzle (8-row groups 128 bytes apart).
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
template <int CTAS>
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                          uint32_t b_scales, uint32_t accumulate) {
    if constexpr (CTAS == 1)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
            : "memory");
}
// a unit of scales to four columns of tensor memory (of both CTAs: each its own)
template <int CTAS>
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
    if constexpr (CTAS == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// 128 rows of a matrix's codes into shared memory: from row m on, or (gated)
// features m ... m + 63 of gate and up in turns of 16, which the matrix's map has
// as dimensions of their own: 16 rows, gate or up, sixteens of features.
template <bool GATED>
__device__ __forceinline__ void load_weights(void* dst, const CUtensorMap* map, int x, int m, int group, uint64_t* bar) {
    if constexpr (!GATED) tma_load_3d(dst, map, x, m, group, bar);
    else
        asm volatile(
            "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %5, %5, %3, %4}], "
            "[%6];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(m >> 4), "r"(group), "r"(0), "r"(smem_u32(bar))
            : "memory");
}
template <bool GATED>
__device__ __forceinline__ void load_weights_pair(uint32_t dst, const CUtensorMap* map, int x, int m, int group, uint32_t bar) {
    if constexpr (!GATED) tma_pair_3d(dst, map, x, m, group, bar);
    else
        asm volatile(
            "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %5, %5, "
            "%3, %4}], [%6];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(m >> 4), "r"(group), "r"(0), "r"(bar)
            : "memory");
}
// a value that is the same in all lanes, so that it may be kept in a register of the warp
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
// both barriers; one vote where both are ready
__device__ __forceinline__ bool bar_wait_both(uint32_t a, uint32_t a_parity, uint32_t b, uint32_t b_parity, const WaitCtl& c) {
    const bool first = bar_try(a, a_parity), second = bar_try(b, b_parity);
    if (__all_sync(0xffffffffu, first && second)) return true;
    return bar_wait(a, a_parity, c) && bar_wait(b, b_parity, c);
}
// The high words of the descriptors, which are constants: of operands in the
// 128-byte swizzle, of units of scales.
constexpr uint32_t kSw128High = (1024 >> 4) | (1u << 14) | (2u << 29), kScaleHigh = (128 >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t sw128_low(uint32_t saddr) { return (saddr & 0x3FFFFu) >> 4 | 1u << 16; }
__device__ __forceinline__ uint32_t scale_low(uint32_t saddr) { return (saddr & 0x3FFFFu) >> 4; }
__device__ __forceinline__ uint64_t wide_desc(uint32_t low, uint32_t high) { return (uint64_t)high << 32 | low; }
// what this thread wrote to shared memory is there for copies and MMAs
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 4 N scales of a row from block b on (0 for those past the last).  Rows start
// anywhere, so the whole words around the bytes are read and shifted; a word that
// holds none of the row's bytes is not touched.
template <int N>
__device__ __forceinline__ void some_scales(const uint8_t* __restrict__ row, int b, int blocks, uint32_t (&out)[N]) {
    const uint8_t* at = row + b;
    const int in = (int)(reinterpret_cast<uintptr_t>(at) & 3), have = blocks - b;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(at - in);
    uint32_t w[N + 1];
#pragma unroll
    for (int i = 0; i <= N; i++) w[i] = 4 * i - in < have ? __ldg(words + i) : 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        out[i] = __funnelshift_r(w[i], w[i + 1], 8 * in);
        const int left = have - 4 * i;
        if (left < 4) out[i] = left > 0 ? out[i] & ((1u << (8 * left)) - 1) : 0;
    }
}
// eight of them; wide: 2 when rows start on 16 bytes, 1 on 8
__device__ __forceinline__ uint2 eight_scales(const uint8_t* __restrict__ row, int b, int blocks, int wide) {
    if (wide && b + 8 <= blocks) return __ldg(reinterpret_cast<const uint2*>(row + b));
    uint32_t w[2];
    some_scales(row, b, blocks, w);
    return make_uint2(w[0], w[1]);
}
// sixteen, b a multiple of 16
__device__ __forceinline__ uint4 sixteen_scales(const uint8_t* __restrict__ row, int b, int blocks, int wide) {
    if (wide && b + 16 <= blocks) {
        if (wide == 2) return __ldg(reinterpret_cast<const uint4*>(row + b));
        const uint2 lo = __ldg(reinterpret_cast<const uint2*>(row + b)), hi = __ldg(reinterpret_cast<const uint2*>(row + b + 8));
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    uint32_t w[4];
    some_scales(row, b, blocks, w);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// limit: infinite when there is none (a branch for each pair of values kept them from overlapping: 140 cycles a value)
__device__ __forceinline__ float2 gated2(float2 gate, float2 up, float limit) {
    const Swiglu2 s = swiglu2<true>(gate, up, limit);
    return unpair(mul2(mul2(s.g, s.sig), s.u));
}

// ------------------------------------------------------------ weights on the MMA's M side
// For groups of few rows, which reading the weights bounds.  A tile is 256
// outputs (two blocks of 128; gated: 128 of gate and the same of up) x up to 64
// rows of x, the MMA's N, rounded up to 16 only.  A cluster of CTAs shares a
// tile's contracted dimension, so that one token through one matrix is read by
// most SMs; each leaves its f32 sums in its shared memory, and then each adds up
// its share of the outputs over all of them, in their order.  No partial sums in
// global memory, so calls need no workspace and may overlap; two CTAs fit on an
// SM, and one's start and end go on behind the other's loads.
//
// Warps: 0 loads codes and the weights' scales, 1 issues the MMAs, 2 finds the
// tile and brings the scales of x; all eight write the output.
constexpr int kFp4Threads = 256;
constexpr int kFp4Rows = 64;                 // most rows of x in a tile
constexpr int kFp4MaxStages = 6;
constexpr int kFp4TmemCols = 256;            // two accumulators of 64 columns, scales behind them
constexpr int kFp4TmemScales = 128;
constexpr int kFp4ScaleCols = 24;            // of one stage: weights 2 x 2 x 4, x 2 x 4
constexpr int kFp4Header = 1024;
__host__ __device__ inline int fp4_stage_bytes(int x_rows) { return x_rows * 128 + 2 * kFp4Tile + 3 * kFp4Scales; }

struct Fp4Tile {
    int group, pos, n;   // matrix, first row of x, rows (none: no such tile)
};

// The tile of rows number `at`, by one warp, in all its lanes.  Groups count as
// in group_tables; `report`: look at all of them and raise an error for offsets
// that make no sense.
__device__ inline Fp4Tile fp4_find(const Fp4Params& p, int at, bool report) {
    if (!p.offsets) return {0, at * kFp4Rows, min(max(p.T - at * kFp4Rows, 0), kFp4Rows)};
    const int lane = threadIdx.x & 31;
    Fp4Tile r{0, 0, 0};
    int before = 0, top = 0;
    bool bad = false, found = false;
    for (int g0 = 0; g0 < p.groups && (report || !found); g0 += 32) {
        const int g = g0 + lane;
        int a = 0, b = 0;
        if (g < p.groups) {
            a = p.offsets[g];
            b = p.offsets[g + 1];
        }
        int most = a;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) most = max(most, __shfl_up_sync(0xffffffffu, most, o));
        most = max(most, top);
        top = __shfl_sync(0xffffffffu, most, 31);
        if (a < most || a < 0 || b < a || b > p.T) {
            bad |= g < p.groups;
            a = b = 0;
        }
        const int tiles = (b - a + kFp4Rows - 1) / kFp4Rows;
        int scan = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        const int in = at - (before + scan - tiles);
        const uint32_t here = __ballot_sync(0xffffffffu, in >= 0 && in < tiles);
        if (here && !found) {
            const int from = __ffs(here) - 1;
            r.group = g0 + from;
            r.pos = __shfl_sync(0xffffffffu, a + in * kFp4Rows, from);
            r.n = __shfl_sync(0xffffffffu, min(b - a - in * kFp4Rows, kFp4Rows), from);
            found = true;
        }
        before += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (report && __any_sync(0xffffffffu, bad) && lane == 0) atomicOr(p.err, (int)ERR_BOUNDS);
    return r;
}

// f32 of a CTA of the cluster, at the address that `mine` has here
__device__ __forceinline__ float load_peer(uint32_t mine, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(mine), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// One output of row t for each lane (m = the lane's; absent ones are not
// written), in the type asked for
__device__ __forceinline__ void store_lane(const Fp4Params& p, long long t, int m, float v) {
    if (m >= p.M) return;
    if (p.type == 0) reinterpret_cast<float*>(p.out)[t * p.ld_out + m] = v;
    else if (p.type == 1) reinterpret_cast<__half*>(p.out)[t * p.ld_out + m] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p.out)[t * p.ld_out + m] = __float2bfloat16_rn(v);
}
// a warp's 32 outputs from m0 on, a block, as 4-bit codes
__device__ __forceinline__ void store_lane4(const Fp4Params& p, long long t, int m0, float v) {
    if (m0 >= p.M) return;
    const int lane = threadIdx.x & 31;
    v = m0 + lane < p.M ? v : 0.f;
    const uint32_t scale = fp4_scale(__reduce_max_sync(0xffffffffu, magnitude(v)));
    uint32_t c;
    asm("{\n .reg .b8 a;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n mov.b32 %0, {a, a, a, a};\n}"
        : "=r"(c)
        : "f"(v * fp4_inverse(scale)), "f"(0.f));
    c = scale == 255 ? 0 : (c & 15) << (4 * (lane & 7));
    c |= __shfl_xor_sync(0xffffffffu, c, 1);
    c |= __shfl_xor_sync(0xffffffffu, c, 2);
    c |= __shfl_xor_sync(0xffffffffu, c, 4);
    uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + t * p.ld_out + m0 / 2;   // rows of codes start on 16 bytes
    if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(out)[lane >> 3] = c;
    if (lane == 0) p.out_scales[t * p.ld_os + m0 / kFp4Block] = (uint8_t)scale;
}

template <int MODE>
__global__ void __launch_bounds__(kFp4Threads, 2)
fp4_split_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                 const __grid_constant__ Fp4Params p, int stages, int x_rows /* room for rows of x in a stage */) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm);   // [stages] copies are there: the weights', those of x
    uint64_t* x_full = full + kFp4MaxStages;            // [stages] scales of x are there
    uint64_t* done = x_full + kFp4MaxStages;            // [stages] their MMAs are done
    uint64_t* done_bar = done + kFp4MaxStages;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + 512);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + 516);
    volatile uint32_t* issued = reinterpret_cast<volatile uint32_t*>(sm + 520);   // stages, once their warp is through
    Fp4Tile* found = reinterpret_cast<Fp4Tile*>(sm + 528);
    const uint32_t stage_bytes = fp4_stage_bytes(x_rows);
    // a stage: codes of x, codes of both blocks, their scales, scales of x
    const uint32_t w_off = x_rows * 128, ws_off = w_off + 2 * kFp4Tile, xs_off = ws_off + 2 * kFp4Scales;
    uint8_t* ring = sm + kFp4Header;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const int tile = blockIdx.x / ranks, row_tile = tile % p.row_tiles, block = tile / p.row_tiles;
    constexpr int kBlock = MODE == kFp4Plain ? 128 : 64;   // outputs of a block
    const int m0 = block * 2 * kBlock;
    const int k0 = (int)((long long)p.steps * rank / ranks), k1 = (int)((long long)p.steps * (rank + 1) / ranks);
    // one matrix: its first stages are asked for before the kernel before has ended, which does not write it
    const int early = p.groups == 1 ? min(stages, k1 - k0) : 0;
    // a stage's copies of the weights, by one thread
    auto load_stage = [&](uint32_t slot, int k, int group) {
        uint8_t* st = ring + slot * stage_bytes;
        mbar_arrive_expect_tx(&full[slot], (uint32_t)(2 * kFp4Tile + 2 * kFp4Scales));
#pragma unroll
        for (int b = 0; b < 2; b++) {
            load_weights<MODE != kFp4Plain>(st + w_off + b * kFp4Tile, &w_map, k * 128, m0 + b * kBlock, group, &full[slot]);
            const long long unit = (long long)group * p.units + min(m0 / kBlock + b, p.units - 1);   // an absent second block is not stored
            bulk_g2s(st + ws_off + b * kFp4Scales, p.w_scales + (unit * p.steps + k) * kFp4Scales, kFp4Scales, &full[slot]);
        }
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; i++) {
            mbar_init(&full[i], 2);
            mbar_init(&x_full[i], 1);
            mbar_init(&done[i], 1);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        *issued = 0;
        fence_barrier_init();
        pdl_trigger();
        for (int i = 0; i < early; i++) load_stage(i, k0 + i, 0);
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), kFp4TmemCols);
    pdl_start();   // nothing before this reads or writes global memory, but for the weights
    if (warp == 2) {
        const Fp4Tile t = fp4_find(p, row_tile, blockIdx.x == 0);
        if (lane == 0) *found = t;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Fp4Tile t = *found;
    if (t.n == 0) {   // (for all of the cluster)
        if (threadIdx.x == 0)
            for (int i = 0; i < early; i++) {   // copies land before the CTA exits
                mbar_arrive(&full[i]);
                mbar_wait(&full[i], 0u);
            }
        if (warp == 1) tmem_dealloc(tmem, kFp4TmemCols);
        return;
    }
    const WaitCtl ctl{abort_flag, p.err};
    const uint32_t full0 = smem_u32(full), x_full0 = smem_u32(x_full), done0 = smem_u32(done);
    const int boxes = (t.n + 15) >> 4;

    if (warp == 0) {
        // ------------------------------------------------ codes and the weights' scales
        Ring r;
        uint32_t n_issued = 0;
        for (int k = k0; k < k1; k++) {
            // (the early stages go through whatever happens: their weights are on their way)
            if (k >= k0 + early && !bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) break;
            if (elect_one()) {
                if (k >= k0 + early) load_stage(r.i, k, t.group);
                mbar_arrive_expect_tx(&full[r.i], (uint32_t)(boxes * 2048));
                for (int b = 0; b < boxes; b++)
                    tma_load_2d(ring + r.i * stage_bytes + b * 2048, &x_map, k * 128, t.pos + 16 * b, &full[r.i]);
            }
            __syncwarp();
            r.next(stages);
            n_issued++;
        }
        if (lane == 0) *issued = n_issued;
    } else if (warp == 1) {
        // ------------------------------------------------ MMAs (one thread issues)
        Ring r;
        const uint32_t ring0 = smem_u32(ring);
        const uint64_t x_desc = sw128_desc(ring0), w_desc = sw128_desc(ring0 + w_off);
        const uint64_t ws_desc = scale_desc(ring0 + ws_off), xs_desc = scale_desc(ring0 + xs_off);
        const uint32_t idesc = umma_idesc_mxf4(128, (t.n + 15) & ~15, 0), odd = umma_idesc_mxf4(0, 0, 2) & ~umma_idesc_mxf4(0, 0, 0);
        for (int k = k0; k < k1; k++) {
            if (!bar_wait(full0 + 8 * r.i, r.phase, ctl) || !bar_wait(x_full0 + 8 * r.i, r.phase, ctl)) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t at = r.i * stage_bytes >> 4;
                const uint32_t ws = tmem + kFp4TmemScales + kFp4ScaleCols * ((k - k0) & 1), xs = ws + 16;
#pragma unroll
                for (int u = 0; u < 4; u++) scales_to_tmem<1>(ws + 4 * u, ws_desc + at + u * (512 >> 4));   // block u / 2, half u % 2
#pragma unroll
                for (int u = 0; u < 2; u++) scales_to_tmem<1>(xs + 4 * u, xs_desc + at + u * (512 >> 4));
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int b = 0; b < 2; b++)
                        umma_mxf4<1>(tmem + 64 * b, w_desc + at + b * (kFp4Tile >> 4) + 2 * j, x_desc + at + 2 * j,
                                     j & 1 ? idesc | odd : idesc, ws + 8 * b + 4 * (j >> 1), xs + 4 * (j >> 1), k > k0 || j > 0);
                umma_commit(&done[r.i]);
            }
            __syncwarp();
            r.next(stages);
        }
        // every MMA of this CTA has completed before its sums are read (or tensor memory is released)
        if (elect_one()) umma_commit(done_bar);
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------ scales of x: rows lane and lane + 32, four stages' at a time
        Ring r;
        const uint8_t* row = p.x_scales + (long long)(t.pos + lane) * p.ld_xs;
        bool ok = true;
        for (int k4 = k0; k4 < k1 && ok; k4 += 4) {
            uint2 four[2][4];   // (by eights: a CTA's first stage may begin inside sixteen)
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    four[c][j] = lane + 32 * c < t.n && k4 + j < k1 ? eight_scales(row + 32 * c * p.ld_xs, 8 * (k4 + j), p.blocks, p.wide_xs)
                                                                    : make_uint2(0, 0);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (k4 + j >= k1) break;
                if (!bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                uint4* to = reinterpret_cast<uint4*>(ring + r.i * stage_bytes + xs_off) + lane;
                to[0] = make_uint4(four[0][j].x, four[1][j].x, 0, 0);
                to[32] = make_uint4(four[0][j].y, four[1][j].y, 0, 0);
                fence_async();
                __syncwarp();
                if (lane == 0) bar_arrive(x_full0 + 8 * r.i);
                r.next(stages);
            }
        }
    }
    __syncwarp();
    // ---------------- every warp: the sums into shared memory, [row of x][output], where the ring was
    mbar_wait(done_bar, 0u);   // (of MMAs that were issued: it comes)
    tc_fence_after();
    __syncthreads();           // no role still waits on the ring
    float* sums = reinterpret_cast<float*>(ring);
    if (threadIdx.x == 0 && *abort_flag) drain_own(full, *issued, stages);
    __syncthreads();
    {
        const int quarter = warp & 3, b = warp >> 2;
        for (int c = 0; c < t.n; c += 16) {
            float v[16];
            tmem_ld16_now(tmem + ((uint32_t)(32 * quarter) << 16) + 64 * b + c, v);
#pragma unroll
            for (int i = 0; i < 16; i++) sums[(c + i) * 256 + 128 * b + 32 * quarter + lane] = v[i];
        }
    }
    tc_fence_before();
    cluster_sync_all();
    if (warp == 1) tmem_dealloc(tmem, kFp4TmemCols);
    // ---------------- this CTA's share of (row, 32 outputs), over all of the cluster
    constexpr int per_row = MODE == kFp4Plain ? 8 : 4;
    const uint32_t mine = smem_u32(sums);
    for (int i = rank + ranks * warp; i < t.n * per_row && !*abort_flag; i += ranks * (kFp4Threads / 32)) {
        const int row = i / per_row, o = 32 * (i % per_row), j = o + lane;
        // (gated: 16 of gate, 16 of up, and so on)
        const uint32_t at = mine + 4 * (row * 256 + (MODE == kFp4Plain ? j : 2 * j - (j & 15)));
        float y = 0.f, up = 0.f;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if (q >= (int)ranks) break;
            y += load_peer(at, q);
            if (MODE != kFp4Plain) up += load_peer(at + 64, q);
        }
        const long long to = t.pos + row;
        if (MODE == kFp4Plain) {
            store_lane(p, to, m0 + o + lane, y);
        } else {
            const float h = gated2(make_float2(y, y), make_float2(up, up), p.limit).x;
            if (MODE == kFp4Gated) store_lane(p, to, m0 + o + lane, h);
            else store_lane4(p, to, m0 + o, h);
        }
    }
    cluster_sync_all();   // the others may still read this CTA's sums
}

// ------------------------------------------------------------ rows of x on the MMA's M side
// For groups of many rows, which the tensor cores bound.  A pair of SMs
// (cta_group::2) shares a tile of 256 rows of x times 256 outputs (gated: 128
// features): each CTA loads 128 rows of x and 128 of the weights, 32 KB of codes for 256 contracted values, 64 bytes a
// cycle at the full MMA rate.
//
// Tensor memory holds two accumulators of 256 columns but for the scales' 48
// columns: the second begins 48 before the first ends, and a tile's MMAs wait
// for the epilogue of the one before to have read its accumulator (a few hundred
// cycles, in which the ring of stages fills up).
//
// Warps: 0 loads codes and the weights' scales, 1 issues the MMAs (in the
// pair's first CTA), 2 and 3 bring the scales of x, 4-11
// write the output: lane quarter (warp & 3), half of the columns (warp >= 8).
constexpr int kFp4PairThreads = 384;
constexpr int kFp4PairStages = 5;
constexpr int kFp4PairTx = 2 * kFp4Tile + 2 * kFp4Scales;            // bytes of a CTA's copies of a stage
constexpr int kFp4PairStage = kFp4PairTx + kFp4Scales;               // and the scales of x
constexpr int kFp4PairSecond = 208, kFp4PairTmemScales = 464;
constexpr int kFp4PairOut = 32 * 144;          // a warp's room for rows on their way out: 32 of 128 bytes, 16 apart
constexpr int kFp4PairTableOff = 1024;
constexpr int kFp4PairRegsFew = 72, kFp4PairRegsMany = 216;
constexpr int kFp4PairRegs = 128 * kFp4PairRegsFew + 256 * kFp4PairRegsMany;
static_assert(kFp4PairRegs <= kFp4PairThreads * 168, "register split");
__host__ __device__ inline int fp4_pair_stage_off(int groups) { return (kFp4PairTableOff + 12 * (groups + 1) + 1023) / 1024 * 1024; }

// the first CTA's barriers, as drain_pair moves them on
struct Fp4PairBars {
    uint64_t* full;
    __device__ void expect(uint32_t slot) { mbar_arrive_expect_tx(&full[slot], kFp4PairTx); }
    __device__ void complete(uint32_t slot) {
        asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[slot])),
                     "r"((uint32_t)kFp4PairTx)
                     : "memory");
    }
    __device__ void wait(uint32_t slot, uint32_t parity) { mbar_wait(&full[slot], parity); }
};
// A warp's 32 rows of 2 N outputs each (a lane holds a row) to out, by way of
// shared memory, so that a store's lanes write neighbouring outputs, of four
// rows at once.  left: how many of a row's exist; rows: how many rows do.
template <typename T, int N>
__device__ __forceinline__ void store_rows(T* out, long long ld, int left, int rows, const float2 (&v)[N], uint8_t* room, bool wide) {
    constexpr int C = 128 / sizeof(T);   // outputs of a row in one go
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 2 * N; c += C) {
        if (c >= left) break;
        __syncwarp();
        uint4* to = reinterpret_cast<uint4*>(room + 144 * lane);
#pragma unroll
        for (int i = 0; i < 8; i++) {   // 16 bytes each
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (sizeof(T) == 4) {
                    const float2 f = v[c / 2 + 2 * i + k / 2];
                    w[k] = __float_as_uint(k & 1 ? f.y : f.x);
                } else {
                    const float2 f = v[c / 2 + 4 * i + k];
                    const T h[2] = {round_to<T>(f.x), round_to<T>(f.y)};
                    memcpy(&w[k], h, 4);
                }
            }
            to[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        if (wide && c + C <= left) {
            const int r0 = lane >> 3, at = 16 * (lane & 7);
            uint8_t* o = reinterpret_cast<uint8_t*>(out + r0 * ld + c) + at;
#pragma unroll
            for (int r = 0; r < 32; r += 4)
                if (r + r0 < rows) *reinterpret_cast<uint4*>(o + r * ld * (long long)sizeof(T)) = *reinterpret_cast<const uint4*>(room + 144 * (r + r0) + at);
        } else {   // one output a lane
            for (int r = 0; r < min(rows, 32); r++)
#pragma unroll
                for (int k = 0; k < C; k += 32)
                    if (c + k + lane < left) out[r * ld + c + k + lane] = reinterpret_cast<const T*>(room + 144 * r)[k + lane];
        }
    }
}
// 2 N outputs of a row in 4-bit blocks, m of them (from a block's start on)
template <int N>
__device__ __forceinline__ void store_row4(uint8_t* codes, uint8_t* scales, int left, const float2 (&h)[N]) {
#pragma unroll
    for (int b = 0; b < N / 16; b++) {
        if (32 * b >= left) return;
        float v[4][8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const float2 f = h[16 * b + i / 2];
            const float x = 32 * b + i < left ? (i & 1 ? f.y : f.x) : 0.f;
            v[i >> 3][i & 7] = x;
            m = max(m, magnitude(x));
        }
        const uint32_t scale = fp4_scale(m);
        reinterpret_cast<uint4*>(codes)[b] = make_uint4(e2m1x8(v[0], scale), e2m1x8(v[1], scale), e2m1x8(v[2], scale), e2m1x8(v[3], scale));
        scales[b] = (uint8_t)scale;
    }
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFp4PairThreads, 1)
fp4_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap s_map,
                const __grid_constant__ CUtensorMap x_map, const __grid_constant__ Fp4Params p, int wide_out) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm);   // first CTA: both CTAs' copies are there
    uint64_t* x_full = full + kFp4PairStages;           // first CTA: both CTAs' scales of x are there
    uint64_t* done = x_full + kFp4PairStages;           // both: the stage's MMAs are done
    uint64_t* tile_done = done + kFp4PairStages;        // [2] both: a tile's are
    uint64_t* tile_read = tile_done + 2;                // first CTA: both epilogues have read an accumulator
    uint64_t* done_bar = tile_read + 1;
    uint64_t* left_bar = done_bar + 1;                  // both, when the first CTA gave up: its commits are through
    __shared__ volatile int given_up;
    __shared__ volatile uint32_t from_peer, issued;     // issued: stages, once their warp is through
    volatile int* abort_flag = &given_up;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + 776);
    int32_t* first_tile = reinterpret_cast<int32_t*>(sm + kFp4PairTableOff);
    int32_t* start = first_tile + p.groups + 1;
    int32_t* rows = start + p.groups + 1;
    uint8_t* ring = sm + fp4_pair_stage_off(p.groups);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;   // in the pair: the cluster is two CTAs along x
    constexpr int kOut = MODE == kFp4Plain ? 256 : 128;   // outputs of a tile
    if (threadIdx.x == 0) {
        for (int i = 0; i < kFp4PairStages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&x_full[i], 4);
            mbar_init(&done[i], 1);
        }
        mbar_init(&tile_done[0], 1);
        mbar_init(&tile_done[1], 1);
        mbar_init(tile_read, 16);
        mbar_init(done_bar, 1);
        mbar_init(left_bar, 1);
        *abort_flag = 0;
        issued = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pdl_start();   // nothing before this reads or writes global memory
    if (warp == 2) group_tables(p.offsets, p.groups, p.T, p.err, first_tile, start, rows, 256, (p.M + kOut - 1) / kOut, blockIdx.x == 0);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers are ready
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const WaitCtl ctl{abort_flag, p.err};
    const uint32_t done0 = smem_u32(done);
    const int tiles = first_tile[p.groups], pairs = gridDim.x >> 1, steps = p.steps;

    struct Tile {
        int group, m;      // matrix, first output
        int pos, rows;     // first row of x of this CTA, rows of the group from there on
    };
    // the tiles of one block of outputs follow each other, so its weights come from HBM once
    auto tile_at = [&](int i) {
        int lo = 0, hi = p.groups;   // the last group with first_tile <= i has rows
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first_tile[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int blocks = (rows[lo] + 255) >> 8, in = i - first_tile[lo];
        const int n = in / blocks, at = (in - n * blocks) * 256 + 128 * (int)rank;
        return Tile{lo, n * kOut, start[lo] + at, rows[lo] - at};
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4PairRegsFew));
        if (warp == 0) {
            // -------------------------------------------- codes and the weights' scales
            bool ok = true;
            Ring r;
            uint32_t n_issued = 0;
            const uint32_t full0 = map_to_rank0(smem_u32(full)), ring0 = smem_u32(ring);
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
                const Tile t = tile_at(i);
                // this CTA's half of the weights; both have all scales
                const int m = t.m + kOut / 2 * (int)rank;
                const int s0 = (t.group * p.units + t.m / (kOut / 2)) * steps * 4, s1 = s0 + steps * 4;
                for (int k = 0; k < steps; k++) {
                    if (!bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                    if (elect_one()) {
                        const uint32_t st = ring0 + r.i * kFp4PairStage, bar = full0 + 8 * r.i;
                        if (rank == 0) mbar_arrive_expect_tx(&full[r.i], 2 * kFp4PairTx);
                        // (no rows for this CTA: from past the end, which is zeros and no traffic)
                        tma_pair_2d(st, &x_map, k * 128, t.rows > 0 ? t.pos : p.T, bar);
                        load_weights_pair<MODE != kFp4Plain>(st + kFp4Tile, &w_map, k * 128, m, t.group, bar);
                        tma_pair_2d(st + 2 * kFp4Tile, &s_map, 0, s0 + 4 * k, bar);
                        tma_pair_2d(st + 2 * kFp4Tile + kFp4Scales, &s_map, 0, s1 + 4 * k, bar);
                    }
                    __syncwarp();
                    r.next(kFp4PairStages);
                    n_issued++;
                }
            }
            if (lane == 0) issued = n_issued;
        } else if (warp == 1 && rank == 0) {
            // -------------------------------------------- MMAs (one thread issues for both CTAs)
            bool ok = true;
            Ring r;
            uint32_t n = 0, buffer = 0;   // tiles; of scales
            const uint32_t full0 = smem_u32(full), x_full0 = smem_u32(x_full), ring0 = smem_u32(ring);
            const uint64_t x_desc = sw128_desc(ring0), w_desc = sw128_desc(ring0 + kFp4Tile);
            const uint64_t ws_desc = scale_desc(ring0 + 2 * kFp4Tile), xs_desc = scale_desc(ring0 + kFp4PairTx);
            constexpr uint32_t idesc[2] = {umma_idesc_mxf4(256, 256, 0), umma_idesc_mxf4(256, 256, 2)};
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs, n++) {
                // the accumulator of the tile before has been read
                if (n > 0 && !bar_wait(smem_u32(tile_read), (n - 1) & 1u, ctl)) break;
                const uint32_t d = tmem + (n & 1 ? kFp4PairSecond : 0);
                for (int k = 0; k < steps; k++) {
                    if (!bar_wait(full0 + 8 * r.i, r.phase, ctl) || !bar_wait(x_full0 + 8 * r.i, r.phase, ctl)) { ok = false; break; }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t at = r.i * (kFp4PairStage >> 4);
                        const uint32_t xs = tmem + kFp4PairTmemScales + kFp4ScaleCols * buffer, ws = xs + 8;
#pragma unroll
                        for (int u = 0; u < 2; u++) {   // half of the stage's contracted values
                            scales_to_tmem<2>(xs + 4 * u, xs_desc + at + u * (512 >> 4));
                            scales_to_tmem<2>(ws + 8 * u, ws_desc + at + u * (512 >> 4));
                            scales_to_tmem<2>(ws + 8 * u + 4, ws_desc + at + (kFp4Scales + u * 512 >> 4));
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            umma_mxf4<2>(d, x_desc + at + 2 * j, w_desc + at + 2 * j, idesc[j & 1], xs + 4 * (j >> 1), ws + 8 * (j >> 1), k > 0 || j > 0);
                        umma_commit_pair(done0 + 8 * r.i);
                        if (k + 1 == steps) umma_commit_pair(smem_u32(tile_done) + 8 * (n & 1));
                    }
                    __syncwarp();
                    r.next(kFp4PairStages);
                    buffer ^= 1;
                }
            }
            // every MMA has completed before tensor memory is released
            if (elect_one()) {
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(done_bar)) : "memory");
                mbar_wait(done_bar, 0u);
            }
            __syncwarp();
        } else if (warp >= 2) {
            // -------------------------------------------- scales of x: rows 64 (warp - 2) + lane and + 32 of the CTA's
            // Four stages' at a time.  The next four's are asked for behind the last of these: a fence waits for loads that
            // are on their way, and with these ahead of it cost up to a quarter of the time.
            bool ok = true;
            Ring r;
            const int first = 64 * (warp - 2) + lane;
            const uint32_t x_full0 = map_to_rank0(smem_u32(x_full));
            uint4 four[2][2];   // [row][half]
            auto load = [&](const Tile& t, int k) {
                const uint8_t* row = p.x_scales + (long long)(t.pos + first) * p.ld_xs;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const bool in = first + 32 * c < t.rows;
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        four[c][h] = in ? sixteen_scales(row + 32 * c * p.ld_xs, 8 * k + 16 * h, p.blocks, p.wide_xs) : make_uint4(0, 0, 0, 0);
                }
            };
            int i = blockIdx.x >> 1;
            if (i < tiles) load(tile_at(i), 0);
            for (; i < tiles && ok; i += pairs) {
                const Tile t = tile_at(i);
                for (int k4 = 0; k4 < steps && ok; k4 += 4) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (k4 + j >= steps) break;
                        const uint4 a = four[0][j >> 1], b = four[1][j >> 1];
                        if (!bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                        uint2* to = reinterpret_cast<uint2*>(ring + r.i * kFp4PairStage + kFp4PairTx) + 2 * lane + (warp - 2);
                        to[0] = j & 1 ? make_uint2(a.z, b.z) : make_uint2(a.x, b.x);
                        to[64] = j & 1 ? make_uint2(a.w, b.w) : make_uint2(a.y, b.y);
                        fence_async();
                        __syncwarp();
                        if (lane == 0) bar_arrive_cluster(x_full0 + 8 * r.i);
                        r.next(kFp4PairStages);
                    }
                    if (k4 + 4 < steps) load(t, k4 + 4);
                    else if (i + pairs < tiles) load(tile_at(i + pairs), 0);
                }
            }
        }
    } else {
        // ------------------------------------------------ output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp4PairRegsMany));
        const int half = (warp - 4) >> 2;
        uint8_t* room = ring + kFp4PairStages * kFp4PairStage + (warp - 4) * kFp4PairOut;
        const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t read0 = map_to_rank0(smem_u32(tile_read));
        uint32_t n = 0;
        for (int i = blockIdx.x >> 1; i < tiles; i += pairs, n++) {
            const Tile t = tile_at(i);
            if (!bar_wait(smem_u32(tile_done) + 8 * (n & 1), (n >> 1) & 1u, ctl)) break;
            tc_fence_after();
            const uint32_t from = taddr + (n & 1 ? kFp4PairSecond : 0);
            float2 acc[64];   // 128 columns
            if (t.rows > 32 * (warp & 3)) {
#pragma unroll
                for (int h = 0; h < 4; h++)
                    tmem_ld32(from + 128 * half + 32 * h, reinterpret_cast<float*>(acc + 16 * h));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(read0);
            const int r0 = 32 * (warp & 3);   // the warp's first row
            if (t.rows > r0) {
                const long long at = t.pos + r0;
                if (MODE == kFp4Plain) {
                    const int m = t.m + 128 * half;
                    const long long o = at * p.ld_out + m;
                    if (p.type == 0) store_rows(reinterpret_cast<float*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, acc, room, wide_out);
                    else if (p.type == 1) store_rows(reinterpret_cast<__half*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, acc, room, wide_out);
                    else store_rows(reinterpret_cast<__nv_bfloat16*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, acc, room, wide_out);
                } else {
                    float2 h[32];
#pragma unroll
                    for (int c = 0; c < 32; c++) h[c] = gated2(acc[2 * c - (c & 7)], acc[2 * c - (c & 7) + 8], p.limit);
                    const int m = t.m + 64 * half;
                    const long long o = at * p.ld_out + m;
                    if (MODE == kFp4GatedRows) {
                        if (lane < t.rows - r0)
                            store_row4(reinterpret_cast<uint8_t*>(p.out) + (at + lane) * p.ld_out + m / 2, p.out_scales + (at + lane) * p.ld_os + m / kFp4Block, p.M - m, h);
                    } else if (p.type == 0) {
                        store_rows(reinterpret_cast<float*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, h, room, wide_out);
                    } else if (p.type == 1) {
                        store_rows(reinterpret_cast<__half*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, h, room, wide_out);
                    } else {
                        store_rows(reinterpret_cast<__nv_bfloat16*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, h, room, wide_out);
                    }
                }
            }
            __syncwarp();
        }
    }
    // ---------------- teardown: every role of both CTAs is done (or gave up); free tensor memory
    tc_fence_before();
    __syncthreads();
    // (as in fp8_pair_kernel: the first CTA learns how many stages the other has issued, which learns whether to stay)
    if (threadIdx.x == 0) store_peer(const_cast<uint32_t*>(&from_peer), rank ^ 1, rank == 0 ? (uint32_t)given_up : issued);
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    if (rank == 0 ? given_up != 0 : from_peer != 0) {
        if (rank == 0 && threadIdx.x == 0) {
            Fp4PairBars bars{full};
            drain_pair(issued, from_peer, kFp4PairStages, bars);
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

// ------------------------------------------------------------ pairs with weights on the MMA's M side
// The same pair of SMs with the operands' places changed: 256 outputs (gated: 128
// features) on the M side, up to 384 rows of x on the N side, rounded up to 32
// only and shared evenly among a group's tiles.  Groups whose rows are no
// multiple of 256 cost what their rows cost, and the weights of a group of up to
// 384 rows are loaded once.  Past 256 rows a step takes two MMAs, of 128 rows and
// of the others.
//
// A lane of tensor memory is an output.  For the gated product the lanes of gate
// and of up exchange half of their columns, so that each has both sums of 16 rows;
// on their way into 4-bit rows, whose blocks are two warps', they meet in shared
// memory, 32 rows of x at a time, [row][feature] in f32.
//
// Two accumulators where two neighbouring tiles have 224 rows at most; else a
// tile's MMAs wait for the one before to be read.
//
// The scales of x go through registers, and a fence between what they write to
// shared memory and the copy to tensor memory waits for loads of the same warp
// that are on their way (a quarter of the time went there).  So the warps that
// load and write them do not fence: they tell another one, which does.
//
// Warps: 0 loads codes and the weights' scales, 1 issues the MMAs (in the
// pair's first CTA), 2 fences, 4-7 bring the scales of x (in both CTAs), 8-11 and
// 12-15 write the output, every second 32 rows each.
constexpr int kFp4FitThreads = 512;
constexpr int kFp4FitMaxStages = 8;
constexpr int kFp4FitRows = 384;
constexpr int kFp4FitSecond = 224, kFp4FitTmemScales = 448, kFp4FitScaleCols = 32;
constexpr int kFp4FitRoom = 32 * 80 * 4;       // four warps' room for 32 rows on their way into 4 bits
constexpr int kFp4FitRegsFew = 56, kFp4FitRegsMany = 200;
constexpr int kFp4FitRegs = 256 * kFp4FitRegsFew + 256 * kFp4FitRegsMany;
static_assert(kFp4FitRegs <= kFp4FitThreads * 128, "register split");
// a stage: codes of the weights, of x (a CTA's half of up to `rows`, the most that a tile has), scales of the weights, of x
__host__ __device__ inline int fp4_fit_codes(int rows) { return kFp4Tile + rows / 2 * 128; }
__host__ __device__ inline int fp4_fit_stage(int rows) { return fp4_fit_codes(rows) + kFp4Scales + (rows + 127) / 128 * kFp4Scales; }

struct Fp4RowMaps {
    CUtensorMap rows[4];   // x in boxes of 256 columns x 16, 32, 64 and 128 rows
};
// the first CTA's barriers, as drain_pair moves them on; the tiles' stages have different numbers of bytes
struct Fp4FitBars {
    uint64_t* full;
    volatile uint32_t* bytes;   // a CTA's share of the stage that it issued last in each slot
    __device__ uint32_t peer_bytes(uint32_t slot) const {
        uint32_t a, v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 1;" : "=r"(a) : "r"(smem_u32(const_cast<uint32_t*>(&bytes[slot]))));
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
        return v;
    }
    __device__ void expect(uint32_t slot) { mbar_arrive_expect_tx(&full[slot], peer_bytes(slot)); }
    __device__ void complete(uint32_t slot) {
        asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[slot])), "r"(bytes[slot])
                     : "memory");
    }
    __device__ void wait(uint32_t slot, uint32_t parity) { mbar_wait(&full[slot], parity); }
};

// whether it holds for all of `threads`, which meet here
__device__ __forceinline__ bool all_of(int barrier, int threads, bool holds) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r)
                 : "r"((uint32_t)holds), "r"(barrier), "r"(threads)
                 : "memory");
    return r != 0;
}
// 32 columns of this warp's lanes of tensor memory, which are there after loaded()
__device__ __forceinline__ void tmem_ld32_later(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
template <int N>
__device__ __forceinline__ void loaded(float (&v)[N][32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 32; j++) asm volatile("" : "+f"(v[i][j]));   // (no use of the registers before the wait)
}
// Output m of rows first, first + step, ..., of which `have` count from row t on,
// by a lane; a warp's lanes write neighbouring outputs.  No way through shared
// memory: copies and MMAs leave its ports little time (32 rows of 128 outputs
// took 1900 cycles that way).
template <typename T, int N>
__device__ __forceinline__ void store_outputs(const Fp4Params& p, long long t, int first, int step, int have, int m, const float (&v)[N]) {
    if (m >= p.M) return;
    T* out = reinterpret_cast<T*>(p.out) + (t + first) * p.ld_out + m;
    const long long ahead = step * p.ld_out;
#pragma unroll
    for (int c = 0; c < N; c++) {
        if (first + c * step < have) *out = round_to<T>(v[c]);
        out += ahead;
    }
}
template <int N>
__device__ __forceinline__ void store_outputs(const Fp4Params& p, long long t, int first, int step, int have, int m, const float (&v)[N]) {
    if (p.type == 0) store_outputs<float>(p, t, first, step, have, m, v);
    else if (p.type == 1) store_outputs<__half>(p, t, first, step, have, m, v);
    else store_outputs<__nv_bfloat16>(p, t, first, step, have, m, v);
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFp4FitThreads, 1)
fp4_fit_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap s_map,
               const __grid_constant__ Fp4RowMaps x_maps, const __grid_constant__ Fp4Params p, int stages,
               int x_rows /* most rows of x in a tile */) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm);   // first CTA: both CTAs' copies are there
    uint64_t* x_full = full + kFp4FitMaxStages;         // first CTA: both CTAs' scales of x are there
    uint64_t* x_written = x_full + kFp4FitMaxStages;    // its own are written
    uint64_t* done = x_written + kFp4FitMaxStages;      // both: the stage's MMAs are done
    uint64_t* tile_done = done + kFp4FitMaxStages;         // [2] both: a tile's are
    uint64_t* tile_read = tile_done + 2;                // [2] first CTA: both epilogues have read an accumulator
    uint64_t* done_bar = tile_read + 2;
    uint64_t* left_bar = done_bar + 1;                  // both, when the first CTA gave up: its commits are through
    __shared__ volatile int given_up;
    __shared__ volatile uint32_t from_peer, issued;     // issued: stages, once their warp is through
    __shared__ volatile uint32_t bytes[kFp4FitMaxStages];
    volatile int* abort_flag = &given_up;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + 776);
    int32_t* first_tile = reinterpret_cast<int32_t*>(sm + kFp4PairTableOff);
    int32_t* start = first_tile + p.groups + 1;
    int32_t* rows = start + p.groups + 1;
    uint8_t* ring = sm + fp4_pair_stage_off(p.groups);
    const uint32_t stage_bytes = fp4_fit_stage(x_rows), ws_off = fp4_fit_codes(x_rows), xs_off = ws_off + kFp4Scales;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;   // in the pair: the cluster is two CTAs along x
    constexpr int kHalf = MODE == kFp4Plain ? 128 : 64;   // outputs of a CTA in a tile
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&x_full[i], 2);
            mbar_init(&x_written[i], 4);
            mbar_init(&done[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&tile_done[i], 1);
            mbar_init(&tile_read[i], 16);
        }
        mbar_init(done_bar, 1);
        mbar_init(left_bar, 1);
        *abort_flag = 0;
        issued = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pdl_start();   // nothing before this reads or writes global memory
    if (warp == 2) group_tables(p.offsets, p.groups, p.T, p.err, first_tile, start, rows, x_rows, (p.M + 2 * kHalf - 1) / (2 * kHalf), blockIdx.x == 0);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // the peer's barriers are ready
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const WaitCtl ctl{abort_flag, p.err};
    const uint32_t done0 = smem_u32(done);
    const int tiles = first_tile[p.groups], pairs = gridDim.x >> 1, steps = p.steps;

    struct Tile {
        int group, m;      // matrix, first output of the pair
        int pos, n;        // first row of x, rows
        int cols;          // n in whole 32s: columns of the accumulator
    };
    // the tiles of one block of outputs follow each other, so its weights come from HBM once
    auto tile_at = [&](int i) {
        int lo = 0, hi = p.groups;   // the last group with first_tile <= i has rows
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first_tile[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int blocks = (rows[lo] + x_rows - 1) / x_rows, in = i - first_tile[lo], m = in / blocks;
        const int per = ((rows[lo] + blocks - 1) / blocks + 31) & ~31, at = (in - m * blocks) * per, n = min(per, rows[lo] - at);
        return Tile{lo, m * 2 * kHalf, start[lo] + at, n, (n + 31) & ~31};
    };

    // where in tensor memory a pair's n-th tile is
    auto place = [](uint32_t n, int cols) { return (n & 1) && cols <= kFp4FitSecond ? kFp4FitSecond : 0; };
    if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4FitRegsFew));
        if (warp == 0) {
            // -------------------------------------------- codes and the weights' scales
            bool ok = true;
            Ring r;
            uint32_t n_issued = 0;
            const uint32_t full0 = map_to_rank0(smem_u32(full)), ring0 = smem_u32(ring);
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
                const Tile t = tile_at(i);
                const int m = t.m + kHalf * (int)rank, first = t.cols > 256 ? 128 : t.cols;
                const uint32_t share = kFp4Tile + (t.cols >> 1) * 128 + kFp4Scales;
                // A copy for each lane: 0 the weights', 1 their scales, 2-5 and 6-9 this CTA's halves of the MMAs' rows of x,
                // a box for each power of two in their number.  (One thread with a loop over the boxes took up to 0.5 us a
                // stage; boxes of 16 rows cost more to issue than to load.)
                const int part = lane >= 6, box = (lane - 2) & 3, rows_of = (part ? t.cols - first : first) >> 1;
                const bool copies = lane < 2 || (lane < 10 && rows_of >> box & 16);
                const int below = rows_of & ((16 << box) - 1);   // rows of the boxes before
                const CUtensorMap* map = lane == 1 ? &s_map : &x_maps.rows[box];
                const uint32_t offset = lane == 1 ? ws_off : kFp4Tile + 128 * ((part ? first >> 1 : 0) + below);
                int x = 0, y = lane == 1 ? (t.group * p.units + m / kHalf) * steps * 4 : t.pos + (part ? first : 0) + rows_of * (int)rank + below;
                const int x_step = lane == 1 ? 0 : 128, y_step = lane == 1 ? 4 : 0;
                for (int k = 0; k < steps; k++) {
                    if (!bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                    const uint32_t st = ring0 + r.i * stage_bytes, bar = full0 + 8 * r.i;
                    if (lane == 0) {
                        bytes[r.i] = share;
                        if (rank == 0) mbar_arrive_expect_tx(&full[r.i], 2 * share);
                        load_weights_pair<MODE != kFp4Plain>(st, &w_map, k * 128, m, t.group, bar);
                    } else if (copies) {
                        tma_pair_2d(st + offset, map, x, y, bar);
                    }
                    x += x_step;
                    y += y_step;
                    __syncwarp();
                    r.next(stages);
                    n_issued++;
                }
            }
            if (lane == 0) issued = n_issued;
        } else if (warp == 1 && rank == 0) {
            // -------------------------------------------- MMAs (one thread issues for both CTAs)
            bool ok = true;
            Ring r;
            uint32_t n = 0, buffer = 0;   // tiles; of scales
            int before = 0, before_end = 0;   // the columns of the tile before
            const uint32_t full0 = smem_u32(full), x_full0 = smem_u32(x_full), ring0 = smem_u32(ring), read0 = smem_u32(tile_read);
            const uint32_t w_low = sw128_low(ring0), x_low = sw128_low(ring0 + kFp4Tile);
            const uint32_t ws_low = scale_low(ring0 + ws_off), xs_low = scale_low(ring0 + xs_off), base = uniform(tmem);
            const uint32_t odd = umma_idesc_mxf4(0, 0, 2) & ~umma_idesc_mxf4(0, 0, 0);
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs, n++) {
                const Tile t = tile_at(i);
                const uint32_t a = n & 1;
                const int cols = uniform(t.cols);
                const int at_col = place(n, cols), first = cols > 256 ? 128 : cols;
                const uint32_t d = base + at_col, idesc = umma_idesc_mxf4(256, first, 0), idesc2 = umma_idesc_mxf4(256, cols - first, 0);
                // the columns have been read: of the tile two before, and of the one before where they are the same
                if (n > 1 && !bar_wait(read0 + 8 * a, ((n >> 1) - 1) & 1u, ctl)) break;
                if (n > 0 && before < at_col + cols && at_col < before_end && !bar_wait(read0 + 8 * (a ^ 1), ((n - 1) >> 1) & 1u, ctl)) break;
                before = at_col;
                before_end = at_col + cols;
                for (int k = 0; k < steps; k++) {
                    if (!bar_wait_both(full0 + 8 * r.i, r.phase, x_full0 + 8 * r.i, r.phase, ctl)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = r.i * stage_bytes >> 4, wl = w_low + at, xl = x_low + at, wsl = ws_low + at, xsl = xs_low + at;
                    const uint32_t ws = base + kFp4FitTmemScales + kFp4FitScaleCols * buffer, xs = ws + 8;   // of x: 12 columns a half
                    const uint32_t more = k > 0;
                    if (elect_one()) {
#pragma unroll
                        for (int u = 0; u < 2; u++) {   // half of the stage's contracted values
                            scales_to_tmem<2>(ws + 4 * u, wide_desc(wsl + u * (512 >> 4), kScaleHigh));
                            scales_to_tmem<2>(xs + 12 * u, wide_desc(xsl + u * (512 >> 4), kScaleHigh));
                            if (cols > 128) scales_to_tmem<2>(xs + 12 * u + 4, wide_desc(xsl + (kFp4Scales + u * 512 >> 4), kScaleHigh));
                            if (cols > 256) scales_to_tmem<2>(xs + 12 * u + 8, wide_desc(xsl + (2 * kFp4Scales + u * 512 >> 4), kScaleHigh));
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint64_t wd = wide_desc(wl + 2 * j, kSw128High);
                            umma_mxf4<2>(d, wd, wide_desc(xl + 2 * j, kSw128High), j & 1 ? idesc | odd : idesc, ws + 4 * (j >> 1), xs + 12 * (j >> 1), j > 0 ? 1 : more);
                            if (cols > 256)
                                umma_mxf4<2>(d + 128, wd, wide_desc(xl + (64 * 128 >> 4) + 2 * j, kSw128High), j & 1 ? idesc2 | odd : idesc2,
                                             ws + 4 * (j >> 1), xs + 12 * (j >> 1) + 4, j > 0 ? 1 : more);
                        }
                        umma_commit_pair(done0 + 8 * r.i);
                        if (k + 1 == steps) umma_commit_pair(smem_u32(tile_done) + 8 * a);
                    }
                    __syncwarp();
                    r.next(stages);
                    buffer ^= 1;
                }
            }
            // every MMA has completed before tensor memory is released
            if (elect_one()) {
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(done_bar)) : "memory");
                mbar_wait(done_bar, 0u);
            }
            __syncwarp();
        } else if (warp == 2) {
            // -------------------------------------------- what the others wrote, handed over
            bool ok = true;
            Ring r;
            const uint32_t x_full0 = map_to_rank0(smem_u32(x_full)), x_written0 = smem_u32(x_written);
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
                for (int k = 0; k < steps; k++) {
                    if (!bar_wait(x_written0 + 8 * r.i, r.phase, ctl)) { ok = false; break; }
                    fence_async();
                    if (lane == 0) bar_arrive_cluster(x_full0 + 8 * r.i);
                    r.next(stages);
                }
            }
        } else if (warp >= 4) {
            // -------------------------------------------- scales of x: rows 32 (warp - 4) + lane, + 128, + 256 of the tile
            // (two stages' at a time, the next two's on their way)
            bool ok = true;
            Ring r;
            const int first = 32 * (warp - 4) + lane;
            const uint32_t x_written0 = smem_u32(x_written);
            uint4 next[3];
            auto load = [&](const Tile& t, int k) {
                const uint8_t* row = p.x_scales + (long long)(t.pos + first) * p.ld_xs;
#pragma unroll
                for (int v = 0; v < 3; v++)
                    next[v] = first + 128 * v < t.n ? sixteen_scales(row + 128 * v * p.ld_xs, 8 * k, p.blocks, p.wide_xs) : make_uint4(0, 0, 0, 0);
            };
            int i = blockIdx.x >> 1;
            if (i < tiles) load(tile_at(i), 0);
            for (; i < tiles && ok; i += pairs) {
                const Tile t = tile_at(i);
                for (int k2 = 0; k2 < steps && ok; k2 += 2) {
                    const uint4 now[3] = {next[0], next[1], next[2]};
                    if (k2 + 2 < steps) load(t, k2 + 2);
                    else if (i + pairs < tiles) load(tile_at(i + pairs), 0);
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if (k2 + j >= steps) break;
                        if (!bar_wait(done0 + 8 * r.i, r.phase ^ 1u, ctl)) { ok = false; break; }
                        uint32_t* to = reinterpret_cast<uint32_t*>(ring + r.i * stage_bytes + xs_off) + 4 * lane + (warp - 4);
#pragma unroll
                        for (int v = 0; v < 3; v++)
                            if (128 * v < t.cols) {
                                to[256 * v] = j ? now[v].z : now[v].x;
                                to[256 * v + 128] = j ? now[v].w : now[v].y;
                            }
                        __syncwarp();
                        if (lane == 0) bar_arrive(x_written0 + 8 * r.i);
                        r.next(stages);
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------ output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp4FitRegsMany));
        const int half = (warp - 8) >> 2, quarter = warp & 3, id = 32 * quarter + lane;   // (warps 8-11, 12-15: quarters 0-3)
        const uint32_t taddr = tmem + ((uint32_t)(32 * quarter) << 16), read0 = map_to_rank0(smem_u32(tile_read));
        float* room = reinterpret_cast<float*>(ring + stages * stage_bytes + half * kFp4FitRoom);
        constexpr int kPitch = 80;   // floats of a row there (the lanes' banks differ)
        uint32_t n = 0;
        for (int i = blockIdx.x >> 1; i < tiles; i += pairs, n++) {
            const Tile t = tile_at(i);
            // (one of the four warps that gives up takes the others along: they meet at barriers from here on)
            if (!all_of(1 + half, 128, bar_wait(smem_u32(tile_done) + 8 * (n & 1), (n >> 1) & 1u, ctl))) break;
            tc_fence_after();
            const uint32_t from = taddr + place(n, t.cols);
            const int m = t.m + kHalf * (int)rank;
            // Every second 32 rows of x are this half's, `mine` of them: all but four, and the last four, whose columns are
            // in registers when the accumulator is handed back.
            const int mine = (t.cols + 32 - 32 * half) >> 6;
#pragma unroll 1
            for (int last = mine > 4 ? 0 : 1; last < 2; last++) {
                const int c0 = last ? max(mine - 4, 0) : 0, count = last ? min(mine, 4) : mine - 4;
                float acc[4][32];
#pragma unroll
                for (int h = 0; h < 4; h++)
                    if (h < count) tmem_ld32_later(from + 64 * (c0 + h) + 32 * half, acc[h]);
                loaded(acc);
                if (last) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive_cluster(read0 + 8 * (n & 1));
                }
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    const int at = 64 * (c0 + h) + 32 * half, have = t.n - at;   // (the same for all four warps)
                    if (h >= count || have <= 0) break;
                    const float (&v)[32] = acc[h];
                    const long long row = t.pos + at;
                    if (MODE == kFp4Plain) {
                        store_outputs(p, row, 0, 1, have, m + id, v);
                    } else {
                        // gate's lanes get both sums of the even rows, up's of the odd ones
                        const bool up = lane & 16;
                        float y[16];
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            const float g0 = __shfl_xor_sync(0xffffffffu, up ? v[c] : v[c + 1], 16);
                            const float g1 = __shfl_xor_sync(0xffffffffu, up ? v[c + 2] : v[c + 3], 16);
                            const float2 own = up ? make_float2(v[c + 1], v[c + 3]) : make_float2(v[c], v[c + 2]);
                            const float2 other = make_float2(g0, g1);
                            const float2 f = gated2(up ? other : own, up ? own : other, p.limit);
                            y[c / 2] = f.x;
                            y[c / 2 + 1] = f.y;
                        }
                        const int feature = 16 * quarter + (lane & 15);
                        if (MODE == kFp4Gated) {
                            store_outputs(p, row, up, 2, have, m + feature, y);
                        } else {
                            named_barrier(1 + half, 128);   // what was in the room is out
                            float* to = room + (up ? kPitch : 0) + feature;
#pragma unroll
                            for (int c = 0; c < 16; c++) to[2 * c * kPitch] = y[c];
                            named_barrier(1 + half, 128);   // 32 rows are there
                            const int left = p.M - m;
#pragma unroll
                            for (int j = 0; j < 2; j++) {   // eight features a lane, four lanes a block
                                const int r = (id + 128 * j) >> 3, o = (id & 7) * 8;
                                const float4* f = reinterpret_cast<const float4*>(room + r * kPitch + o);
                                const float4 a = f[0], b = f[1];
                                float e[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                                uint32_t top = 0;
#pragma unroll
                                for (int k = 0; k < 8; k++) {
                                    if (o + k >= left) e[k] = 0.f;
                                    top = max(top, magnitude(e[k]));
                                }
                                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                                const uint32_t scale = fp4_scale(top), q = e2m1x8(e, scale);
                                if (r < have && o / kFp4Block * kFp4Block < left) {
                                    *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + (row + r) * p.ld_out + (m + o) / 2) = q;
                                    if ((id & 3) == 0) p.out_scales[(row + r) * p.ld_os + (m + o) / kFp4Block] = (uint8_t)scale;
                                }
                            }
                        }
                    }
                }
            }
        }
    }
    // ---------------- teardown: every role of both CTAs is done (or gave up); free tensor memory
    tc_fence_before();
    __syncthreads();
    // (as in fp8_pair_kernel: the first CTA learns how many stages the other has issued, which learns whether to stay)
    if (threadIdx.x == 0) store_peer(const_cast<uint32_t*>(&from_peer), rank ^ 1, rank == 0 ? (uint32_t)given_up : issued);
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    if (rank == 0 ? given_up != 0 : from_peer != 0) {
        if (rank == 0 && threadIdx.x == 0) {
            Fp4FitBars bars{full, bytes};
            drain_pair(issued, from_peer, stages, bars);
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

// ------------------------------------------------------------ a matrix's scales into units
// scales [groups][rows][blocks] of 32 columns -> [groups][units][steps][2][512];
// unit i holds rows 128 i ... (f = 0), or of a gated matrix's f features 64 i ...
// those of gate and up in turns of 16.  What does not exist is 0.
__global__ void fp4_scale_units_kernel(const uint8_t* __restrict__ scales, int rows, int blocks, int f, int units, int steps,
                                       uint32_t* __restrict__ out) {
    pdl_start();
    // a word: four scales of one row; blockIdx.z: matrix, y: unit, x: its 128 words along the contracted dimension
    const int word = threadIdx.x, r = 32 * (word & 3) + (word >> 2);
    int row = 128 * blockIdx.y + r;
    if (f) {
        const int feature = 64 * blockIdx.y + 16 * (r >> 5) + (r & 15);
        row = feature < f ? feature + (r & 16 ? f : 0) : rows;
    }
    const size_t g = blockIdx.z;
    uint32_t w = 0;
    if (row < rows) {
        const uint8_t* from = scales + (g * rows + row) * blocks;
        for (int i = 0; i < 4; i++) {
            const int b = 4 * blockIdx.x + i;
            if (b < blocks) w |= (uint32_t)from[b] << (8 * i);
        }
    }
    out[((g * units + blockIdx.y) * 2 * steps + blockIdx.x) * 128 + word] = w;
}
// codes past the last column of a row are 0: cols of them, in whole blocks of 32
__global__ void fp4_clear_tail_kernel(uint8_t* codes, long long rows, int cols, int pitch) {
    pdl_start();
    const long long r = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    uint8_t* p = codes + r * pitch;
    if (cols & 1) p[cols / 2] &= 15;
    for (int i = (cols + 1) / 2; i < pitch; i++) p[i] = 0;
}

}  // namespace qrm
