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
    int across;                // weights on the M side: tiles of 256 outputs
    int row_tiles, tile_rows;  // weights on the M side: room for tiles of rows in the grid, most rows of one
    int wide_xs;               // rows of scales start on 16 bytes: 2, on 8: 1
};

// Instruction descriptor of kind::mxf4: f32 accumulators, e2m1 A and B, e8m0
// scales, of which bytes `part` and `part` + 1 of each word are used (0 or 2).
__device__ __forceinline__ constexpr uint32_t umma_idesc_mxf4(int m, int n, int part) {
    return ((uint32_t)part << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) |
           ((uint32_t)part << 29);
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
// Descriptors in two words, of which the high ones are constants: of operands in
// the 128-byte swizzle (as sw128_desc), and of units of scales for tcgen05.cp, 32
// rows of 16 bytes one after the other without a swizzle (8-row groups 128 bytes
// apart).  With that, and with what goes into them in registers of the warp, a
// stage's instructions take the issuing thread 420 cycles in place of 620.
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
// outputs (two blocks of 128; gated: 128 features) x up to tile_rows <= 64 rows
// of x, the MMA's N, rounded up to 16 only.  A cluster of CTAs shares a tile's
// contracted dimension, so that one token through one matrix is read by most
// SMs; each leaves its f32 sums in its shared memory, and then each adds up its
// share of the outputs over all of them, in their order.  No partial sums in
// global memory, so calls need no workspace and may overlap.
//
// Two CTAs fit on an SM, so one's start and end, or the next launch's start, go on
// behind the other's loads; where there is one matrix, its first stages are asked
// for before the launch before has ended.  Together with a search for the tile that
// one matrix does not need, that took one row through 4096 x 7168 (15.6 MB) from
// 12.2 to 7.4 us, the rest of which is latencies: the first loads, the MMAs, two
// cluster barriers and reads of other SMs between them.  256 rows over 32 x 4096 x
// 7168 (499 MB): 81 us, 6.2 TB/s; 16 rows, which 12.7 of the 32 have on average: 37
// us (floor 30).
//
// Warps: 0 loads codes and the weights' scales, 1 issues the MMAs, 2 finds the
// tile and brings the scales of x; all eight write the output.
constexpr int kFp4Threads = 256;
constexpr int kFp4Rows = 64;                 // most rows of x in a tile
constexpr int kFp4MaxStages = 4;
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
        const int tiles = (b - a + p.tile_rows - 1) / p.tile_rows;
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
            r.pos = __shfl_sync(0xffffffffu, a + in * p.tile_rows, from);
            r.n = __shfl_sync(0xffffffffu, min(b - a - in * p.tile_rows, p.tile_rows), from);
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

// GROUPED: more than one matrix
template <int MODE, bool GROUPED>
__global__ void __launch_bounds__(kFp4Threads, 2)
fp4_split_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                 const __grid_constant__ Fp4Params p, int stages) {
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
    const uint32_t stage_bytes = fp4_stage_bytes(p.tile_rows);
    // a stage: codes of x, codes of both blocks, their scales, scales of x
    const uint32_t w_off = p.tile_rows * 128, ws_off = w_off + 2 * kFp4Tile, xs_off = ws_off + 2 * kFp4Scales;
    uint8_t* ring = sm + kFp4Header;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    // The outputs of a tile of rows are neighbours in the grid, so the CTAs of tiles that have rows come first and do not
    // wait for those that find none (16 tokens of a rank with 32 of 256 experts, 6 of which have rows: 37 us in place of 42)
    const int tile = blockIdx.x / ranks, row_tile = tile / p.across, block = tile % p.across;
    constexpr int kBlock = MODE == kFp4Plain ? 128 : 64;   // outputs of a block
    const int m0 = block * 2 * kBlock;
    const int k0 = (int)((long long)p.steps * rank / ranks), k1 = (int)((long long)p.steps * (rank + 1) / ranks);
    // one matrix: the tile's outputs are known, and its first stages are asked for before the kernel before has ended, which
    // does not write them
    Fp4Tile t{0, 0, 0};
    const int early = GROUPED ? 0 : min(stages, k1 - k0);
    // a stage's copies of the weights, by one thread
    auto load_stage = [&](uint32_t slot, int k) {
        uint8_t* st = ring + slot * stage_bytes;
        mbar_arrive_expect_tx(&full[slot], (uint32_t)(2 * kFp4Tile + 2 * kFp4Scales));
#pragma unroll
        for (int b = 0; b < 2; b++) {
            load_weights<MODE != kFp4Plain>(st + w_off + b * kFp4Tile, &w_map, k * 128, m0 + b * kBlock, t.group, &full[slot]);
            const long long unit = (long long)t.group * p.units + min(m0 / kBlock + b, p.units - 1);   // an absent second block is not stored
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
        for (int i = 0; i < early; i++) load_stage(i, k0 + i);
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), kFp4TmemCols);
    pdl_start();   // nothing before this reads or writes global memory, but for the weights
    if (GROUPED && warp == 2) {
        const Fp4Tile mine = fp4_find(p, row_tile, blockIdx.x == 0);
        if (lane == 0) *found = mine;
    }
    if (!GROUPED) {   // its rows (see fp4_find)
        int a = 0, b = p.T;
        if (p.offsets) {
            a = p.offsets[0];
            b = p.offsets[1];
            if (a < 0 || b < a || b > p.T) {
                a = b = 0;
                if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(p.err, (int)ERR_BOUNDS);
            }
        }
        const int in = row_tile * p.tile_rows;
        t.pos = a + in;
        t.n = max(0, min(b - a - in, p.tile_rows));
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (GROUPED) t = *found;
    if (t.n == 0) {   // (for all of the cluster)
        if (threadIdx.x == 0)
            for (int i = 0; i < early; i++) {   // copies land before the CTA exits
                mbar_arrive(&full[i]);
                if (!mbar_wait(&full[i], 0u)) atomicOr(p.err, (int)ERR_TIMEOUT);
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
                if (k >= k0 + early) load_stage(r.i, k);
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
        const uint32_t x_low = sw128_low(ring0), w_low = sw128_low(ring0 + w_off);
        const uint32_t ws_low = scale_low(ring0 + ws_off), xs_low = scale_low(ring0 + xs_off), base = uniform(tmem);
        const uint32_t idesc = umma_idesc_mxf4(128, uniform(t.n + 15) & ~15, 0), odd = umma_idesc_mxf4(0, 0, 2) & ~umma_idesc_mxf4(0, 0, 0);
        for (int k = k0; k < k1; k++) {
            if (!bar_wait_both(full0 + 8 * r.i, r.phase, x_full0 + 8 * r.i, r.phase, ctl)) break;
            tc_fence_after();
            const uint32_t at = r.i * stage_bytes >> 4, wl = w_low + at, xl = x_low + at, wsl = ws_low + at, xsl = xs_low + at;
            const uint32_t ws = base + kFp4TmemScales + kFp4ScaleCols * ((k - k0) & 1), xs = ws + 16, more = k > k0;
            if (elect_one()) {
#pragma unroll
                for (int u = 0; u < 4; u++) scales_to_tmem<1>(ws + 4 * u, wide_desc(wsl + u * (512 >> 4), kScaleHigh));   // block u / 2, half u % 2
#pragma unroll
                for (int u = 0; u < 2; u++) scales_to_tmem<1>(xs + 4 * u, wide_desc(xsl + u * (512 >> 4), kScaleHigh));
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int b = 0; b < 2; b++)
                        umma_mxf4<1>(base + 64 * b, wide_desc(wl + b * (kFp4Tile >> 4) + 2 * j, kSw128High), wide_desc(xl + 2 * j, kSw128High),
                                     j & 1 ? idesc | odd : idesc, ws + 8 * b + 4 * (j >> 1), xs + 4 * (j >> 1), j > 0 ? 1 : more);
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
    if (!mbar_wait(done_bar, 0u)) {   // (of MMAs that were issued: it comes; if not, this CTA writes nothing)
        *abort_flag = 1;
        atomicOr(p.err, (int)ERR_TIMEOUT);
    }
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
    constexpr int per_row = MODE == kFp4Plain ? 8 : 4, kAtOnce = 4;
    const uint32_t mine = smem_u32(sums);
    const int items = *abort_flag ? 0 : t.n * per_row, step = ranks * (kFp4Threads / 32);
    for (int i0 = rank + ranks * warp; i0 < items; i0 += kAtOnce * step) {   // kAtOnce of them, whose loads are on their way together
        const int now = min((items - i0 + step - 1) / step, kAtOnce);
        float y[kAtOnce], up[kAtOnce];
        uint32_t at[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int i = i0 + u * step, j = 32 * (i % per_row) + lane;
            // (gated: 16 of gate, 16 of up, and so on)
            at[u] = mine + 4 * (i / per_row * 256 + (MODE == kFp4Plain ? j : 2 * j - (j & 15)));
            y[u] = up[u] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if (q >= (int)ranks) break;
            float a[kAtOnce], b[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                a[u] = b[u] = 0.f;
                if (u >= now) break;
                a[u] = load_peer(at[u], q);
                if (MODE != kFp4Plain) b[u] = load_peer(at[u] + 64, q);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                y[u] += a[u];
                if (MODE != kFp4Plain) up[u] += b[u];
            }
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int i = i0 + u * step, o = 32 * (i % per_row);
            if (u >= now) break;
            const long long to = t.pos + i / per_row;
            if (MODE == kFp4Plain) {
                store_lane(p, to, m0 + o + lane, y[u]);
            } else {
                const float h = gated2(make_float2(y[u], y[u]), make_float2(up[u], up[u]), p.limit).x;
                if (MODE == kFp4Gated) store_lane(p, to, m0 + o + lane, h);
                else store_lane4(p, to, m0 + o, h);
            }
        }
    }
    cluster_sync_all();   // the others may still read this CTA's sums
}

// ------------------------------------------------------------ rows of x on the MMA's M side
// For groups of many rows, which the tensor cores bound.  A pair of SMs
// (cta_group::2) shares a tile of 256 rows of x times 256 outputs (gated: 128
// features): each CTA loads 128 rows of x and 128 of the weights, 32 KB of codes
// for 256 contracted values, and the MMA reads both halves of the weights.
//
// 4096 rows, 28672 x 4096: 186 us in bursts, 5.2 PFLOP/s, and 217 under sustained
// load: the power cap bounds it.  What took it from 310 us to 176 in bursts: the scales of x handed over without a cluster-scope release
// (a full memory barrier with every stage) and asked for four stages at a time,
// rows out by way of shared memory, descriptors with constant high words.
//
// The MMAs of both CTAs are issued by a thread of the first, which has to know
// that the other's scales of x, written by its own warps, are there.  They go
// first: a CTA's copies of a stage are issued by a thread that has waited for the
// stage's scales, so what completes on the first CTA's barrier, the copies' bytes
// (a release of cluster scope), comes behind them.  An arrive of those warps on
// that barrier would need such a release of its own: 396 us in place of 217 under
// sustained load, 370 with a warp that does nothing else.  The copies wait some
// hundred cycles for it, which a tile by itself shows: 256 rows through 4096 x 7168
// take 16.4 us.
//
// Groups of uneven numbers of rows leave most of their last tile empty.  So up to
// 64 rows behind a group's last whole tile, its tail, go with that tile: each stage
// brings half of them to each CTA, and a second MMA takes them against the weights
// that are there already, with the operands' places changed (weights on the M
// side, the tail's rows, rounded up to 32, on the N side).  8192 rows over 32 x 4096
// x 7168, one draw of groups in bursts: 145 -> 120 us (floor 91; 148 -> 142 over
// three draws).  Tiles of their own in that form gained
// nothing (their weights come from L2 once more), nor did a kernel with all rows on
// the N side, 384 a tile (137 us there, but 217 in place of 176 for one matrix).
//
// Tensor memory holds two accumulators of 256 columns but for the scales' 48
// columns: the second begins 48 before the first ends, and a tile's MMAs wait
// for the epilogue of the one before to have read its accumulator (some 1000
// cycles, in which the ring of stages fills up).
//
// Warps: 2 and 3 bring the scales of x, 0 then loads codes and the weights'
// scales, 1 issues the MMAs (in the pair's first CTA), 4-11 write the output: lane
// quarter (warp & 3), half of the columns (warp >= 8).
constexpr int kFp4PairThreads = 384;
constexpr int kFp4PairStages = 5;
constexpr int kFp4PairTx = 2 * kFp4Tile + 2 * kFp4Scales;            // bytes of a CTA's copies of a stage
constexpr int kFp4PairStage = kFp4PairTx + kFp4Scales;               // and the scales of x
constexpr int kFp4PairSecond = 208, kFp4PairTmemScales = 464;
// With tails: half of the tail's rows, this CTA's weights' scales once more, the
// tail's scales; tensor memory for a second accumulator, and 16 columns of scales a stage
constexpr int kFp4TailRows = 64;
constexpr int kFp4TailTx = kFp4TailRows / 2 * 128 + kFp4Scales;
constexpr int kFp4TailStages = 5;             // where they fit (up to 255 matrices), 4 of them else
constexpr int kFp4TailStage = kFp4PairStage + kFp4TailTx + kFp4Scales;
constexpr int kFp4TailSecond = 176, kFp4TailTmemScales = 432, kFp4TailScaleCols = 40;
// a group's tail, by its rows: few rows behind its last whole tile of 256
__host__ __device__ inline int fp4_tail(int rows) { return rows > 256 && (rows & 255) <= kFp4TailRows ? rows & 255 : 0; }
constexpr int kFp4PairOut = 32 * 144;          // a warp's room for rows on their way out: 32 of 128 bytes, 16 apart
constexpr int kFp4TailOut = 32 * 64;           // with tails: 32 of 64 bytes
constexpr int kFp4TailBlocks = 16 * 144;       // gated into 4 bits, of two warps: 16 of 36 floats
constexpr int kFp4PairTableOff = 1024;
constexpr int kFp4PairRegsFew = 72, kFp4PairRegsMany = 216;
constexpr int kFp4PairRegs = 128 * kFp4PairRegsFew + 256 * kFp4PairRegsMany;
static_assert(kFp4PairRegs <= kFp4PairThreads * 168, "register split");
constexpr int kFp4TailRoom = 8 * kFp4TailOut;
static_assert(kFp4TailRoom >= 4 * kFp4TailBlocks, "room");
__host__ __device__ inline int fp4_pair_stage_off(int groups) { return (kFp4PairTableOff + 12 * (groups + 1) + 1023) / 1024 * 1024; }

// the first CTA's barriers, as drain_pair moves them on; the tiles' stages have different numbers of bytes
struct Fp4PairBars {
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
    __device__ void wait(uint32_t slot, uint32_t parity) { (void)mbar_wait(&full[slot], parity); }   // (an error is raised already)
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

// A warp's 32 rows of 2 N outputs each (a lane holds a row) to out, by way of
// shared memory, so that a store's lanes write neighbouring outputs, PIECE bytes of
// each of several rows at once.  left: how many of a row's exist; rows: how many rows
// do.  The room has 32 rows of a piece, 16 bytes apart or (of 64) their four parts in
// another order for every two rows: eight lanes' parts are in eight places.
template <int PIECE>
__device__ __forceinline__ int part_at(int row, int part) {
    return PIECE == 128 ? 144 * row + 16 * part : 64 * row + 16 * (part ^ ((row >> 1) & 3));
}
template <int PIECE, typename T, int N>
__device__ __forceinline__ void store_rows(T* out, long long ld, int left, int rows, const float2 (&v)[N], uint8_t* room, bool wide) {
    constexpr int C = PIECE / sizeof(T), P = PIECE / 16;   // outputs of a row in one go, parts of 16 bytes
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 2 * N; c += C) {
        if (c >= left) break;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P; i++) {
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
            *reinterpret_cast<uint4*>(room + part_at<PIECE>(lane, i)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        if (wide && c + C <= left) {
            const int r0 = lane / P, part = lane % P;
            uint8_t* o = reinterpret_cast<uint8_t*>(out + r0 * ld + c) + 16 * part;
#pragma unroll
            for (int r = 0; r < 32; r += 32 / P)
                if (r + r0 < rows)
                    *reinterpret_cast<uint4*>(o + r * ld * (long long)sizeof(T)) = *reinterpret_cast<const uint4*>(room + part_at<PIECE>(r + r0, part));
        } else {   // one output a lane
            for (int r = 0; r < min(rows, 32); r++)
#pragma unroll
                for (int k = 0; k < C; k += 32) {
                    const int o = k + lane;
                    if (o < C && c + o < left) out[r * ld + c + o] = *reinterpret_cast<const T*>(room + part_at<PIECE>(r, o * (int)sizeof(T) / 16) + o * (int)sizeof(T) % 16);
                }
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

// Output m of rows first, first + step, ..., of which `have` count from row t on,
// by a lane; a warp's lanes write neighbouring outputs
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
// 16 rows of a tail from row t on, of which `have` exist: the lane's output of
// each, number `id` of the CTA's 128 (gated: a row of the MMA's A, gate's and up's in
// turns of 16), which begin at m.  room: gated into 4 bits, of two warps, whose 32
// features are a block.
template <int MODE>
__device__ __forceinline__ void tail_rows(const Fp4Params& p, long long t, int have, int m, int id, const float (&v)[16], float* room,
                                          int barrier) {
    if constexpr (MODE == kFp4Plain) {
        store_outputs(p, t, 0, 1, have, m + id, v);
    } else {
        const int lane = threadIdx.x & 31;
        // gate's lanes get both sums of the even rows, up's of the odd ones
        const bool up = lane & 16;
        float y[8];
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
            const float g0 = __shfl_xor_sync(0xffffffffu, up ? v[c] : v[c + 1], 16);
            const float g1 = __shfl_xor_sync(0xffffffffu, up ? v[c + 2] : v[c + 3], 16);
            const float2 own = up ? make_float2(v[c + 1], v[c + 3]) : make_float2(v[c], v[c + 2]), other = make_float2(g0, g1);
            const float2 f = gated2(up ? other : own, up ? own : other, p.limit);
            y[c / 2] = f.x;
            y[c / 2 + 1] = f.y;
        }
        const int feature = (id >> 5) * 16 + (lane & 15);   // of the CTA's 64
        if constexpr (MODE == kFp4Gated) {
            store_outputs(p, t, up, 2, have, m + feature, y);
        } else {
            constexpr int kPitch = 36;   // floats of a row in the room
            named_barrier(barrier, 64);  // what was in the room is out
#pragma unroll
            for (int c = 0; c < 8; c++) room[(2 * c + (up ? 1 : 0)) * kPitch + (feature & 31)] = y[c];
            named_barrier(barrier, 64);  // 16 rows of 32 features are there: a thread takes a quarter of one
            const int r = (id & 63) >> 2, o = 8 * (id & 3), first = m + (feature & 32), left = p.M - first;
            const float4* from = reinterpret_cast<const float4*>(room + r * kPitch + o);
            const float4 a = from[0], b = from[1];
            float e[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (o + k >= left) e[k] = 0.f;
                top = max(top, magnitude(e[k]));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const uint32_t scale = fp4_scale(top);
            if (r < have && left > 0) {
                *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + (t + r) * p.ld_out + (first + o) / 2) = e2m1x8(e, scale);
                if (o == 0) p.out_scales[(t + r) * p.ld_os + first / kFp4Block] = (uint8_t)scale;
            }
        }
    }
}

// TAILS: tiles may have a tail
template <int MODE, bool TAILS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFp4PairThreads, 1)
fp4_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap s_map,
                const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap tail_map,
                const __grid_constant__ Fp4Params p, int wide_out, int stages) {
    constexpr int kMost = TAILS ? kFp4TailStages : kFp4PairStages, kStage = TAILS ? kFp4TailStage : kFp4PairStage;
    const int n_stages = TAILS ? stages : kFp4PairStages;
    constexpr int kSecond = TAILS ? kFp4TailSecond : kFp4PairSecond, kTmemScales = TAILS ? kFp4TailTmemScales : kFp4PairTmemScales;
    constexpr int kCols = TAILS ? kFp4TailScaleCols : kFp4ScaleCols;   // of scales in tensor memory, a stage's
    constexpr int kTailX = kFp4PairStage, kTailW = kTailX + kFp4TailRows / 2 * 128, kTailS = kTailW + kFp4Scales;   // in a stage
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm);   // first CTA: both CTAs' copies are there
    uint64_t* x_full = full + kMost;           // both: the stage is free and this CTA's scales of x are in it
    uint64_t* done = x_full + kMost;           // both: the stage's MMAs are done
    uint64_t* tile_done = done + kMost;        // [2] both: a tile's are
    uint64_t* tile_read = tile_done + 2;                // first CTA: both epilogues have read an accumulator
    uint64_t* done_bar = tile_read + 1;
    uint64_t* left_bar = done_bar + 1;                  // both, when the first CTA gave up: its commits are through
    __shared__ volatile int given_up;
    __shared__ volatile uint32_t from_peer, issued;     // issued: stages, once their warp is through
    __shared__ volatile uint32_t bytes[kMost];
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
        for (int i = 0; i < n_stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&x_full[i], 2);
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
    if (warp == 2)
        group_tables(p.offsets, p.groups, p.T, p.err, first_tile, start, rows,
                     [&](int n) { return ((n - (TAILS ? fp4_tail(n) : 0) + 255) >> 8) * ((p.M + kOut - 1) / kOut); }, blockIdx.x == 0);
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
        int tail;          // rows behind the pair's 256 that go with them
    };
    // the tiles of one block of outputs follow each other, so its weights come from HBM once
    auto tile_at = [&](int i) {
        int lo = 0, hi = p.groups;   // the last group with first_tile <= i has rows
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first_tile[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int tail = TAILS ? fp4_tail(rows[lo]) : 0, blocks = (rows[lo] - tail + 255) >> 8, in = i - first_tile[lo];
        const int n = in / blocks, r = in - n * blocks, at = r * 256 + 128 * (int)rank;
        return Tile{lo, n * kOut, start[lo] + at, rows[lo] - at, r + 1 == blocks ? tail : 0};
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4PairRegsFew));
        if (warp == 0) {
            // -------------------------------------------- codes and the weights' scales
            bool ok = true;
            Ring r;
            uint32_t n_issued = 0;
            const uint32_t full0 = map_to_rank0(smem_u32(full)), x_full0 = smem_u32(x_full), ring0 = smem_u32(ring);
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs) {
                const Tile t = tile_at(i);
                // this CTA's half of the weights; both have all scales
                const int m = t.m + kOut / 2 * (int)rank;
                const int s0 = (t.group * p.units + t.m / (kOut / 2)) * steps * 4, s1 = s0 + steps * 4, own = s0 + steps * 4 * (int)rank;
                // half of the tail's rows, in whole 16s
                const int tail_at = t.pos - 128 * (int)rank + 256 + ((t.tail + 31) >> 5 << 4) * (int)rank;
                const uint32_t share = kFp4PairTx + (t.tail ? kFp4TailTx : 0);
                for (int k = 0; k < steps; k++) {
                    if (!bar_wait(x_full0 + 8 * r.i, r.phase, ctl)) { ok = false; break; }
                    if (elect_one()) {
                        const uint32_t st = ring0 + r.i * kStage, bar = full0 + 8 * r.i;
                        bytes[r.i] = share;
                        if (rank == 0) mbar_arrive_expect_tx(&full[r.i], 2 * share);
                        // (no rows for this CTA: from past the end, which is zeros and no traffic)
                        tma_pair_2d(st, &x_map, k * 128, t.rows > 0 ? t.pos : p.T, bar);
                        load_weights_pair<MODE != kFp4Plain>(st + kFp4Tile, &w_map, k * 128, m, t.group, bar);
                        tma_pair_2d(st + 2 * kFp4Tile, &s_map, 0, s0 + 4 * k, bar);
                        tma_pair_2d(st + 2 * kFp4Tile + kFp4Scales, &s_map, 0, s1 + 4 * k, bar);
                        if (TAILS && t.tail) {
                            tma_pair_2d(st + kTailX, &tail_map, k * 128, tail_at, bar);
                            tma_pair_2d(st + kTailW, &s_map, 0, own + 4 * k, bar);
                        }
                    }
                    __syncwarp();
                    r.next(n_stages);
                    n_issued++;
                }
            }
            if (lane == 0) issued = n_issued;
        } else if (warp == 1 && rank == 0) {
            // -------------------------------------------- MMAs (one thread issues for both CTAs)
            bool ok = true;
            Ring r;
            uint32_t n = 0, buffer = 0;   // tiles; of scales
            const uint32_t full0 = smem_u32(full), ring0 = smem_u32(ring);
            const uint32_t x_low = sw128_low(ring0), w_low = sw128_low(ring0 + kFp4Tile);
            const uint32_t ws_low = scale_low(ring0 + 2 * kFp4Tile), xs_low = scale_low(ring0 + kFp4PairTx), base = uniform(tmem);
            constexpr uint32_t idesc[2] = {umma_idesc_mxf4(256, 256, 0), umma_idesc_mxf4(256, 256, 2)};
            for (int i = blockIdx.x >> 1; i < tiles && ok; i += pairs, n++) {
                const uint32_t tail = TAILS ? uniform(tile_at(i).tail) : 0;   // (looked up while the epilogue is at work)
                // the accumulator of the tile before has been read
                if (n > 0 && !bar_wait(smem_u32(tile_read), (n - 1) & 1u, ctl)) break;
                const uint32_t d = base + (n & 1 ? kSecond : 0);
                // the tail's: weights on the M side, its rows on the N side, beside the other accumulator
                const uint32_t tail_d = base + (n & 1 ? 0 : 256), tail_idesc = umma_idesc_mxf4(256, (tail + 31) & ~31u, 0);
                for (int k = 0; k < steps; k++) {
                    if (!bar_wait_cluster(full0 + 8 * r.i, r.phase, ctl)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = r.i * (kStage >> 4), wl = w_low + at, xl = x_low + at, wsl = ws_low + at, xsl = xs_low + at;
                    const uint32_t xs = base + kTmemScales + kCols * buffer, ws = xs + 8, more = k > 0;
                    if (elect_one()) {
#pragma unroll
                        for (int u = 0; u < 2; u++) {   // half of the stage's contracted values
                            scales_to_tmem<2>(xs + 4 * u, wide_desc(xsl + u * (512 >> 4), kScaleHigh));
                            scales_to_tmem<2>(ws + 8 * u, wide_desc(wsl + u * (512 >> 4), kScaleHigh));
                            scales_to_tmem<2>(ws + 8 * u + 4, wide_desc(wsl + (kFp4Scales + u * 512 >> 4), kScaleHigh));
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            umma_mxf4<2>(d, wide_desc(xl + 2 * j, kSw128High), wide_desc(wl + 2 * j, kSw128High), idesc[j & 1], xs + 4 * (j >> 1),
                                         ws + 8 * (j >> 1), j > 0 ? 1 : more);
                        if (TAILS && tail) {
                            const uint32_t tws = xs + 24, txs = tws + 8;
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                scales_to_tmem<2>(tws + 4 * u, wide_desc(wsl + (kTailW - 2 * kFp4Tile + u * 512 >> 4), kScaleHigh));
                                scales_to_tmem<2>(txs + 4 * u, wide_desc(wsl + (kTailS - 2 * kFp4Tile + u * 512 >> 4), kScaleHigh));
                            }
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                umma_mxf4<2>(tail_d, wide_desc(wl + 2 * j, kSw128High), wide_desc(xl + (kTailX >> 4) + 2 * j, kSw128High),
                                             j & 1 ? tail_idesc | (idesc[1] & ~idesc[0]) : tail_idesc, tws + 4 * (j >> 1), txs + 4 * (j >> 1), j > 0 ? 1 : more);
                        }
                        umma_commit_pair(done0 + 8 * r.i);
                        if (k + 1 == steps) umma_commit_pair(smem_u32(tile_done) + 8 * (n & 1));
                    }
                    __syncwarp();
                    r.next(n_stages);
                    buffer ^= 1;
                }
            }
            // every MMA has completed before tensor memory is released
            if (elect_one()) {
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(done_bar)) : "memory");
                if (!mbar_wait(done_bar, 0u)) {
                    *abort_flag = 1;
                    atomicOr(p.err, (int)ERR_TIMEOUT);
                }
            }
            __syncwarp();
        } else if (warp >= 2) {
            // -------------------------------------------- scales of x: rows 64 (warp - 2) + lane and + 32 of the CTA's
            // Four stages' at a time.  The next four's are asked for behind the last of these: a fence waits for loads that
            // are on their way, and with these ahead of it cost up to a quarter of the time.
            bool ok = true;
            Ring r;
            const int first = 64 * (warp - 2) + lane;
            const uint32_t x_full0 = smem_u32(x_full);
            uint4 four[2][2];   // [row][half]
            uint4 of_tail[2];   // of its row 32 (warp - 2) + lane
            bool tail = false;
            auto load = [&](const Tile& t, int k) {
                const uint8_t* row = p.x_scales + (long long)(t.pos + first) * p.ld_xs;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const bool in = first + 32 * c < t.rows;
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        four[c][h] = in ? sixteen_scales(row + 32 * c * p.ld_xs, 8 * k + 16 * h, p.blocks, p.wide_xs) : make_uint4(0, 0, 0, 0);
                }
                if (!TAILS) return;
                tail = t.tail != 0;
                if (tail) {
                    const int r = 32 * (warp - 2) + lane;
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        of_tail[h] = r < t.tail ? sixteen_scales(p.x_scales + (long long)(t.pos - 128 * (int)rank + 256 + r) * p.ld_xs, 8 * k + 16 * h, p.blocks, p.wide_xs)
                                                : make_uint4(0, 0, 0, 0);
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
                        uint2* to = reinterpret_cast<uint2*>(ring + r.i * kStage + kFp4PairTx) + 2 * lane + (warp - 2);
                        to[0] = j & 1 ? make_uint2(a.z, b.z) : make_uint2(a.x, b.x);
                        to[64] = j & 1 ? make_uint2(a.w, b.w) : make_uint2(a.y, b.y);
                        if (TAILS && tail) {
                            uint32_t* more = reinterpret_cast<uint32_t*>(ring + r.i * kStage + kTailS) + 4 * lane + (warp - 2);
                            const uint4 c = of_tail[j >> 1];
                            more[0] = j & 1 ? c.z : c.x;
                            more[128] = j & 1 ? c.w : c.y;
                        }
                        fence_async();
                        __syncwarp();
                        if (lane == 0) bar_arrive(x_full0 + 8 * r.i);
                        r.next(n_stages);
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
        uint8_t* room = ring + n_stages * kStage + (warp - 4) * (TAILS ? kFp4TailOut : kFp4PairOut);
        const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t read0 = map_to_rank0(smem_u32(tile_read));
        constexpr int kPiece = TAILS ? 64 : 128;
        const int two = 1 + ((warp - 4) >> 1);
        uint32_t n = 0;
        for (int i = blockIdx.x >> 1; i < tiles; i += pairs, n++) {
            const Tile t = tile_at(i);
            bool there = bar_wait(smem_u32(tile_done) + 8 * (n & 1), (n >> 1) & 1u, ctl);
            // (two warps share a tail's blocks of features: as one of them gives up, both do, since they meet at barriers)
            if (TAILS && MODE == kFp4GatedRows) there = all_of(two, 64, there);
            if (!there) break;
            tc_fence_after();
            const uint32_t from = taddr + (n & 1 ? kSecond : 0);
            // a tail's lanes are outputs, its columns rows of x, every second 16 of them for this half
#pragma unroll 1
            for (int c = 16 * half; TAILS && c < t.tail; c += 32) {
                float v[16];
                tmem_ld16_now(taddr + (n & 1 ? 0 : 256) + c, v);
                tail_rows<MODE>(p, (long long)t.pos - 128 * (int)rank + 256 + c, t.tail - c, t.m + kOut / 2 * (int)rank,
                                32 * (warp & 3) + lane, v, reinterpret_cast<float*>(ring + n_stages * kStage + ((warp - 4) >> 1) * kFp4TailBlocks), two);
            }
            __syncwarp();
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
                    if (p.type == 0) store_rows<kPiece>(reinterpret_cast<float*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, acc, room, wide_out);
                    else if (p.type == 1) store_rows<kPiece>(reinterpret_cast<__half*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, acc, room, wide_out);
                    else store_rows<kPiece>(reinterpret_cast<__nv_bfloat16*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, acc, room, wide_out);
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
                        store_rows<kPiece>(reinterpret_cast<float*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, h, room, wide_out);
                    } else if (p.type == 1) {
                        store_rows<kPiece>(reinterpret_cast<__half*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, h, room, wide_out);
                    } else {
                        store_rows<kPiece>(reinterpret_cast<__nv_bfloat16*>(p.out) + o, p.ld_out, p.M - m, t.rows - r0, h, room, wide_out);
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
            Fp4PairBars bars{full, bytes};
            drain_pair(issued, from_peer, n_stages, bars);
        }
        if (warp == 1) {
            if (rank == 0 && elect_one()) umma_commit_pair(smem_u32(left_bar));
            __syncwarp();
            if (lane == 0) (void)mbar_wait(left_bar, 0u);
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
