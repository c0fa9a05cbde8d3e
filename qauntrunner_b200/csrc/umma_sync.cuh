// umma_sync.cuh -- what the block-scaled products (fp8.cuh, fp4.cuh) share: loads
// into pairs of CTAs, reads of tensor memory, bounded waits, rings, the tables
// of the groups that their tiles go by.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "umma_ptx.cuh"

namespace qrm {

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
struct WaitCtl {
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
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const WaitCtl& c) {
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
static __device__ __noinline__ void drain_own(uint64_t* full, uint32_t issued, uint32_t stages) {
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

// ------------------------------------------------------------ pairs of CTAs
__device__ __forceinline__ uint32_t map_to_rank0(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
// That this warp has read an accumulator, and no more: its loads from tensor
// memory are waited for and the tcgen05 fence is before it.  Without a scope an
// arrive releases to threads of its own CTA, so nothing that was written goes
// with this one.  (With cluster scope here a full memory barrier came with every
// block: 1010 us in place of 560 at 4096 x 28672 x 4096, then.)
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// bar_wait for a barrier that copies of both CTAs complete on
__device__ __forceinline__ bool bar_try_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_wait_cluster(uint32_t bar, uint32_t parity, const WaitCtl& c) {
    if (__all_sync(0xffffffffu, bar_try_cluster(bar, parity))) return true;
    if (!bar_wait_slow(bar, parity, c.abort_flag, c.err)) return false;
    return __all_sync(0xffffffffu, bar_try_cluster(bar, parity));   // (this phase is over, and the next one is not)
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
// ------------------------------------------------------------ rows out
// 2 N outputs of one row that starts on 16 bytes, or on 32 (`wide`): a warp
// writes 32 rows at once, so what counts is how few stores a row takes (32 bytes
// a store, in the 8-bit product: 495 us in place of 531 at 4096 x 28672 x 4096 in bf16, 542 in place
// of 621 in f32, 420 in place of 435 for 8192 rows over 32 x 4096 x 7168, each
// under sustained load).  One value at a time took some 20 us
// a tile: where the rows of out do not start on 16 bytes, the other kernel
// runs, whose warps write neighbouring outputs.
template <typename T, int N>
__device__ __forceinline__ void store_row(T* out, int left, const float2 (&acc)[N], bool wide) {
    constexpr int V = 32 / sizeof(T);   // values of one store
#pragma unroll
    for (int c = 0; c < 2 * N / V; c++) {
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

// ------------------------------------------------------------ groups
// The groups' tables in shared memory, by one warp; the caller synchronises.
// Offsets that do not ascend within [0, T] make a group empty and raise an
// error, and so does a start below any offset before it: no row outside x or
// out is ever touched, and none belongs to two groups (whose CTAs would both
// write it, and whose tiles together could be more than a count of them holds).
// tiles_of: a group's tiles (or what they cost) by its rows; none for no rows.
template <typename Tiles>
__device__ inline void group_tables(const int32_t* offsets, int groups, int T, int32_t* err, int32_t* first_tile, int32_t* start,
                                    int32_t* rows, Tiles tiles_of, bool report) {
    const int lane = threadIdx.x & 31;
    int before = 0, top = 0;   // tiles, largest offset so far
    bool bad = false;
    for (int g0 = 0; g0 < groups; g0 += 32) {
        const int g = g0 + lane;
        int a = 0, b = 0;
        if (g < groups) {
            a = offsets ? offsets[g] : 0;
            b = offsets ? offsets[g + 1] : T;
        }
        int most = a;   // of the offsets up to this one
        if (groups > 1) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) most = max(most, __shfl_up_sync(0xffffffffu, most, o));   // (lanes below o get their own)
            most = max(most, top);
            top = __shfl_sync(0xffffffffu, most, 31);
        }
        if (a < most || a < 0 || b < a || b > T) {
            bad |= g < groups;
            a = b = 0;
        }
        const int tiles = tiles_of(b - a);
        int scan = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (g < groups) {
            first_tile[g] = before + scan - tiles;
            start[g] = a;
            rows[g] = b - a;
        }
        before += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (lane == 0) first_tile[groups] = before;
    if (__any_sync(0xffffffffu, bad) && report && lane == 0) atomicOr(err, (int)ERR_BOUNDS);
}

// the same for tiles of tile_rows rows of x, `across` of them along the outputs
__device__ inline void group_tables(const int32_t* offsets, int groups, int T, int32_t* err, int32_t* first_tile, int32_t* start,
                                    int32_t* rows, int tile_rows, int across, bool report) {
    group_tables(offsets, groups, T, err, first_tile, start, rows, [&](int n) { return (n + tile_rows - 1) / tile_rows * across; }, report);
}

}  // namespace qrm
