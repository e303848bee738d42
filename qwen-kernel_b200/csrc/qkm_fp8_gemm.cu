// Products of many rows with E4M3 weights and block scales on the 5th-generation tensor cores (tcgen05, kind::f8f6f4).
//
// A tile of y is 128 rows (256 for a pair of blocks) x BN weight rows.  The sum over one block of 128 columns is four MMAs (K = 32 each) into a set of
// tensor-memory columns of its own; eight warps read the set back, multiply it by the block's two scales and add it to the tile's f32 sums in registers,
// while the MMAs of the next block run into another set.  Activation rows are the lanes (M), weight rows the columns (N): a thread holds one
// row and a run of columns inside one block of 128 weight rows, so the scale is one number a thread and the scaling one FMA an element.
//
// What bounds it (4096 x 8192 x 4096 in tiles of 256 x 256, 122 us = 2.24 PFLOP/s; under the power cap, back to back, 154): the way out of tensor memory.  A block of 128 columns
// is 514 cycles of MMA for a tile, but its 128 KB of sums take 340 cycles to read and 280 of FMAs (two elements each), which do not overlap much, and the hand-over of a set
// either way some 100 each; with a tile's stores 900 in all.  1000 x 4096 x 2048: 12.6 us, of which 3.5 are the launch, 2 the stores.  Sixteen warps to scale and add took 138 us (the one that
// issues MMAs waits behind 20 warps' polls), sets of 128 columns 139, an arrival with cluster scope 261 (a membar each).
#include <cuda.h>

#include "qkm_common.cuh"
#include "qkm_fp8.cuh"
#include "qkm_fp8_choice.h"
#include "qkm_umma.cuh"
#include "qkm_wait.h"

namespace qkm {
namespace {

namespace tg {
constexpr int kThreads = 384;                    // 4 warps that load and issue, 8 that scale and add
constexpr int kAux = 4, kAdders = 8;
constexpr int kRegAux = 40, kRegAdd = 232;       // registers a thread after the split
constexpr int kRegLaunch = 168;
static_assert(kAux * 32 * kRegAux + kAdders * 32 * kRegAdd <= kThreads * kRegLaunch, "the shares must not exceed the launch's registers");
// BN weight rows a tile; CG blocks share a tile of CG * 128 rows
template <int CG, int BN> struct Tile {
    static constexpr uint32_t kRowsW = BN / CG;                       // weight rows that a block loads
    static constexpr uint32_t kStage = 128 * 128 + kRowsW * 128;
    static constexpr uint32_t kStages = 196608u / kStage < 8 ? 196608u / kStage : 8;
    static constexpr uint32_t kSets = BN == 256 ? 2 : 4;              // tensor-memory column sets
    static constexpr uint32_t kPut = kStages * kStage;                // 4 KB a warp: the way of the results to coalesced stores
    static constexpr uint32_t kSmem = kPut + kAdders * 4096 + 1024;   // (+ what aligning the start may take)
    static constexpr int kCols = BN / 2;                              // columns of a thread
    static constexpr int kLoad = kCols < 64 ? kCols : 64;             // and of a load
};
}  // namespace tg

// a box of rows into this block's shared memory; of a pair (CG 2) the barrier may be the other block's
template <int CG>
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, uint32_t x0, uint32_t r0, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x0), "r"(r0), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x0), "r"(r0), "r"(bar) : "memory");
}
// ---- pairs of blocks (cta_group::2): one MMA over both blocks' tiles, issued by the first; both hold half of each operand
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the same shared-memory address in the cluster's first block
__device__ __forceinline__ uint32_t in_first(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
template <int CG> __device__ __forceinline__ void tmem_take(uint32_t smem_dst) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_dst) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        umma::tmem_alloc(smem_dst, 512);
        umma::tmem_relinquish();
    }
}
template <int CG> __device__ __forceinline__ void tmem_give_back(uint32_t taddr) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
    else umma::tmem_dealloc(taddr, 512);
}
// the MMAs issued so far arrive on the barrier at this address of every block of the pair
template <int CG> __device__ __forceinline__ void commit_all(uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
    else
        umma::commit(bar);
}
// instruction descriptor: E4M3 x E4M3 -> f32, both operands K-major
__device__ __forceinline__ uint32_t instr_desc_e4m3(uint32_t m, uint32_t n) { return 1u << 4 | (n >> 3) << 17 | (m >> 4) << 24; }
template <int CG>
__device__ __forceinline__ void mma_e4m3_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
    const uint32_t acc = accumulate ? 1u : 0u;
    if constexpr (CG == 2)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
            : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
          "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]),
          "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
// the registers of a load that has been waited for (keeps their uses behind the wait)
__device__ __forceinline__ void tmem_ld_done(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                   "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]),
                   "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 ::"memory");
}

// A few polls that end at once when the phase does, then such that let the thread sleep (which take 60 cycles more to wake up); false after about half a second.
__device__ __forceinline__ bool wait_phase(uint32_t b, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
        if (mbar_try_wait(b, parity)) return true;
    return mbar_wait_timed(b, parity);
}
// whether the phase is through, without waiting for it
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// 64, 32 or 16 columns of this warp's lanes, waited for
__device__ __forceinline__ void tmem_load(uint32_t t, float (&v)[64]) {
    float (&lo)[32] = reinterpret_cast<float (&)[32]>(v[0]), (&hi)[32] = reinterpret_cast<float (&)[32]>(v[32]);
    tmem_ld32(t, lo);
    tmem_ld32(t + 32, hi);
    tmem_ld_done(lo);
    tmem_ld_done(hi);
}
__device__ __forceinline__ void tmem_load(uint32_t t, float (&v)[32]) {
    tmem_ld32(t, v);
    tmem_ld_done(v);
}
__device__ __forceinline__ void tmem_load(uint32_t t, float (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]),
                   "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
                 : "r"(t));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(v[i]));
}
// acc += v * s, two elements an instruction
template <int N>
__device__ __forceinline__ void add_scaled(float* acc, const float (&v)[N], float s) {
    uint64_t s2;
    asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
#pragma unroll
    for (int i = 0; i < N; i += 2)
        asm("{\n"
            ".reg .b64 v, c;\n"
            "mov.b64 v, {%2, %3};\n"
            "mov.b64 c, {%0, %1};\n"
            "fma.rn.f32x2 c, v, %4, c;\n"
            "mov.b64 {%0, %1}, c;\n"
            "}\n"
            : "+f"(acc[i]), "+f"(acc[i + 1]) : "f"(v[i]), "f"(v[i + 1]), "l"(s2));
}

struct WideArgs {
    const float *w_scale, *x_scale;
    float* y;
    uint32_t M, n, KB, MB;
    uint32_t x_tiles, n_tiles;     // tiles along the rows of x; all of them
    uint32_t vec;                  // 16-byte stores
    uint32_t* status;
};

template <int CG, int BN>
__global__ void __launch_bounds__(tg::kThreads, 1)
fp8_wide_kernel(const WideArgs a, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map) {
    using T = tg::Tile<CG, BN>;
    extern __shared__ uint8_t smem_dyn[];
    __shared__ __align__(8) unsigned long long s_bar[2 * T::kStages + 2 * T::kSets];
    __shared__ uint32_t s_tmem;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0u, unit0 = blockIdx.x / CG, units = gridDim.x / CG;
    const uint32_t base = (smem_addr(smem_dyn) + 1023u) & ~1023u;
    const uint32_t bar_full = smem_addr(s_bar), bar_empty = bar_full + 8 * T::kStages, bar_set = bar_empty + 8 * T::kStages, bar_free = bar_set + 8 * T::kSets;
    if (tid == 0) {
        for (uint32_t i = 0; i < T::kStages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
        for (uint32_t i = 0; i < T::kSets; ++i) { mbar_init(bar_set + 8 * i, 1); mbar_init(bar_free + 8 * i, CG * tg::kAdders); }
        mbar_fence_init();
    }
    if (warp == 2) tmem_take<CG>(smem_addr(&s_tmem));
    umma::fence_before_sync();
    pdl_trigger();
    pdl_wait();
    __syncwarp();
    if (CG == 2) cluster_sync();
    else __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = s_tmem;
    Waits waits;
    auto wait_bar = [&](uint32_t b, uint32_t parity) { waits.wait([&] { return wait_phase(b, parity); }); };

    if (warp >= (uint32_t)tg::kAux) {
        // ---- scale and add: TMEM lanes 32 q .., half h of a set's columns, weight rows of one block of 128
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(tg::kRegAdd));
        const uint32_t q = warp & 3u, h = (warp - tg::kAux) >> 2;
        const uint32_t put = base + T::kPut + (warp - tg::kAux) * 4096u;
        const uint32_t t0 = tmem + ((32 * q) << 16) + h * T::kCols, free0 = CG == 2 ? in_first(bar_free) : bar_free;
        uint32_t set = 0, parity = 0;                                    // the next set, and its barrier's phase
        bool ready = false;                                              // the next set's barrier is through
        for (uint32_t u = unit0; u < a.n_tiles; u += units) {
            const uint32_t xt = u % a.x_tiles, wt = u / a.x_tiles;
            const uint32_t r0 = (xt * CG + rank) * 128u + 32 * q, m0 = wt * BN + h * T::kCols;
            const float* xs = a.x_scale + (size_t)min(r0 + lane, a.n - 1) * a.KB;
            const float* ws = a.w_scale + (size_t)min(m0 / 128u, a.MB - 1) * a.KB;
            constexpr int kParts = T::kCols / T::kLoad;
            float acc[kParts][T::kLoad];
#pragma unroll
            for (int p = 0; p < kParts; ++p)
#pragma unroll
                for (int i = 0; i < T::kLoad; ++i) acc[p][i] = 0.f;
            float x0 = xs[0], w0 = ws[0];                                // (the next block's scales are on their way while this one's are used)
            for (uint32_t kb = 0; kb < a.KB; ++kb) {
                const uint32_t t = t0 + set * BN;
                const float xc = x0, wc = w0;
                if (kb + 1 < a.KB) { x0 = xs[kb + 1]; w0 = ws[kb + 1]; }
                if (!ready) wait_bar(bar_set + 8 * set, parity);
                __syncwarp();                                            // (each lane polls; the loads are the whole warp's)
                umma::fence_after_sync();
                const float s = xc * wc;
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    float v[T::kLoad];
                    tmem_load(t + T::kLoad * p, v);
                    if (p + 1 == kParts) {
                        umma::fence_before_sync();
                        __syncwarp();
                        if (lane == 0) { if (CG == 2) mbar_arrive_cluster(free0 + 8 * set); else mbar_arrive(free0 + 8 * set); }
                        if (++set == T::kSets) { set = 0; parity ^= 1u; }
                        ready = mbar_test(bar_set + 8 * set, parity);    // its answer comes while the additions run
                    }
                    add_scaled(acc[p], v, s);
                }
            }
            if (__any_sync(0xFFFFFFFFu, waits.out)) break;
            // 32 rows x 32 columns at a time (16, where a thread has no more) through shared memory: lanes along the columns for the stores
            constexpr int kPiece = T::kCols < 32 ? T::kCols : 32, kQuads = kPiece / 4, kRows = 32 / kQuads;   // rows of a store
            auto place = [](uint32_t r, uint32_t j) -> uint32_t { return r * (4u * kPiece) + ((j ^ (kQuads == 8 ? r & 7u : (r >> 1) & (kQuads - 1))) << 4); };
#pragma unroll
            for (int c = 0; c < T::kCols / kPiece; ++c) {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < kQuads; ++j) {
                    const float* e = &acc[c * kPiece / T::kLoad][c * kPiece % T::kLoad + 4 * j];
                    asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(put + place(lane, j)), "f"(e[0]), "f"(e[1]), "f"(e[2]), "f"(e[3]) : "memory");
                }
                __syncwarp();
                const uint32_t j = lane % kQuads, m = m0 + kPiece * c + 4 * j;
#pragma unroll
                for (int i = 0; i < 32 / kRows; ++i) {
                    const uint32_t r = kRows * i + lane / kQuads, row = r0 + r;
                    const uint4 o = lds128(put + place(r, j));
                    if (row >= a.n) continue;
                    float* y = a.y + (size_t)row * a.M + m;
                    if (a.vec) {
                        if (m < a.M) *reinterpret_cast<uint4*>(y) = o;
                    } else {
                        const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (m + k < a.M) y[k] = __uint_as_float(w[k]);
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(tg::kRegAux));
        if (warp == 0) {
            // ---- loads
            uint32_t it = 0;
            for (uint32_t u = unit0; u < a.n_tiles; u += units) {
                const uint32_t xt = u % a.x_tiles, wt = u / a.x_tiles;
                for (uint32_t kb = 0; kb < a.KB; ++kb, ++it) {
                    const uint32_t s = it % T::kStages, dst = base + s * T::kStage;
                    if (it >= T::kStages) wait_bar(bar_empty + 8 * s, (it / T::kStages - 1) & 1u);
                    if (__any_sync(0xFFFFFFFFu, waits.out)) break;   // a barrier that still counts bytes takes no second arrival
                    if (lane == 0) {
                        // (the first block's barrier counts the bytes of both; the other's may arrive ahead of their announcement, which
                        // the phase still waits for)
                        const uint32_t full = CG == 2 ? in_first(bar_full + 8 * s) : bar_full + 8 * s;
                        if (rank == 0) mbar_expect_tx(bar_full + 8 * s, CG * T::kStage);
                        tma_tile<CG>(dst, &x_map, kb * 128u, (xt * CG + rank) * 128u, full);
                        tma_tile<CG>(dst + 16384u, &w_map, kb * 128u, wt * BN + rank * T::kRowsW, full);
                    }
                    __syncwarp();
                }
            }
            // the MMAs have read everything, and their arrivals here are in
            for (uint32_t i = it > T::kStages ? it - T::kStages : 0; i < it; ++i) wait_bar(bar_empty + 8 * (i % T::kStages), (i / T::kStages) & 1u);
        } else if (warp == 1 && rank == 0) {
            // ---- MMAs.  The way from a set's return to the next MMA into it is part of the loop that bounds the kernel: as few
            // instructions as may be, counters that are added to instead of remainders.
            const bool leader = umma::elect_one();
            const uint32_t idesc = instr_desc_e4m3(128 * CG, BN);
            const uint32_t steps = unit0 < a.n_tiles ? ((a.n_tiles - unit0 + units - 1) / units) * a.KB : 0u;
            const uint64_t da0 = umma::smem_desc(base);
            uint32_t s = 0, full_parity = 0, set = 0, free_parity = 1;   // (the first pass over the sets waits for the phase before the first)
            uint64_t da = da0;
            for (uint32_t i = 0; i < steps; ++i) {
                wait_bar(bar_full + 8 * s, full_parity);
                wait_bar(bar_free + 8 * set, free_parity);
                umma::fence_after_sync();
                if (leader) {   // (after a wait that ran out the MMAs run on: their operands are in bounds, and the tile is never stored)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_e4m3_ss<CG>(tmem + set * BN, da + 2 * j, da + 1024 + 2 * j, idesc, j != 0);
                    commit_all<CG>(bar_set + 8 * set);
                    commit_all<CG>(bar_empty + 8 * s);
                }
                __syncwarp();
                da += T::kStage / 16;
                if (++s == T::kStages) { s = 0; da = da0; full_parity ^= 1u; }
                if (++set == T::kSets) { set = 0; free_parity ^= 1u; }
            }
        }
    }
    umma::fence_before_sync();
    const int any_timed_out = __syncthreads_or(waits.out ? 1 : 0);
    if (any_timed_out) for (int i = 0; i < 100; ++i) __nanosleep(1000);   // copies and MMAs still under way end long before this does
    __syncwarp();
    if (CG == 2) cluster_sync();   // nothing of this block is read, written or signalled by the other one any more
    if (warp == 2) tmem_give_back<CG>(tmem);
    if (any_timed_out && tid == 0) atomicExch(a.status, (uint32_t)kStatusWaitTimeout);
}

// ---- products grouped by expert (and dense ones of at most 32 rows) -------------------------------------------------------------
// Weight rows are the lanes here (M = 128) and a run of at most 32 pairs the columns, as many as there are: the weights are what has to be read.  A unit is
// the gate and the up rows of one 128-row tile, or two tiles of one matrix, times a run; blocks take consecutive units, so that the runs of an expert
// with more than 32 pairs read a tile from the L2.  Weight tiles come by TMA, the rows of the pairs with 16-byte copies, each row's scale of a
// column block beside them; the eight warps that scale and add take the row scales from shared memory.
//
// What bounds it: memory, once it runs (gate/up of 16 tokens 32 us, 5.6 TB/s behind 5 us of start: the list of units, the first tiles; the 151,936 x 2048 head 55 us = 5.7 TB/s).  Up to some 37
// pairs an expert (gate/up; down 58) it beats the kernels below; 64 columns a unit instead of 32 took 121 us for gate/up of 1024 tokens, against 113, and 89 for down, against 73.
namespace gg {
constexpr int kThreads = 512;                    // warps: 0 weights, 1 MMAs, 2 tensor memory, 4 - 7 rows, 8 - 15 scale and add
constexpr int kRegAux = 40, kRegRows = 72, kRegAdd = 200;
constexpr int kRegLaunch = 128;
static_assert(128 * (kRegAux + kRegRows) + 256 * kRegAdd <= kThreads * kRegLaunch, "the shares must not exceed the launch's registers");
constexpr uint32_t kMaxExperts = 512, kScales = 8, kMeta = 4;   // scale slots; units whose columns' destinations are kept
constexpr uint32_t kNT = 32, kStage = 2 * 16384 + kNT * 128, kStages = 5;   // columns at most; weights and rows of a column block
constexpr uint32_t kSets = 4, kSetCols = 512 / kSets;                      // sets of 2 kNT tensor-memory columns
static_assert(kStages + kSets <= kScales + 2, "a scale slot comes back before its next use is due");
constexpr uint32_t kScale0 = kStages * kStage;                             // [kScales][2][kNT] f32: row scale times either matrix's block scale
constexpr uint32_t kSmem = kScale0 + kScales * kNT * 8 + 1024;
constexpr int kChunk = 8, kChunks = kNT / 2 / kChunk;                      // columns of a load, loads of a warp and matrix
}  // namespace gg

struct GroupUnit { uint32_t e, m0, p0, n; };     // expert, first weight row, first pair, pairs

// The units of a product: experts that have pairs (of a dense product or the shared expert the one matrix), their runs of pairs cut into parts of PART at most,
// every part with all row units of the expert; the parts of a row unit next to one another.
template <int MODE, int PART, uint32_t ROWS>
struct UnitList {
    static constexpr bool kGrouped = MODE == kFp8GateUp || MODE == kFp8Down;
    static constexpr uint32_t kMax = kGrouped ? gg::kMaxExperts : 1u;
    uint32_t unit[kMax + 1], p0[kMax], p1[kMax];     // per live expert: first unit, run
    uint32_t scan[16][2], n_live, n_units;
    uint16_t expert[kMax];

    // by all threads of the block (256 or more; two experts each); __syncthreads behind it
    __device__ __forceinline__ void make(const Fp8Args& a) {
        const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, row_units = (a.M + ROWS - 1) / ROWS;
        uint32_t q0[2] = {}, q1[2] = {}, units[2], c = 0, v = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t e = 2 * tid + i;
            if (kGrouped) { if (e < a.n_experts) fp8_run(a, e, q0[i], q1[i]); }
            else if (e == 0) q1[i] = a.n;
            units[i] = (q1[i] - q0[i] + PART - 1) / PART * row_units;
            c += units[i] ? 1u : 0u;
            v += units[i];
        }
        const uint32_t c_mine = c, v_mine = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t c1 = __shfl_up_sync(0xFFFFFFFFu, c, o), v1 = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= (uint32_t)o) { c += c1; v += v1; }
        }
        if (lane == 31) { scan[warp][0] = c; scan[warp][1] = v; }
        __syncthreads();
        for (uint32_t w = 0; w < warp; ++w) { c += scan[w][0]; v += scan[w][1]; }
        if (tid == blockDim.x - 1) { n_live = c; n_units = v; unit[c] = v; }
        c -= c_mine; v -= v_mine;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (units[i]) {
                expert[c] = (uint16_t)(2 * tid + i); p0[c] = q0[i]; p1[c] = q1[i]; unit[c] = v;
                ++c;
                v += units[i];
            }
    }
    // number of this block's r-th unit, dealt to and fro (the row units of an expert at the same time in neighbouring blocks); n_units or more: none
    __device__ __forceinline__ uint32_t number(uint32_t r) const { return r * gridDim.x + (r & 1u ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }
    // position in the list of the expert that unit u belongs to
    __device__ __forceinline__ uint32_t find(uint32_t u) const {
        uint32_t i = 0;
        if (kGrouped)
#pragma unroll 1
            for (uint32_t step = kMax / 2; step; step >>= 1)
                if (i + step < n_live && unit[i + step] <= u) i += step;
        return i;
    }
    __device__ __forceinline__ GroupUnit at(uint32_t u) const { return of(u, find(u)); }
    // the same for units in ascending order: i is the position of the one before
    __device__ __forceinline__ GroupUnit at(uint32_t u, uint32_t& i) const {
        while (u >= unit[i + 1]) ++i;
        return of(u, i);
    }
    __device__ __forceinline__ GroupUnit of(uint32_t u, uint32_t i) const {
        const uint32_t run = p1[i] - p0[i], parts = (run + PART - 1) / PART, k = u - unit[i], ru = k / parts, part = k - ru * parts;
        GroupUnit g;
        g.e = kGrouped ? expert[i] : 0u;
        g.m0 = ru * ROWS;
        g.p0 = p0[i] + part * PART;
        g.n = min((uint32_t)PART, run - part * PART);
        return g;
    }
};

__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "r"(taddr));
}
// waits for the loads, whose registers are used behind it
template <int N> __device__ __forceinline__ void tmem_done(float (&a)[N], float (&b)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(a[i]), "+f"(b[i]));
}
// acc[0..3] += v[0..3] * x[0..3]
__device__ __forceinline__ void add4(float* a, const float* v, const uint4& x) {
#pragma unroll
    for (int i = 0; i < 4; i += 2)
        asm("{\n"
            ".reg .b64 v, c, x;\n"
            "mov.b64 v, {%2, %3};\n"
            "mov.b64 c, {%0, %1};\n"
            "mov.b64 x, {%4, %5};\n"
            "fma.rn.f32x2 c, v, x, c;\n"
            "mov.b64 {%0, %1}, c;\n"
            "}\n"
            : "+f"(a[i]), "+f"(a[i + 1]) : "f"(v[i]), "f"(v[i + 1]), "r"(i ? x.z : x.x), "r"(i ? x.w : x.y));
}
// silu(g) * u with the fast division (2 ulp; 0 where e^-g passes 2^126, of a result below 2^-119 |u|)
__device__ __forceinline__ float silu_times(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }

template <int MODE>
__global__ void __launch_bounds__(gg::kThreads, 1)
fp8_group_kernel(const Fp8Args a, const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1) {
    constexpr bool kGateUp = MODE == kFp8GateUp, kGrouped = MODE != kFp8Dense;   // (of one matrix only a dense product)
    static_assert(MODE == kFp8Dense || MODE == kFp8GateUp || MODE == kFp8Down, "the shared expert takes other kernels");
    extern __shared__ uint8_t smem_dyn[];
    __shared__ __align__(8) unsigned long long s_bar[2 * gg::kStages + 2 * gg::kSets + 2 * gg::kScales + gg::kMeta];
    __shared__ uint32_t s_tmem;
    __shared__ UnitList<MODE, gg::kNT, kGateUp ? 128u : 256u> s_list;
    __shared__ uint64_t s_out[gg::kMeta][gg::kNT];        // per unit: where a column's results go, ~0: nowhere; its routing weight
    __shared__ float s_wt[gg::kMeta][gg::kNT];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t base = (smem_addr(smem_dyn) + 1023u) & ~1023u;
    const uint32_t bar_full = smem_addr(s_bar), bar_empty = bar_full + 8 * gg::kStages, bar_set = bar_empty + 8 * gg::kStages, bar_free = bar_set + 8 * gg::kSets;
    const uint32_t bar_sfull = bar_free + 8 * gg::kSets, bar_sfree = bar_sfull + 8 * gg::kScales, bar_meta = bar_sfree + 8 * gg::kScales;
    if (tid == 0) {
        for (uint32_t i = 0; i < gg::kStages; ++i) { mbar_init(bar_full + 8 * i, 1 + 4); mbar_init(bar_empty + 8 * i, 1); }
        for (uint32_t i = 0; i < gg::kSets; ++i) { mbar_init(bar_set + 8 * i, 1); mbar_init(bar_free + 8 * i, 8); }
        for (uint32_t i = 0; i < gg::kScales; ++i) { mbar_init(bar_sfull + 8 * i, 4); mbar_init(bar_sfree + 8 * i, 8); }
        for (uint32_t i = 0; i < gg::kMeta; ++i) mbar_init(bar_meta + 8 * i, 8);
        mbar_fence_init();
    }
    if (warp == 2) { umma::tmem_alloc(smem_addr(&s_tmem), 512); umma::tmem_relinquish(); }
    umma::fence_before_sync();
    pdl_trigger();
    pdl_wait();
    const uint32_t KB = fp8_blocks(a.K), MB = fp8_blocks(a.M);
    s_list.make(a);
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = s_tmem, n_units = s_list.n_units;
    const uint32_t u_first = (uint32_t)((uint64_t)n_units * blockIdx.x / gridDim.x), u_end = (uint32_t)((uint64_t)n_units * (blockIdx.x + 1) / gridDim.x);
    uint32_t live_i = s_list.find(u_first);
    auto unit_of = [&](uint32_t u, uint32_t& i) -> GroupUnit { return s_list.at(u, i); };
    Waits waits;
    auto wait_bar = [&](uint32_t b, uint32_t parity) { waits.wait([&] { return wait_phase(b, parity); }); };

    if (warp >= 8) {
        // ---- scale and add
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(gg::kRegAdd));
        const uint32_t q = warp & 3u, h = (warp - 8) >> 2;
        uint32_t blk = 0, set = 0, set_parity = 0, meta = 0;
        for (uint32_t u = u_first; u < u_end; ++u, meta = (meta + 1) % gg::kMeta) {
            const GroupUnit g = unit_of(u, live_i);
            float acc[2][gg::kChunks][gg::kChunk];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < gg::kChunks; ++j)
#pragma unroll
                    for (int i = 0; i < gg::kChunk; ++i) acc[m][j][i] = 0.f;
            for (uint32_t kb = 0; kb < KB; ++kb, ++blk) {
                const uint32_t slot = blk % gg::kScales, sc = base + gg::kScale0 + slot * gg::kNT * 8, t = tmem + ((32 * q) << 16) + set * gg::kSetCols;
                wait_bar(lane == 1 ? bar_sfull + 8 * slot : bar_set + 8 * set, lane == 1 ? (blk / gg::kScales) & 1u : set_parity);   // two barriers in one poll
                __syncwarp();
                umma::fence_after_sync();
#pragma unroll
                for (int j = 0; j < gg::kChunks; ++j) {
                    const uint32_t col = (2 * j + h) * gg::kChunk;
                    if (col >= g.n) continue;
                    float v0[gg::kChunk], v1[gg::kChunk];
                    tmem_ld(t + col, v0);
                    tmem_ld(t + gg::kNT + col, v1);
                    tmem_done(v0, v1);
#pragma unroll
                    for (int i = 0; i < gg::kChunk; i += 4) {
                        add4(&acc[0][j][i], &v0[i], lds128(sc + 4 * (col + i)));
                        add4(&acc[1][j][i], &v1[i], lds128(sc + 4 * (gg::kNT + col + i)));
                    }
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) { mbar_arrive(bar_free + 8 * set); mbar_arrive(bar_sfree + 8 * slot); }
                if (++set == gg::kSets) { set = 0; set_parity ^= 1u; }
            }
            if (!__any_sync(0xFFFFFFFFu, waits.out)) {
                const uint32_t m = g.m0 + 32 * q + lane;
                const bool in0 = m < a.M, in1 = m + 128 < a.M;
#pragma unroll
                for (int j = 0; j < gg::kChunks; ++j)
#pragma unroll
                    for (int i = 0; i < gg::kChunk; ++i) {
                        const uint32_t col = (2 * j + h) * gg::kChunk + i;
                        if (col >= g.n) continue;
                        const uint64_t at = s_out[meta][col];
                        if (at == ~0ull) continue;
                        float* out = a.out + at + m;
                        if (kGateUp) {
                            if (in0) *out = silu_times(acc[0][j][i], acc[1][j][i]);
                        } else {
                            const float wt = MODE == kFp8Dense ? 1.f : s_wt[meta][col];
                            if (in0) *out = MODE == kFp8Dense ? acc[0][j][i] : wt * acc[0][j][i];
                            if (in1) out[128] = MODE == kFp8Dense ? acc[1][j][i] : wt * acc[1][j][i];
                        }
                    }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_meta + 8 * meta);
        }
    } else if (warp >= 4) {
        // ---- rows of the pairs: four rows x 128 columns an instruction; a stage is announced two stages later, so that three are under way.  Beside them,
        // a lane for each column: the scales, multiplied, and where the column's results go.  The list of the next unit's pairs is read a unit ahead.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(gg::kRegRows));
        constexpr int kGroups = gg::kNT / 16;                 // of four rows, this warp's
        const uint32_t w = warp - 4, rr = lane >> 3, ck = lane & 7u, mine = w * 32 + lane;
        uint32_t blk = 0, unit = 0;
        auto announce = [&](uint32_t i) {
            umma::fence_smem_to_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(bar_full + 8 * (i % gg::kStages)); mbar_arrive(bar_sfull + 8 * (i % gg::kScales)); }
        };
        // entry of the list for a column, the last one past the end (nobody looks at those columns)
        auto entry = [&](const GroupUnit& g, uint32_t col) -> uint32_t { const uint32_t p = g.p0 + min(col, g.n - 1); return kGrouped ? a.pairs[p] : p; };
        GroupUnit g{};
        uint32_t pr[kGroups], pr_mine = 0;
        auto entries = [&](uint32_t u) {
            g = unit_of(u, live_i);
#pragma unroll
            for (int i = 0; i < kGroups; ++i) pr[i] = entry(g, 16 * i + 4 * w + rr);
            if (mine < gg::kNT) pr_mine = entry(g, mine);
        };
        if (u_first < u_end) entries(u_first);
        bool out = false;
        for (uint32_t u = u_first; u < u_end && !out; ++u, ++unit) {
            const uint32_t n = g.n, meta = unit % gg::kMeta;
            const uint8_t* src[kGroups];
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const Fp8Place r = fp8_place<MODE>(a, pr[i]);
                src[i] = a.xq + (uint64_t)(r.row == kFp8NoRow ? 0u : r.row) * a.K + ck * 16u;
            }
            const Fp8Place me = fp8_place<MODE>(a, pr_mine);
            const float* xs = a.x_scale + (uint64_t)(me.row == kFp8NoRow ? 0u : me.row) * KB;
            const float* ws0 = a.w_scale[0] + ((uint64_t)g.e * MB + g.m0 / 128u) * KB;
            const float* ws1 = kGateUp ? a.w_scale[1] + ((uint64_t)g.e * MB + g.m0 / 128u) * KB : ws0 + (g.m0 / 128u + 1 < MB ? KB : 0u);
            const float wt = me.row == kFp8NoRow || mine >= gg::kNT ? 0.f : fp8_weight<MODE>(a, pr_mine);
            float x0 = xs[0], wa0 = ws0[0], wb0 = ws1[0], x1 = KB > 1 ? xs[1] : 0.f, wa1 = KB > 1 ? ws0[1] : 0.f, wb1 = KB > 1 ? ws1[1] : 0.f;
            if (unit >= gg::kMeta) wait_bar(bar_meta + 8 * meta, (unit / gg::kMeta - 1) & 1u);
            if (mine < gg::kNT) s_out[meta][mine] = mine >= n || me.row == kFp8NoRow ? ~0ull : me.out * a.M;
            if (u + 1 < u_end) entries(u + 1);
            for (uint32_t kb = 0; kb < KB; ++kb, ++blk) {
                const uint32_t s = blk % gg::kStages, slot = blk % gg::kScales;
                const bool there = kb * 128u + ck * 16u < a.K;
                const float xc = x0, wac = wa0, wbc = wb0;
                x0 = x1; wa0 = wa1; wb0 = wb1;
                if (kb + 2 < KB) { x1 = xs[kb + 2]; wa1 = ws0[kb + 2]; wb1 = ws1[kb + 2]; }
                if (blk >= gg::kStages) wait_bar(bar_empty + 8 * s, (blk / gg::kStages - 1) & 1u);
                if (blk >= gg::kScales) wait_bar(bar_sfree + 8 * slot, (blk / gg::kScales - 1) & 1u);
                if (__any_sync(0xFFFFFFFFu, waits.out)) { out = true; break; }
                const uint32_t dst = base + s * gg::kStage + 32768u;
#pragma unroll
                for (int i = 0; i < kGroups; ++i)
                    if (16u * i < n)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + umma::sw128_chunk(16 * i + 4 * w + rr, ck)), "l"(there ? src[i] + kb * 128u : a.xq),
                                     "r"(there ? 16u : 0u) : "memory");
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (mine < gg::kNT) {
                    const uint32_t sc = base + gg::kScale0 + (slot * 2 * gg::kNT + mine) * 4u;
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(sc), "f"(xc * wac) : "memory");
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(sc + gg::kNT * 4u), "f"(xc * wbc) : "memory");
                    if (kb + 1 == KB) s_wt[meta][mine] = wt;
                }
                if (blk >= 2) {
                    asm volatile("cp.async.wait_group 2;" ::: "memory");
                    announce(blk - 2);
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (!out)
            for (uint32_t i = blk > 2 ? blk - 2 : 0; i < blk; ++i) announce(i);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(gg::kRegAux));
        if (warp == 0) {
            // ---- weights
            uint32_t blk = 0;
            bool out = false;
            for (uint32_t u = u_first; u < u_end && !out; ++u) {
                const GroupUnit g = unit_of(u, live_i);
                const uint32_t r0 = g.e * a.M + g.m0, r1 = kGateUp ? r0 : r0 + 128;
                for (uint32_t kb = 0; kb < KB; ++kb, ++blk) {
                    const uint32_t s = blk % gg::kStages, dst = base + s * gg::kStage, full = bar_full + 8 * s;
                    if (blk >= gg::kStages) wait_bar(bar_empty + 8 * s, (blk / gg::kStages - 1) & 1u);
                    if (__any_sync(0xFFFFFFFFu, waits.out)) { out = true; break; }   // a barrier that still counts bytes takes no second arrival
                    if (lane == 0) {
                        mbar_expect_tx(full, 32768u);
                        tma_tile<1>(dst, &map0, kb * 128u, r0, full);
                        tma_tile<1>(dst + 16384u, kGateUp ? &map1 : &map0, kb * 128u, r1, full);
                    }
                    __syncwarp();
                }
            }
            for (uint32_t i = blk > gg::kStages ? blk - gg::kStages : 0; i < blk && !out; ++i) wait_bar(bar_empty + 8 * (i % gg::kStages), (i / gg::kStages) & 1u);
        } else if (warp == 1) {
            // ---- MMAs
            const bool leader = umma::elect_one();
            const uint64_t da0 = umma::smem_desc(base);
            uint32_t s = 0, full_parity = 0, set = 0, free_parity = 1;
            uint64_t da = da0;
            for (uint32_t u = u_first; u < u_end; ++u) {
                const GroupUnit g = unit_of(u, live_i);
                const uint32_t idesc = instr_desc_e4m3(128, (g.n + 15u) & ~15u);
                for (uint32_t kb = 0; kb < KB; ++kb) {
                    wait_bar(bar_full + 8 * s, full_parity);
                    wait_bar(bar_free + 8 * set, free_parity);
                    umma::fence_after_sync();
                    if (leader) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            mma_e4m3_ss<1>(tmem + set * gg::kSetCols, da + 2 * j, da + 2048 + 2 * j, idesc, j != 0);
                            mma_e4m3_ss<1>(tmem + set * gg::kSetCols + gg::kNT, da + 1024 + 2 * j, da + 2048 + 2 * j, idesc, j != 0);
                        }
                        umma::commit(bar_set + 8 * set);
                        umma::commit(bar_empty + 8 * s);
                    }
                    __syncwarp();
                    da += gg::kStage / 16;
                    if (++s == gg::kStages) { s = 0; da = da0; full_parity ^= 1u; }
                    if (++set == gg::kSets) { set = 0; free_parity ^= 1u; }
                }
            }
        }
    }
    umma::fence_before_sync();
    const int any_timed_out = __syncthreads_or(waits.out ? 1 : 0);
    if (any_timed_out) for (int i = 0; i < 100; ++i) __nanosleep(1000);   // copies and MMAs still under way end long before this does
    __syncwarp();
    if (warp == 2) umma::tmem_dealloc(tmem, 512);
    if (any_timed_out && tid == 0) atomicExch(a.status, (uint32_t)kStatusWaitTimeout);
}

// Where a warp's 32 rows of results go: of the rows 8 i + lane / 4 the row of `out`, kFp8NoRow nowhere.
struct OutRows { uint32_t row[4]; };
__device__ __forceinline__ OutRows out_rows(uint32_t mine) {
    OutRows o;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) o.row[i] = __shfl_sync(0xFFFFFFFFu, mine, 8 * i + ((threadIdx.x & 31u) >> 2));
    return o;
}
// 16 columns of them, by way of 2 KB of shared memory at `put`: four lanes a row for the stores.  All loads ahead of the stores and no branch but their predicates: with
// the address, a shuffle and a branch ahead of each the stores took 350 cycles apiece, 60 us of down at 4096 tokens.
__device__ __forceinline__ void put_columns(const float (&r)[16], uint32_t put, const OutRows& rows, float* out, uint32_t M) {
    const uint32_t lane = threadIdx.x & 31u, j = lane & 3u;
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(put + lane * 64u + ((i ^ ((lane >> 1) & 3u)) << 4)), "f"(r[4 * i]), "f"(r[4 * i + 1]), "f"(r[4 * i + 2]), "f"(r[4 * i + 3])
                     : "memory");
    __syncwarp();
    uint4 o[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t row = 8 * i + (lane >> 2);
        o[i] = lds128(put + row * 64u + ((j ^ ((row >> 1) & 3u)) << 4));
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (rows.row[i] != kFp8NoRow) *reinterpret_cast<uint4*>(out + (uint64_t)rows.row[i] * M + 4 * j) = o[i];
}

// ---- the same with the pairs as lanes, for experts of many pairs ------------------------------------------------------------------------
// A unit is up to 128 pairs (the MMAs' rows, a lane each) times 256 weight rows: the gate and the up rows of a 128-row tile, or two tiles of one matrix.  What a
// thread scales is then one row's, as in the dense kernel: an FMA for two elements and nothing else.  (With the weight rows as lanes the scales of 128 columns came from shared
// memory and the sums went out by single words: gate/up of 4096 tokens 281 us, down 243.)  Now gate/up takes 176 us (196 to 215 back to back, under the power cap): 35 of them go
// when nothing is scaled and added, 18 when no rows are copied, 13 when nothing is stored, 65 without all three - 565 MB from memory, 1.9 GB through the L2, tiles of 128 for 1.6 times the
// pairs that there are.
namespace pg {
constexpr int kThreads = 512;                    // warps: 0 weights, 1 MMAs, 2 - 7 rows (2: tensor memory), 8 - 15 scale and add
constexpr int kRowWarps = 6;
constexpr int kRegAux = 64, kRegAdd = 192;
constexpr int kRegLaunch = 128;
static_assert(256 * kRegAux + 256 * kRegAdd <= kThreads * kRegLaunch, "the shares must not exceed the launch's registers");
constexpr uint32_t kStage = 3 * 16384, kStages = 4, kPut = kStages * kStage, kSmem = kPut + 8 * 2048 + 1024;   // 2 KB a warp on the way to coalesced stores
}  // namespace pg

template <int MODE>
__global__ void __launch_bounds__(pg::kThreads, 1)
fp8_pairs_kernel(const Fp8Args a, const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1) {
    constexpr bool kGateUp = MODE == kFp8GateUp || MODE == kFp8SharedGateUp, kGrouped = MODE == kFp8GateUp || MODE == kFp8Down;
    extern __shared__ uint8_t smem_dyn[];
    __shared__ __align__(8) unsigned long long s_bar[2 * pg::kStages + 4];
    __shared__ uint32_t s_tmem;
    __shared__ UnitList<MODE, 128, kGateUp ? 128u : 256u> s_list;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t base = (smem_addr(smem_dyn) + 1023u) & ~1023u;
    const uint32_t bar_full = smem_addr(s_bar), bar_empty = bar_full + 8 * pg::kStages, bar_set = bar_empty + 8 * pg::kStages, bar_free = bar_set + 16;
    if (tid == 0) {
        for (uint32_t i = 0; i < pg::kStages; ++i) { mbar_init(bar_full + 8 * i, 1 + pg::kRowWarps); mbar_init(bar_empty + 8 * i, 1); }
        for (uint32_t i = 0; i < 2; ++i) { mbar_init(bar_set + 8 * i, 1); mbar_init(bar_free + 8 * i, 8); }
        mbar_fence_init();
    }
    if (warp == 2) { umma::tmem_alloc(smem_addr(&s_tmem), 512); umma::tmem_relinquish(); }
    umma::fence_before_sync();
    pdl_trigger();
    pdl_wait();
    const uint32_t KB = fp8_blocks(a.K), MB = fp8_blocks(a.M);
    s_list.make(a);
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = s_tmem, n_units = s_list.n_units;
    const uint32_t u_end = n_units;
    Waits waits;
    auto wait_bar = [&](uint32_t b, uint32_t parity) { waits.wait([&] { return wait_phase(b, parity); }); };
    // entry of the list of pairs for a row of a unit, the last one past its end (nobody looks at those rows)
    auto entry = [&](const GroupUnit& g, uint32_t row) -> uint32_t { const uint32_t p = g.p0 + min(row, g.n - 1); return kGrouped ? a.pairs[p] : p; };

    if (warp >= 8) {
        // ---- scale and add: TMEM lanes 32 q ..; of gate/up 64 columns of either matrix, else 128 columns of one tile
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(pg::kRegAdd));
        const uint32_t q = warp & 3u, h = (warp - 8) >> 2, row = 32 * q + lane;
        const uint32_t put = base + pg::kPut + (warp - 8) * 2048u;
        const uint32_t c0 = kGateUp ? 64 * h : 128 * h, c1 = kGateUp ? 128 + 64 * h : 128 * h + 64;   // first columns of the two runs of 64
        const uint32_t t0 = tmem + ((32 * q) << 16);
        uint32_t blk = 0, next = 0;                          // next: this row's entry of the list, read a unit ahead
        bool ready = false;
        GroupUnit g{};
        if (s_list.number(0) < u_end) { g = s_list.at(s_list.number(0)); next = entry(g, row); }
        for (uint32_t r = 0, u; (u = s_list.number(r)) < u_end; ++r) {
            const GroupUnit cur = g;
            const uint32_t mine = next;
            const Fp8Place me = fp8_place<MODE>(a, mine);
            const float* xs = a.x_scale + (uint64_t)(me.row == kFp8NoRow ? 0u : me.row) * KB;
            const float* ws0 = a.w_scale[0] + ((uint64_t)cur.e * MB + (kGateUp ? cur.m0 / 128u : min(cur.m0 / 128u + h, MB - 1))) * KB;
            const float* ws1 = kGateUp ? a.w_scale[1] + ((uint64_t)cur.e * MB + cur.m0 / 128u) * KB : ws0;
            float x0 = xs[0], wa0 = ws0[0], wb0 = ws1[0];
            const float wt = me.row == kFp8NoRow ? 0.f : fp8_weight<MODE>(a, mine);
            if (const uint32_t u1 = s_list.number(r + 1); u1 < u_end) { g = s_list.at(u1); next = entry(g, row); }
            float acc[2][64];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i >> 6][i & 63] = 0.f;
            const bool work = 32 * q < cur.n;                // some row of this warp's is there
            for (uint32_t kb = 0; kb < KB; ++kb, ++blk) {
                const uint32_t set = blk & 1u, t = t0 + set * 256u;
                const float xc = x0, wac = wa0, wbc = wb0;
                if (kb + 1 < KB) { x0 = xs[kb + 1]; wa0 = ws0[kb + 1]; wb0 = ws1[kb + 1]; }
                if (!ready) wait_bar(bar_set + 8 * set, (blk >> 1) & 1u);
                __syncwarp();                                // (each lane polls; the loads are the whole warp's)
                umma::fence_after_sync();
                float v[32];
                if (work) {
                    const float s = xc * wac;
#pragma unroll
                    for (int c = 0; c < 3; ++c) {
                        tmem_ld32(t + (c < 2 ? c0 + 32 * c : c1), v);
                        tmem_ld_done(v);
                        add_scaled(&acc[c >> 1][32 * (c & 1)], v, c < 2 ? s : xc * (kGateUp ? wbc : wac));
                    }
                    tmem_ld32(t + c1 + 32, v);
                    tmem_ld_done(v);
                }
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_free + 8 * set);
                ready = mbar_test(bar_set + 8 * (set ^ 1u), ((blk + 1) >> 1) & 1u);
                if (work) add_scaled(&acc[1][32], v, xc * (kGateUp ? wbc : wac));
            }
            if (__any_sync(0xFFFFFFFFu, waits.out)) break;
            if (!work) continue;
            const OutRows to = out_rows(row >= cur.n || me.row == kFp8NoRow ? kFp8NoRow : (uint32_t)me.out);
            const uint32_t m0 = cur.m0 + (kGateUp ? 64 * h : 128 * h);
#pragma unroll
            for (int c = 0; c < (kGateUp ? 4 : 8); ++c) {
                float r[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i] = kGateUp ? silu_times(acc[0][(16 * c + i) & 63], acc[1][(16 * c + i) & 63]) : wt * acc[c >> 2][16 * (c & 3) + i];
                put_columns(r, put, to, a.out + m0 + 16 * c, a.M);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pg::kRegAux));
        if (warp >= 2) {
            // ---- rows: four x 128 columns an instruction.  A warp issues one about every 130 cycles, so six warps share a stage (two: 1.5 times the
            // time of the whole at 128 pairs an expert); a stage is announced two stages later, so that three are under way.
            const uint32_t w = warp - 2, rr = lane >> 3, ck = lane & 7u;
            constexpr int kFours = (32 + pg::kRowWarps - 1) / pg::kRowWarps;   // this warp's fours of rows: w, w + 6, ..
            uint32_t blk = 0;
            auto announce = [&](uint32_t i) {
                umma::fence_smem_to_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_full + 8 * (i % pg::kStages));
            };
            GroupUnit g{};
            uint32_t next = 0;                               // entry of the warp's row number lane, read a unit ahead
            auto entries = [&](uint32_t u) {
                g = s_list.at(u);
                next = entry(g, ((lane >> 2) * pg::kRowWarps + w) * 4 + (lane & 3u));
            };
            if (s_list.number(0) < u_end) entries(s_list.number(0));
            bool out = false;
            for (uint32_t r = 0, u; (u = s_list.number(r)) < u_end && !out; ++r) {
                const uint32_t n = g.n;
                const Fp8Place me = fp8_place<MODE>(a, next);
                const uint8_t* src[kFours];
#pragma unroll
                for (int i = 0; i < kFours; ++i)
                    src[i] = a.xq + (uint64_t)__shfl_sync(0xFFFFFFFFu, me.row == kFp8NoRow ? 0u : me.row, 4 * i + rr) * a.K + ck * 16u;
                if (const uint32_t u1 = s_list.number(r + 1); u1 < u_end) entries(u1);
                for (uint32_t kb = 0; kb < KB; ++kb, ++blk) {
                    const uint32_t s = blk % pg::kStages;
                    const bool there = kb * 128u + ck * 16u < a.K;
                    if (blk >= pg::kStages) wait_bar(bar_empty + 8 * s, (blk / pg::kStages - 1) & 1u);
                    if (__any_sync(0xFFFFFFFFu, waits.out)) { out = true; break; }
                    const uint32_t dst = base + s * pg::kStage;
#pragma unroll
                    for (int i = 0; i < kFours; ++i) {
                        const uint32_t row0 = (i * pg::kRowWarps + w) * 4;
                        if (row0 < n)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + umma::sw128_chunk(row0 + rr, ck)), "l"(there ? src[i] + kb * 128u : a.xq),
                                         "r"(there ? 16u : 0u) : "memory");
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (blk >= 2) {
                        asm volatile("cp.async.wait_group 2;" ::: "memory");
                        announce(blk - 2);
                    }
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (!out)
                for (uint32_t i = blk > 2 ? blk - 2 : 0; i < blk; ++i) announce(i);
        } else if (warp == 0) {
            // ---- weights
            uint32_t blk = 0;
            bool out = false;
            for (uint32_t r = 0, u; (u = s_list.number(r)) < u_end && !out; ++r) {
                const GroupUnit g = s_list.at(u);
                const uint32_t r0 = g.e * a.M + g.m0, r1 = kGateUp ? r0 : r0 + 128;
                for (uint32_t kb = 0; kb < KB; ++kb, ++blk) {
                    const uint32_t s = blk % pg::kStages, dst = base + s * pg::kStage + 16384u, full = bar_full + 8 * s;
                    if (blk >= pg::kStages) wait_bar(bar_empty + 8 * s, (blk / pg::kStages - 1) & 1u);
                    if (__any_sync(0xFFFFFFFFu, waits.out)) { out = true; break; }   // a barrier that still counts bytes takes no second arrival
                    if (lane == 0) {
                        mbar_expect_tx(full, 32768u);
                        tma_tile<1>(dst, &map0, kb * 128u, r0, full);
                        tma_tile<1>(dst + 16384u, kGateUp ? &map1 : &map0, kb * 128u, r1, full);
                    }
                    __syncwarp();
                }
            }
            for (uint32_t i = blk > pg::kStages ? blk - pg::kStages : 0; i < blk && !out; ++i) wait_bar(bar_empty + 8 * (i % pg::kStages), (i / pg::kStages) & 1u);
        } else {
            // ---- MMAs
            const bool leader = umma::elect_one();
            const uint32_t idesc = instr_desc_e4m3(128, 256), rounds = u_end / gridDim.x, steps = (rounds + (s_list.number(rounds) < u_end ? 1u : 0u)) * KB;
            const uint64_t da0 = umma::smem_desc(base);
            uint32_t s = 0, full_parity = 0, set = 0, free_parity = 1;
            uint64_t da = da0;
            for (uint32_t i = 0; i < steps; ++i) {
                wait_bar(bar_full + 8 * s, full_parity);
                wait_bar(bar_free + 8 * set, free_parity);
                umma::fence_after_sync();
                if (leader) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_e4m3_ss<1>(tmem + set * 256u, da + 2 * j, da + 1024 + 2 * j, idesc, j != 0);
                    umma::commit(bar_set + 8 * set);
                    umma::commit(bar_empty + 8 * s);
                }
                __syncwarp();
                da += pg::kStage / 16;
                if (++s == pg::kStages) { s = 0; da = da0; full_parity ^= 1u; }
                set ^= 1u;
                free_parity ^= set ^ 1u;
            }
        }
    }
    umma::fence_before_sync();
    const int any_timed_out = __syncthreads_or(waits.out ? 1 : 0);
    if (any_timed_out) for (int i = 0; i < 100; ++i) __nanosleep(1000);   // copies and MMAs still under way end long before this does
    __syncwarp();
    if (warp == 2) umma::tmem_dealloc(tmem, 512);
    if (any_timed_out && tid == 0) atomicExch(a.status, (uint32_t)kStatusWaitTimeout);
}

// ---- down products of many pairs and short sums ------------------------------------------------------------------------------------------
// Of four column blocks or fewer a unit's results take as long to store as its sums to make.  Here a unit is 128 pairs times 512 weight rows, in tiles of 128: the pairs' rows stay in
// shared memory for all of them, tiles come through a ring, and the two halves of the warps that scale and add take the tiles in turns, so that one stores while the other
// adds.  (down of 4096 tokens, K = 512: the kernel above 174 us, 70 of them stores that nothing overlaps; this one 150, 45 of them stores.)
namespace dg {
constexpr uint32_t kMaxBlocks = 4, kRows = 512, kX = kMaxBlocks * 16384, kStages = 4, kSets = 4;
constexpr uint32_t kW = 2 * kX, kPut = kW + kStages * 16384, kSmem = kPut + 8 * 2048 + 1024;   // x twice, weight tiles, 2 KB a warp on the way to coalesced stores
}  // namespace dg

template <int MODE>
__global__ void __launch_bounds__(pg::kThreads, 1)
fp8_down_kernel(const Fp8Args a, const __grid_constant__ CUtensorMap map) {
    constexpr bool kGrouped = MODE == kFp8Down;
    static_assert(MODE == kFp8Down || MODE == kFp8SharedDown, "one matrix");
    extern __shared__ uint8_t smem_dyn[];
    __shared__ __align__(8) unsigned long long s_bar[4 + 2 * dg::kStages + 3 * dg::kSets];
    __shared__ uint32_t s_tmem;
    __shared__ UnitList<MODE, 128, dg::kRows> s_list;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t base = (smem_addr(smem_dyn) + 1023u) & ~1023u;
    const uint32_t bar_xfull = smem_addr(s_bar), bar_xempty = bar_xfull + 16, bar_full = bar_xempty + 16, bar_empty = bar_full + 8 * dg::kStages;
    const uint32_t bar_set = bar_empty + 8 * dg::kStages, bar_free = bar_set + 16 * dg::kSets;   // sets: [half][set]
    if (tid == 0) {
        for (uint32_t i = 0; i < 2; ++i) { mbar_init(bar_xfull + 8 * i, pg::kRowWarps); mbar_init(bar_xempty + 8 * i, 1); }
        for (uint32_t i = 0; i < dg::kStages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
        for (uint32_t i = 0; i < dg::kSets; ++i) { mbar_init(bar_set + 8 * i, 1); mbar_init(bar_set + 8 * (dg::kSets + i), 1); mbar_init(bar_free + 8 * i, 4); }
        mbar_fence_init();
    }
    if (warp == 2) { umma::tmem_alloc(smem_addr(&s_tmem), 512); umma::tmem_relinquish(); }
    umma::fence_before_sync();
    pdl_trigger();
    pdl_wait();
    const uint32_t KB = fp8_blocks(a.K), MB = fp8_blocks(a.M);
    s_list.make(a);
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = s_tmem, u_end = s_list.n_units;
    Waits waits;
    auto wait_bar = [&](uint32_t b, uint32_t parity) { waits.wait([&] { return wait_phase(b, parity); }); };
    auto entry = [&](const GroupUnit& g, uint32_t row) -> uint32_t { const uint32_t p = g.p0 + min(row, g.n - 1); return kGrouped ? a.pairs[p] : p; };
    auto tiles_of = [&](const GroupUnit& g) -> uint32_t { return (min(dg::kRows, a.M - g.m0) + 127) / 128; };

    if (warp >= 8) {
        // ---- scale and add: TMEM lanes 32 q .., every other tile this half's
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(pg::kRegAdd));
        const uint32_t q = warp & 3u, h = (warp - 8) >> 2, row = 32 * q + lane;
        const uint32_t put = base + dg::kPut + (warp - 8) * 2048u, t0 = tmem + ((32 * q) << 16);
        // A phase of a barrier is told from the next one only, and a set's next use may be the other half's: each half has barriers of its own.
        const uint32_t set0 = bar_set + 8 * dg::kSets * h;
        uint32_t tile = 0, phases = 0, next = 0;             // tiles before; a bit a set: parity of its next phase; this row's entry of the list, read a unit ahead
        if (s_list.number(0) < u_end) next = entry(s_list.at(s_list.number(0)), row);
        for (uint32_t r = 0, u; (u = s_list.number(r)) < u_end; ++r) {
            const GroupUnit g = s_list.at(u);
            const uint32_t tiles = tiles_of(g);
            const Fp8Place me = fp8_place<MODE>(a, next);
            const float wt = me.row == kFp8NoRow ? 0.f : fp8_weight<MODE>(a, next);
            const OutRows to = out_rows(row >= g.n || me.row == kFp8NoRow ? kFp8NoRow : (uint32_t)me.out);
            const bool work = 32 * q < g.n;                  // some row of this warp's is there
            float x[dg::kMaxBlocks];
#pragma unroll
            for (uint32_t kb = 0; kb < dg::kMaxBlocks; ++kb) x[kb] = kb < KB ? a.x_scale[(uint64_t)(me.row == kFp8NoRow ? 0u : me.row) * KB + kb] : 0.f;
            if (const uint32_t u1 = s_list.number(r + 1); u1 < u_end) next = entry(s_list.at(u1), row);
            const float* ws = a.w_scale[0] + ((uint64_t)g.e * MB + g.m0 / 128u) * KB;
            for (uint32_t i = 0; i < tiles; ++i, ++tile) {
                if ((tile & 1u) != h) continue;
                float w[dg::kMaxBlocks];
#pragma unroll
                for (uint32_t kb = 0; kb < dg::kMaxBlocks; ++kb) w[kb] = kb < KB ? ws[i * KB + kb] : 0.f;
                float acc[2][64];
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j >> 6][j & 63] = 0.f;
#pragma unroll
                for (uint32_t kb = 0; kb < dg::kMaxBlocks; ++kb) {
                    if (kb >= KB) break;
                    const uint32_t set = (tile * KB + kb) % dg::kSets, t = t0 + set * 128u;
                    wait_bar(set0 + 8 * set, phases >> set & 1u);
                    __syncwarp();                            // (each lane polls; the loads are the whole warp's)
                    phases ^= 1u << set;
                    umma::fence_after_sync();
                    const float s = x[kb] * w[kb];
                    float v[32];
                    if (work) {
#pragma unroll
                        for (int c = 0; c < 3; ++c) {
                            tmem_ld32(t + 32 * c, v);
                            tmem_ld_done(v);
                            add_scaled(&acc[c >> 1][32 * (c & 1)], v, s);
                        }
                        tmem_ld32(t + 96, v);
                        tmem_ld_done(v);
                    }
                    umma::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_free + 8 * set);
                    if (work) add_scaled(&acc[1][32], v, s);
                }
                if (!work || __any_sync(0xFFFFFFFFu, waits.out)) continue;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    float r[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) r[j] = wt * acc[c >> 2][16 * (c & 3) + j];
                    put_columns(r, put, to, a.out + g.m0 + i * 128u + 16 * c, a.M);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pg::kRegAux));
        if (warp >= 2) {
            // ---- rows: four x 128 columns an instruction, all of a unit's into one of two places
            const uint32_t w = warp - 2, rr = lane >> 3, ck = lane & 7u;
            constexpr int kFours = (32 + pg::kRowWarps - 1) / pg::kRowWarps;   // this warp's fours of rows: w, w + 6, ..
            uint32_t unit = 0, n = 0, next = 0;              // next: entry of the warp's row number lane, read a unit ahead
            auto entries = [&](uint32_t u) {
                const GroupUnit g = s_list.at(u);
                n = g.n;
                next = entry(g, ((lane >> 2) * pg::kRowWarps + w) * 4 + (lane & 3u));
            };
            if (s_list.number(0) < u_end) entries(s_list.number(0));
            for (uint32_t u; (u = s_list.number(unit)) < u_end; ++unit) {
                const uint32_t rows = n, place = unit & 1u, dst = base + place * dg::kX;
                const Fp8Place me = fp8_place<MODE>(a, next);
                const uint8_t* src[kFours];
#pragma unroll
                for (int i = 0; i < kFours; ++i)
                    src[i] = a.xq + (uint64_t)__shfl_sync(0xFFFFFFFFu, me.row == kFp8NoRow ? 0u : me.row, 4 * i + rr) * a.K + ck * 16u;
                if (const uint32_t u1 = s_list.number(unit + 1); u1 < u_end) entries(u1);
                if (unit >= 2) wait_bar(bar_xempty + 8 * place, (unit / 2 - 1) & 1u);
                if (__any_sync(0xFFFFFFFFu, waits.out)) break;
                for (uint32_t kb = 0; kb < KB; ++kb) {
                    const bool there = kb * 128u + ck * 16u < a.K;
#pragma unroll
                    for (int i = 0; i < kFours; ++i) {
                        const uint32_t row0 = (i * pg::kRowWarps + w) * 4;
                        if (row0 < rows)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + kb * 16384u + umma::sw128_chunk(row0 + rr, ck)), "l"(there ? src[i] + kb * 128u : a.xq),
                                         "r"(there ? 16u : 0u) : "memory");
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                umma::fence_smem_to_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_xfull + 8 * place);
            }
        } else if (warp == 0) {
            // ---- weight tiles
            uint32_t blk = 0;
            bool out = false;
            for (uint32_t r = 0, u; (u = s_list.number(r)) < u_end && !out; ++r) {
                const GroupUnit g = s_list.at(u);
                const uint32_t steps = tiles_of(g) * KB;
                uint32_t row = g.e * a.M + g.m0, kb = 0;
                for (uint32_t i = 0; i < steps; ++i, ++blk) {
                    const uint32_t s = blk % dg::kStages, full = bar_full + 8 * s;
                    if (blk >= dg::kStages) wait_bar(bar_empty + 8 * s, (blk / dg::kStages - 1) & 1u);
                    if (__any_sync(0xFFFFFFFFu, waits.out)) { out = true; break; }   // a barrier that still counts bytes takes no second arrival
                    if (lane == 0) {
                        mbar_expect_tx(full, 16384u);
                        tma_tile<1>(base + dg::kW + s * 16384u, &map, kb * 128u, row, full);
                    }
                    __syncwarp();
                    if (++kb == KB) { kb = 0; row += 128; }
                }
            }
            for (uint32_t i = blk > dg::kStages ? blk - dg::kStages : 0; i < blk && !out; ++i) wait_bar(bar_empty + 8 * (i % dg::kStages), (i / dg::kStages) & 1u);
        } else {
            // ---- MMAs
            const bool leader = umma::elect_one();
            const uint32_t idesc = instr_desc_e4m3(128, 128);
            const uint64_t dx0 = umma::smem_desc(base), dw0 = umma::smem_desc(base + dg::kW);
            uint32_t s = 0, full_parity = 0, set = 0, free_parity = 1, half = bar_set, unit = 0;
            for (uint32_t u; (u = s_list.number(unit)) < u_end; ++unit) {
                const uint32_t tiles = tiles_of(s_list.at(u)), place = unit & 1u;
                wait_bar(bar_xfull + 8 * place, (unit / 2) & 1u);
                for (uint32_t i = 0; i < tiles; ++i) {
                    for (uint32_t kb = 0; kb < KB; ++kb) {
                        wait_bar(bar_full + 8 * s, full_parity);
                        wait_bar(bar_free + 8 * set, free_parity);
                        umma::fence_after_sync();
                        const uint64_t da = dx0 + (place * dg::kX + kb * 16384u) / 16, db = dw0 + s * 1024u;
                        if (leader) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) mma_e4m3_ss<1>(tmem + set * 128u, da + 2 * j, db + 2 * j, idesc, j != 0);
                            umma::commit(half + 8 * set);
                            umma::commit(bar_empty + 8 * s);
                        }
                        __syncwarp();
                        if (++s == dg::kStages) { s = 0; full_parity ^= 1u; }
                        if (++set == dg::kSets) { set = 0; free_parity ^= 1u; }
                    }
                    half = 2 * bar_set + 8 * dg::kSets - half;   // the other half's barriers
                }
                if (leader) umma::commit(bar_xempty + 8 * place);
                __syncwarp();
            }
            // (the last arrivals are in)
            for (uint32_t i = unit > 2 ? unit - 2 : 0; i < unit; ++i) wait_bar(bar_xempty + 8 * (i & 1u), (i / 2) & 1u);
        }
    }
    umma::fence_before_sync();
    const int any_timed_out = __syncthreads_or(waits.out ? 1 : 0);
    if (any_timed_out) for (int i = 0; i < 100; ++i) __nanosleep(1000);   // copies and MMAs still under way end long before this does
    __syncwarp();
    if (warp == 2) umma::tmem_dealloc(tmem, 512);
    if (any_timed_out && tid == 0) atomicExch(a.status, (uint32_t)kStatusWaitTimeout);
}

// tensor map over E4M3 rows [rows][K]: boxes of `box` rows x 128 columns, 128-byte swizzle, zeros outside
bool fp8_map(CUtensorMap* map, const void* p, uint64_t rows, uint32_t K, uint32_t box) {
    typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const EncodeFn encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult qres;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres) == cudaSuccess ? (EncodeFn)fn : (EncodeFn) nullptr;
    }();
    if (!encode) return false;
    const cuuint64_t dim[2] = {K, rows}, stride[1] = {K};
    const cuuint32_t boxes[2] = {128, box}, estride[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dim, stride, boxes, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The register split needs what the launch bounds promise: less would leave the warps that ask for more waiting for good.
template <auto Kernel, int Want>
cudaError_t check_registers() {
    static const int regs = [] {
        cudaFuncAttributes f{};
        return cudaFuncGetAttributes(&f, Kernel) == cudaSuccess ? f.numRegs : 0;
    }();
    return regs >= Want ? cudaSuccess : cudaErrorInvalidKernelImage;
}

template <int CG, int BN>
cudaError_t wide_launch(const Launch& L, const Fp8Args& a, uint32_t n_sms) {
    using T = tg::Tile<CG, BN>;
    if (const cudaError_t e = allow_dynamic_smem<fp8_wide_kernel<CG, BN>>((int)T::kSmem)) return e;
    if (const cudaError_t e = check_registers<fp8_wide_kernel<CG, BN>, tg::kRegLaunch>()) return e;
    CUtensorMap xm, wm;
    if (!fp8_map(&xm, a.xq, a.n, a.K, 128) || !fp8_map(&wm, a.w[0], a.M, a.K, T::kRowsW)) return cudaErrorInvalidValue;
    WideArgs w{};
    w.w_scale = a.w_scale[0]; w.x_scale = a.x_scale; w.y = a.out; w.M = a.M; w.n = a.n; w.KB = (a.K + 127) / 128; w.MB = (a.M + 127) / 128;
    w.x_tiles = (a.n + 128 * CG - 1) / (128 * CG);
    const uint64_t tiles = (uint64_t)w.x_tiles * ((a.M + BN - 1) / BN);
    if (tiles > 0x7FFFFFFFu) return cudaErrorInvalidValue;
    w.n_tiles = (uint32_t)tiles;
    w.vec = a.M % 4 == 0 && ((uintptr_t)a.out & 15u) == 0;
    w.status = a.status;
    const uint32_t grid = CG * (uint32_t)(tiles < n_sms / CG ? tiles : n_sms / CG);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(tg::kThreads); cfg.dynamicSmemBytes = T::kSmem; cfg.stream = L.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG; attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = CG == 2 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_wide_kernel<CG, BN>, w, xm, wm);
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <int MODE>
cudaError_t group_launch(const Launch& L, const Fp8Args& a, uint32_t n_sms) {
    constexpr bool kGateUp = MODE == kFp8GateUp, kGrouped = MODE != kFp8Dense;
    if (const cudaError_t e = allow_dynamic_smem<fp8_group_kernel<MODE>>((int)gg::kSmem)) return e;
    if (const cudaError_t e = check_registers<fp8_group_kernel<MODE>, gg::kRegLaunch>()) return e;
    const uint64_t rows = (uint64_t)(kGrouped ? a.n_experts : 1u) * a.M;
    CUtensorMap m0, m1;
    if (rows > 0x7FFFFFFFu || !fp8_map(&m0, a.w[0], rows, a.K, 128) || !fp8_map(&m1, kGateUp ? a.w[1] : a.w[0], rows, a.K, 128)) return cudaErrorInvalidValue;
    // blocks: as many as there can be units
    const uint64_t per = kGateUp ? (a.M + 127) / 128 : (a.M + 255) / 256, pairs = kGrouped ? (uint64_t)a.n * a.n_used : a.n;
    const uint64_t runs = kGrouped ? (pairs < a.n_experts ? pairs : pairs / gg::kNT + a.n_experts) : (pairs + gg::kNT - 1) / gg::kNT, units = per * runs;
    const cudaError_t e = launch_kernel(Launch{L.stream, nullptr, true}, fp8_group_kernel<MODE>, dim3((uint32_t)(units < n_sms ? units : n_sms)), dim3(gg::kThreads), gg::kSmem, a, m0, m1);
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <int MODE>
cudaError_t pairs_launch(const Launch& L, const Fp8Args& a, uint32_t n_sms) {
    constexpr bool kGateUp = MODE == kFp8GateUp || MODE == kFp8SharedGateUp, kGrouped = MODE == kFp8GateUp || MODE == kFp8Down;
    if (const cudaError_t e = allow_dynamic_smem<fp8_pairs_kernel<MODE>>((int)pg::kSmem)) return e;
    if (const cudaError_t e = check_registers<fp8_pairs_kernel<MODE>, pg::kRegLaunch>()) return e;
    const uint64_t rows = (uint64_t)(kGrouped ? a.n_experts : 1u) * a.M;
    CUtensorMap m0, m1;
    if (rows > 0x7FFFFFFFu || !fp8_map(&m0, a.w[0], rows, a.K, 128) || !fp8_map(&m1, kGateUp ? a.w[1] : a.w[0], rows, a.K, 128)) return cudaErrorInvalidValue;
    const uint64_t per = kGateUp ? (a.M + 127) / 128 : (a.M + 255) / 256, pairs = kGrouped ? (uint64_t)a.n * a.n_used : a.n;
    const uint64_t runs = kGrouped ? (pairs < a.n_experts ? pairs : pairs / 128 + a.n_experts) : (pairs + 127) / 128, units = per * runs;
    const cudaError_t e = launch_kernel(Launch{L.stream, nullptr, true}, fp8_pairs_kernel<MODE>, dim3((uint32_t)(units < n_sms ? units : n_sms)), dim3(pg::kThreads), pg::kSmem, a, m0, m1);
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <int MODE>
cudaError_t down_launch(const Launch& L, const Fp8Args& a, uint32_t n_sms) {
    constexpr bool kGrouped = MODE == kFp8Down;
    if (const cudaError_t e = allow_dynamic_smem<fp8_down_kernel<MODE>>((int)dg::kSmem)) return e;
    if (const cudaError_t e = check_registers<fp8_down_kernel<MODE>, pg::kRegLaunch>()) return e;
    const uint64_t rows = (uint64_t)(kGrouped ? a.n_experts : 1u) * a.M;
    CUtensorMap map;
    if (rows > 0x7FFFFFFFu || !fp8_map(&map, a.w[0], rows, a.K, 128)) return cudaErrorInvalidValue;
    const uint64_t per = (a.M + dg::kRows - 1) / dg::kRows, pairs = kGrouped ? (uint64_t)a.n * a.n_used : a.n;
    const uint64_t runs = kGrouped ? (pairs < a.n_experts ? pairs : pairs / 128 + a.n_experts) : (pairs + 127) / 128, units = per * runs;
    const cudaError_t e = launch_kernel(Launch{L.stream, nullptr, true}, fp8_down_kernel<MODE>, dim3((uint32_t)(units < n_sms ? units : n_sms)), dim3(pg::kThreads), dg::kSmem, a, map);
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

// Products of many rows with the rows as lanes
template <int MODE>
cudaError_t many_rows(const Launch& L, const Fp8Args& a, uint32_t n_sms) {
    if constexpr (MODE == kFp8Down || MODE == kFp8SharedDown)
        if (a.K <= 128 * dg::kMaxBlocks) return down_launch<MODE>(L, a, n_sms);
    return pairs_launch<MODE>(L, a, n_sms);
}

template <int MODE>
cudaError_t group_any(const Launch& L, const Fp8Args& a, uint32_t n_sms) {
    return fp8_pairs_as_lanes(MODE == kFp8Down, a.n, a.n_used, a.n_table) ? many_rows<MODE>(L, a, n_sms) : group_launch<MODE>(L, a, n_sms);
}

cudaError_t dense_any(const Launch& L, const Fp8Args& a, uint32_t n_sms) {
    switch (fp8_dense_kernel(a.n, a.M, a.K, n_sms)) {
        case Fp8Dense::kRows: return launch_fp8_rows(L, kFp8Dense, a);
        case Fp8Dense::kGroup: return group_launch<kFp8Dense>(L, a, n_sms);
        case Fp8Dense::k128x32: return wide_launch<1, 32>(L, a, n_sms);
        case Fp8Dense::k128x64: return wide_launch<1, 64>(L, a, n_sms);
        case Fp8Dense::k256x128: return wide_launch<2, 128>(L, a, n_sms);
        case Fp8Dense::k128x256: return wide_launch<1, 256>(L, a, n_sms);
        case Fp8Dense::k256x256: return wide_launch<2, 256>(L, a, n_sms);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_fp8_product(const Launch& L, int mode, const Fp8Args& a, uint32_t n_sms) {
    if (a.n == 0 || a.M == 0) return cudaSuccess;
    switch (mode) {
        case kFp8Dense: return dense_any(L, a, n_sms);
        case kFp8GateUp: return group_any<kFp8GateUp>(L, a, n_sms);
        case kFp8Down: return group_any<kFp8Down>(L, a, n_sms);
        case kFp8SharedGateUp: if (!fp8_shared_few_rows(false, a.n, a.M, a.K)) return many_rows<kFp8SharedGateUp>(L, a, n_sms); break;
        case kFp8SharedDown: if (!fp8_shared_few_rows(true, a.n, a.M, a.K)) return many_rows<kFp8SharedDown>(L, a, n_sms); break;
    }
    return launch_fp8_rows(L, mode, a);
}

}  // namespace qkm
