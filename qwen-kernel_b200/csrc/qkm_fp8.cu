// Products with E4M3 weights, a scale for each block of 128 x 128: the rows' quantiser, and the products of few rows.
#include "qkm_common.cuh"
#include "qkm_fp8.cuh"

namespace qkm {

// ---- quantiser: f32 rows -> E4M3 with a power of two for each 128 columns -------------------------------------------------------
// The scale is the smallest power of two that keeps the block's largest finite magnitude at or below 448 = 1.75 * 2^8, E4M3's largest:
// dividing by it is exact, so an element is rounded once, by at most 2^-4 of itself (2^-10 of the scale below 2^-6 of it).
// A warp takes a block of 128 columns, a lane four of them; of many blocks, four at a time, so that 2 KB a warp are under way (4096 x 4096: 12.5 us, 6.7 TB/s; one at a time 45).
namespace {

constexpr int kQuantThreads = 256, kQuantWarps = kQuantThreads / 32;

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// BLOCKS consecutive blocks a warp; the matrix is one run of blocks where K is a multiple of 128 (WHOLE)
template <int BLOCKS, bool WHOLE>
__global__ void __launch_bounds__(kQuantThreads)
fp8_quantize_kernel(const float* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scale, uint64_t n_blocks, uint32_t K, uint32_t KB) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t b0 = ((uint64_t)blockIdx.x * kQuantWarps + (threadIdx.x >> 5)) * BLOCKS;
    pdl_trigger();
    pdl_wait();
    float4 v[BLOCKS];
    uint64_t at[BLOCKS];
    bool in[BLOCKS];
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
        const uint64_t b = b0 + i;
        if (WHOLE) {
            at[i] = b * 128u + lane * 4u;
            in[i] = b < n_blocks;
        } else {
            const uint64_t row = b / KB;
            const uint32_t col = (uint32_t)(b - row * KB) * 128u + lane * 4u;
            at[i] = row * K + col;
            in[i] = b < n_blocks && col < K;
        }
        v[i] = in[i] ? __ldcs(reinterpret_cast<const float4*>(x + at[i])) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
        float* e = &v[i].x;
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t m = __float_as_uint(e[j]) & 0x7FFFFFFFu;
            if (m < 0x7F800000u) most = max(most, m);
            else e[j] = __uint_as_float(0x7FC00000u);          // E4M3 has no infinity: what is not finite becomes NaN
        }
        most = __reduce_max_sync(0xFFFFFFFFu, most);
        // 1.75 * 2^E <= 448 * 2^(E - 8): the exponent moves up one where the mantissa is above 1.75
        const uint32_t up = (most + 0x1FFFFFu) >> 23;
        const uint32_t eb = most == 0 ? 127u : up > 9u ? up - 8u : 1u;
        const float inv = __uint_as_float((254u - eb) << 23);
        if (in[i]) *reinterpret_cast<uint32_t*>(q + at[i]) = e4m3x4(e[0] * inv, e[1] * inv, e[2] * inv, e[3] * inv);
        if (lane == 0 && b0 + i < n_blocks) scale[b0 + i] = __uint_as_float(eb << 23);
    }
}

}  // namespace

cudaError_t launch_fp8_quantize(const Launch& L, const float* x, uint32_t n, uint32_t K, void* q, float* scale) {
    if (n == 0) return cudaSuccess;
    const uint32_t KB = (K + 127) / 128;
    const uint64_t blocks = (uint64_t)n * KB;
    auto go = [&](auto kernel, uint32_t per_warp) {
        const uint64_t grid = (blocks + (uint64_t)kQuantWarps * per_warp - 1) / ((uint64_t)kQuantWarps * per_warp);
        if (grid > 0x7FFFFFFFu) return cudaErrorInvalidValue;
        return launch_kernel(Launch{L.stream, nullptr, true}, kernel, dim3((uint32_t)grid), dim3(kQuantThreads), 0, x, (uint8_t*)q, scale, blocks, K, KB);
    };
    // few blocks: as many warps as there are
    cudaError_t e;
    if (K % 128 == 0) e = blocks <= 8192 ? go(fp8_quantize_kernel<1, true>, 1) : go(fp8_quantize_kernel<4, true>, 4);
    else e = blocks <= 8192 ? go(fp8_quantize_kernel<1, false>, 1) : go(fp8_quantize_kernel<4, false>, 4);
    if (e == cudaErrorInvalidValue) return e;
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

// ---- products of few rows --------------------------------------------------------------------------------------------------------
// Warp-level MMAs (m16n8k32) on operands that come straight from global memory: a tile of 16 weight rows x 128 columns is four 16-byte loads a lane,
// and a lane's 16 consecutive bytes serve as its part of two MMAs - the order in which a sum's columns meet is free as long as both operands
// take the same one.  The eight warps of a block share a tile's column blocks; their sums meet in shared memory, in a fixed order.  Bound by latency (1 x 4096 x 2048 4.8 us of a
// graph of them, 16 rows 5.1), large matrices by memory (1 x 151,936 x 2048 60 us, the group kernel's ring 55).
namespace {

constexpr int kRowsThreads = 256, kRowsWarps = kRowsThreads / 32;

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ld16(const uint8_t* p, bool there) { return there ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0); }

template <int MODE> constexpr int rows_mats() { return MODE == kFp8SharedGateUp ? 2 : 1; }

// U: column blocks that a warp loads ahead of their MMAs.  16 weight rows from m0 times rows [p0, p0 + 8 NT); NT: groups of eight rows
template <int MODE, int NT, int U>
__device__ __forceinline__ void rows_tile(const Fp8Args& a, uint32_t m0, uint32_t p0, float* s_red) {
    constexpr int MATS = rows_mats<MODE>();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t KB = fp8_blocks(a.K), p1 = a.n;
    const uint8_t* xrow[NT];
    const float* xsc[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t p = p0 + 8 * j + g;
        xrow[j] = p < p1 ? a.xq + (uint64_t)fp8_place<MODE>(a, p).row * a.K : nullptr;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t pc = p0 + 8 * j + 2 * t + c;
            xsc[j][c] = pc < p1 ? a.x_scale + (uint64_t)fp8_place<MODE>(a, pc).row * KB : nullptr;
        }
    }
    const uint8_t* wrow[MATS];
    const float* wsc[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
        wrow[m] = a.w[m] + (uint64_t)(m0 + g) * a.K;
        wsc[m] = a.w_scale[m] + (uint64_t)(m0 / 128) * KB;
    }
    const bool has0 = m0 + g < a.M, has1 = m0 + g + 8 < a.M;
    float acc[MATS][NT][4] = {};
    for (uint32_t kb0 = warp; kb0 < KB; kb0 += U * kRowsWarps) {
        uint4 wv[U][MATS][2][2], xv[U][NT][2];
        float ws[U][MATS], x0[U][NT], x1[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t kb = kb0 + u * kRowsWarps, c0 = kb * 128 + t * 16;
            const bool there = kb < KB, in[2] = {there && c0 < a.K, there && c0 + 64 < a.K};
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    wv[u][m][c][0] = ld16(wrow[m] + c0 + 64 * c, has0 && in[c]);
                    wv[u][m][c][1] = ld16(wrow[m] + (uint64_t)8 * a.K + c0 + 64 * c, has1 && in[c]);
                }
                ws[u][m] = there ? __ldg(wsc[m] + kb) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int c = 0; c < 2; ++c) xv[u][j][c] = ld16(xrow[j] + c0 + 64 * c, xrow[j] != nullptr && in[c]);
                x0[u][j] = there && xsc[j][0] ? xsc[j][0][kb] : 0.f;
                x1[u][j] = there && xsc[j][1] ? xsc[j][1][kb] : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (kb0 + u * kRowsWarps >= KB) break;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint4 &w0 = wv[u][m][c][0], &w1 = wv[u][m][c][1], &x = xv[u][j][c];
                        mma_e4m3(d, w0.x, w1.x, w0.y, w1.y, x.x, x.y);
                        mma_e4m3(d, w0.z, w1.z, w0.w, w1.w, x.z, x.w);
                    }
                    const float s0 = x0[u][j] * ws[u][m], s1 = x1[u][j] * ws[u][m];
                    acc[m][j][0] += d[0] * s0; acc[m][j][1] += d[1] * s1; acc[m][j][2] += d[2] * s0; acc[m][j][3] += d[3] * s1;
                }
        }
    }
    // s_red[warp][mat][column][16 rows]
    constexpr uint32_t kCols = 8 * NT, kTile = MATS * kCols * 16;
    __syncthreads();   // (the tile before has been read)
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s_red[warp * kTile + (m * kCols + 8 * j + 2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[m][j][i];
    __syncthreads();
    for (uint32_t i = tid; i < kCols * 16; i += kRowsThreads) {
        const uint32_t col = i >> 4, m = m0 + (i & 15u), p = p0 + col;
        if (p >= p1 || m >= a.M) continue;
        float v[MATS] = {};
#pragma unroll
        for (int mat = 0; mat < MATS; ++mat)
            for (int w = 0; w < kRowsWarps; ++w) v[mat] += s_red[w * kTile + mat * kCols * 16 + i];
        a.out[fp8_place<MODE>(a, p).out * a.M + m] = MATS == 2 ? swiglu(v[0], v[MATS - 1]) : MODE == kFp8Dense ? v[0] : fp8_weight<MODE>(a, p) * v[0];
    }
}

template <int MODE, int NT, int U>
__global__ void __launch_bounds__(kRowsThreads)
fp8_rows_kernel(const Fp8Args a) {
    constexpr uint32_t kCols = 8 * NT;
    __shared__ float s_red[kRowsWarps * rows_mats<MODE>() * kCols * 16];
    pdl_trigger();
    // The weights' lines come into the L2 while the kernel before ends (nothing is read yet: what that kernel may still write is seen by the loads).  With weights that are
    // not there, quantiser and product in a graph: 1 x 8192 x 2048 8.3 -> 6.6 us, 1 x 4096 x 2048 5.8 -> 5.4.
    if (blockIdx.y == 0) {
        const uint32_t lane = threadIdx.x & 31u, row = blockIdx.x * 16u + (lane >> 1);
        if (row < a.M)
            for (uint32_t kb = threadIdx.x >> 5; kb < fp8_blocks(a.K); kb += kRowsWarps) {
                const uint32_t c = kb * 128u + (lane & 1u) * 64u;
                if (c < a.K)
#pragma unroll
                    for (int m = 0; m < rows_mats<MODE>(); ++m) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w[m] + (uint64_t)row * a.K + c));
            }
    }
    pdl_wait();
    for (uint32_t p = blockIdx.y * kCols; p < a.n; p += gridDim.y * kCols) rows_tile<MODE, NT, U>(a, blockIdx.x * 16u, p, s_red);
}

template <int MODE>
cudaError_t rows_launch(const Launch& L, const Fp8Args& a) {
    const Launch P{L.stream, nullptr, true};
    auto go = [&](auto kernel, uint32_t cols) {
        const uint32_t chunks = (a.n + cols - 1) / cols;
        return launch_kernel(P, kernel, dim3((a.M + 15) / 16, chunks < 65535 ? chunks : 65535), dim3(kRowsThreads), 0, a);
    };
    // As many blocks of columns at once as a warp has (one row, K = 4096, M = 2048: two 6.4 us, four 3.9, 16 rows 7.3 and 5.4; K = 2048, where it has two, four cost
    // occupancy: M = 8192 6.2 against 9.7)
    const bool wide = a.K > 2048;
    cudaError_t e;
    if (rows_mats<MODE>() == 2) e = a.n <= 8 ? go(fp8_rows_kernel<MODE, 1, 1>, 8) : go(fp8_rows_kernel<MODE, 2, 1>, 16);
    else if (a.n <= 8) e = wide ? go(fp8_rows_kernel<MODE, 1, 4>, 8) : go(fp8_rows_kernel<MODE, 1, 2>, 8);
    else e = wide ? go(fp8_rows_kernel<MODE, 2, 4>, 16) : go(fp8_rows_kernel<MODE, 2, 2>, 16);
    L.count();
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp8_rows(const Launch& L, int mode, const Fp8Args& a) {
    switch (mode) {
        case kFp8Dense: return rows_launch<kFp8Dense>(L, a);
        case kFp8SharedGateUp: return rows_launch<kFp8SharedGateUp>(L, a);
        case kFp8SharedDown: return rows_launch<kFp8SharedDown>(L, a);
    }
    return cudaErrorInvalidValue;
}

}  // namespace qkm
