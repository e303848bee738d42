// E4M3 operands with a scale for each block of 128: what the kernels of qkm_fp8.cu and qkm_fp8_gemm.cu share.
//
// A product is  y[row][m] = sum over column blocks b of  x_scale[row][b] * w_scale[m / 128][b] * (sum over the block's columns of xq * wq):
// the tensor cores add the products of one block, exact to their f32 accumulators, and the block's two scales are applied to that sum in f32.
#pragma once

#include "qkm_kernels.h"
#include "qkm_stream.cuh"

namespace qkm {

// Where the activation rows of a unit come from and its results go.  A "pair" is (token << 4) | slot; of the shared expert and of a dense
// product pair p is row p.
enum Fp8Mode { kFp8Dense = 0, kFp8GateUp = 1, kFp8Down = 2, kFp8SharedGateUp = 3, kFp8SharedDown = 4 };
constexpr uint32_t kFp8NoRow = 0xFFFFFFFFu;

struct Fp8Args {
    const uint8_t* w[2];           // E4M3 rows [experts][M][K]; gate and up, or one matrix
    const float* w_scale[2];       // [experts][ceil(M / 128)][ceil(K / 128)]
    const uint8_t* xq;             // E4M3 rows of K
    const float* x_scale;          // [rows][ceil(K / 128)]
    const uint32_t *offsets, *pairs;
    const qkm_sel* sel;            // routing weights of the down products
    float* out;
    uint32_t M, K, n;              // n: rows (dense), tokens otherwise
    uint32_t n_experts, n_used;    // experts of w and offsets
    uint32_t n_table;              // experts of the whole table, of which these may be a shard
    uint32_t* status;
};

__device__ __forceinline__ uint32_t fp8_blocks(uint32_t v) { return (v + 127u) / 128u; }

// Entry of a list of pairs (of the shared expert and of a dense product: row number) -> row of xq and of the results; kFp8NoRow where it names a
// token or slot that there is none of
struct Fp8Place { uint32_t row; uint64_t out; };
template <int MODE>
__device__ __forceinline__ Fp8Place fp8_place(const Fp8Args& a, uint32_t entry) {
    if (MODE == kFp8Dense) return {entry, entry};
    if (MODE == kFp8SharedGateUp) return {entry, (uint64_t)entry * (a.n_used + 1) + a.n_used};
    if (MODE == kFp8SharedDown) return {entry * (a.n_used + 1) + a.n_used, entry};
    const uint32_t t = entry >> 4, s = entry & 15u;
    if (t >= a.n || s >= a.n_used) return {kFp8NoRow, 0};
    if (MODE == kFp8GateUp) return {t, (uint64_t)t * (a.n_used + 1) + s};
    return {t * (a.n_used + 1) + s, (uint64_t)t * a.n_used + s};
}
// routing weight of an entry that has a place
template <int MODE>
__device__ __forceinline__ float fp8_weight(const Fp8Args& a, uint32_t entry) {
    if (MODE == kFp8SharedDown) return a.sel[entry].w_shared;
    if (MODE == kFp8Down) return a.sel[entry >> 4].w[entry & 15u];
    return 1.f;
}
// expert e's run of the list of pairs, whatever the offsets hold inside the list
__device__ __forceinline__ void fp8_run(const Fp8Args& a, uint32_t e, uint32_t& p0, uint32_t& p1) {
    const uint32_t most = a.n * a.n_used;
    p0 = min(a.offsets[e], most);
    p1 = min(a.offsets[e + 1], most);
    if (p1 < p0) p1 = p0;
}

}  // namespace qkm
