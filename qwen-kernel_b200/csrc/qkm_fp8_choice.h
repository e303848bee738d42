// Which kernel an FP8 product takes (qkm_fp8_gemm.cu).  Host arithmetic only.
#pragma once

#include <math.h>
#include <stdint.h>

#include "qkm_units.h"

namespace qkm {

// Pairs an expert, on average, from which the pairs are the MMAs' lanes and the weight rows the columns, not the other way round.  256 experts of 2048 x 512, us with the pairs as
// columns and as lanes, where there are 32, 36, 40, 48, 56 and 64: gate/up 117 126, 121 121, 128 124, 137 122, 152 124, 163 127; down 73 100, 78 94, 81 100, 90 97, 102 105, 110 105.
constexpr double kFp8LanesGateUp = 37.0, kFp8LanesDown = 58.0;

// The mean over the whole table of n_expert: a shard's list holds only the pairs of its own experts, so theirs is the same.  (Of rows that came to the shard because they chose
// one of its experts it is more, 1.5 times with 32 of 256 experts and 8 a row; that is not known here.)
inline bool fp8_pairs_as_lanes(bool down, uint32_t n, uint32_t n_used, uint32_t n_expert) {
    return mean_pairs(n, n_used, n_expert, n_expert, false) >= (down ? kFp8LanesDown : kFp8LanesGateUp);
}

// Whether the shared expert's n rows go through the kernel of few rows, 16 weight rows x 16 of them a block, or as lanes (128 of them) with 128 to 512 weight rows a block.  Estimates in
// us, fitted to matrices of 1024 x 256 to 5120 x 2560 and 32 to 512 rows: the first does work in proportion to the rows, the second takes the time of one block until there are more of
// them than SMs.  2048 x 512, 64, 200, 320 and 512 rows: gate/up 6.1 9.6 13.9 19.0 against 15.1 15.9 16.0 16.2, down 4.8 11.5 16.9 25.9 against 13.1 15.4 15.5 15.6;
// 4096 x 1536, 32, 64 and 100 rows: gate/up 10.1 16.4 22.8 against 24.7 25.1 25.7, down 6.7 11.8 17.6 against 12.4 13.0 14.2.
inline bool fp8_shared_few_rows(bool down, uint32_t n, uint32_t M, uint32_t K) {
    const double few = 2.5 + 0.44e-6 * M * (K < 768 ? 768 : K) * ((n + 15) / 16);
    const uint32_t blocks = (K + 127) / 128;
    const double lanes = !down ? 6.5 + 0.6 * blocks : K <= 512 ? 14.0 : 8.0 + 0.55 * blocks;
    return few <= lanes;
}

// Of a dense product: the kernel of few rows, the experts' kernel with one matrix, tiles of rows x weight rows (256 rows: pairs of blocks).
enum class Fp8Dense { kRows, kGroup, k128x32, k128x64, k256x128, k128x256, k256x256 };

// The least of these estimates, in us, fitted to measurements from 1 to 4096 rows, 1000 to 151,936 weight rows and K = 1040 to 4096.
// Tiles go over the machine in waves whose length is that of a tile (at K = 2048: 5.0 us for 128 x 32, 5.5 for 128 x 64, 8.5 for 128 x 256; of pairs of blocks 6.2 for
// 256 x 128, 8.5 for 256 x 256), so that few rows or a small matrix want small tiles and large ones those that read least.  Of at most 32 rows the weights are what is
// read: by warps straight from memory where the matrix is small (16 x 4096 x 2048 5.2 us, group tiles 9.8, 128 x 32 8.4), through the group kernel's ring where it is large
// (1 x 151,936 x 2048 55 us against 60 and 65; 16 rows 57 against 111 and 59).  Below 128 columns there is no box for the copies of the tiles: the kernel of few rows.
inline Fp8Dense fp8_dense_kernel(uint32_t n, uint32_t M, uint32_t K, uint32_t n_sms) {
    const double mb = (double)M * K * 1e-6, k = K / 2048.0;
    auto waves = [&](uint32_t rows, uint32_t cols, uint32_t slots) {
        const uint64_t tiles = (uint64_t)((n + rows - 1) / rows) * (((uint64_t)M + cols - 1) / cols);
        return (double)((tiles + slots - 1) / slots) * k;
    };
    if (K < 128) return Fp8Dense::kRows;
    const double rows = (n <= 8 ? 0.19 : 0.3 * ((n + 15) / 16)) * mb - 0.5;
    const double group = n > 32 ? 1e30 : fmax(6.3 * waves(32, 256, n_sms), mb / 5.9), read = mb / 4.9;
    const double wide[5] = {5.0 * waves(128, 32, n_sms), 5.5 * waves(128, 64, n_sms), 6.2 * waves(256, 128, n_sms / 2), 8.5 * waves(128, 256, n_sms), 8.5 * waves(256, 256, n_sms / 2)};
    int best = 0;
    for (int i = 1; i < 5; ++i)
        if (wide[i] <= wide[best]) best = i;
    const double tiles = fmax(wide[best], read);
    if (rows <= group && rows <= tiles) return Fp8Dense::kRows;
    if (group <= tiles) return Fp8Dense::kGroup;
    return (Fp8Dense)((int)Fp8Dense::k128x32 + best);
}

}  // namespace qkm
