// Which kernel an FP8 product takes (qkm_fp8_gemm.cu).  Host arithmetic only.
#pragma once

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

}  // namespace qkm
