// Which kernel an FP8 product takes (qkm_fp8_gemm.cu).  Host arithmetic only.
#pragma once

#include <stdint.h>

#include "qkm_units.h"

namespace qkm {

// Pairs an expert, on average, from which the pairs are the MMAs' lanes: gate/up of 2048 tokens (64) 162 us as columns, 135 as lanes, of 1024 113 and 124; down 112, 108 and 73, 96.
constexpr double kFp8ManyPairs = 44.0;

// The mean over the whole table of n_expert: a shard's list holds only the pairs of its own experts, so theirs is the same.  (Of rows that came to the shard because they chose
// one of its experts it is more, 1.5 times with 32 of 256 experts and 8 a row; that is not known here.)
inline bool fp8_pairs_as_lanes(uint32_t n, uint32_t n_used, uint32_t n_expert) { return mean_pairs(n, n_used, n_expert, n_expert, false) >= kFp8ManyPairs; }

}  // namespace qkm
