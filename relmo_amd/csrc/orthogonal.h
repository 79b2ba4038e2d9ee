// What the orthogonalised update's kernels and entry point share.
#pragma once

#include <cstdint>

#include "relm_mp.h"

namespace relm_mp {

// One update, turned so that m <= n; mp and np are m and n rounded up to 32.
struct OrthoMatrix {
    const void* in;
    void* out;
    int64_t in_stride;
    int32_t m, n, mp, np;
    int32_t tall;      // the update is [n, m]
    float scale;       // of X's pairs: a power of two
    uint64_t inv_cols;      // 2^40 / columns of the update, rounded up: divides indices below 2^21
    int64_t first_tile[2];  // of the symmetric products' and the update's tiles
    int64_t x, xt[2], a, b, partial;  // bytes into the workspace
};

// Descriptors travel as kernel arguments (at most 4 KB).
constexpr int kOrthoBatch = 28;
constexpr int kNormParts = 256;  // partial sums of squares of a matrix: a wave adds them
// Tiles of 128 x 128 from which on they are taken instead of 64 x 64 ones: of the symmetric
// products, of the update.  Symmetric: 2048 x 2048 (136 tiles) takes 855 us with large ones,
// 1018 with small.  Update: 2048 x 2048 (256 tiles) 836 us with large ones, 941 with small,
// 1500 x 2600 (252) 661 and 732.  The thresholds between measured counts are not tuned.
constexpr int64_t kLargeTiles[2] = {100, 128};

struct OrthoRule {
    float a, b, c, eps;
    float scale_a, scale_b;  // of A's and B's pairs: powers of two
    int32_t steps;
};

}  // namespace relm_mp
