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
// products, of the update.  A call's us with large ones and with small, in a loop.  Symmetric:
// 1200 x 1200 (55 tiles) 461 and 284, 1500 x 1500 (78) 596 and 528, 1700 x 1700 (105) 631 and 602, 1800 x
// 1800 (120) 708 and 690, 2048 x 2048 (136) 742 and 897.  Update: 1200 x 1200 (100) 330 and 283, 2048 x
// 1024 (128) 322 and 293, 1450 x 1600 (156) 492 and 511, 1500 x 2600 (252) 627 and 712, 2048 x 2048
// (256) 742 and 851.  (Both thresholds lie some 25 tiles too low.)
constexpr int64_t kLargeTiles[2] = {100, 128};

struct OrthoRule {
    float a, b, c, eps;
    float scale_a, scale_b;  // of A's and B's pairs: powers of two
    int32_t steps;
};

}  // namespace relm_mp
