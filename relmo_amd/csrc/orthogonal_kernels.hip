// Orthogonalised update by Newton-Schulz products: X = G / (|G|_F + eps), then `steps` times
//
//   A = X X^T,   B = b A + c A A,   X <- a X + B X
//
// on the shorter side (a taller G is read and written transposed), which drives the
// singular values towards 1 and keeps the singular vectors.  The iteration is Schulz's (1933);
// the quintic with the facade's default coefficients was published with the optimiser
// Muon (Jordan and others, 2024).
//
// Arithmetic.  The iteration multiplies small singular values by about a per step, and the
// rounding of what it multiplies with them, so 11 or 8 bits are too few for the iterates.
// Every iterate is held as two halves, x = hi + lo with hi = half(x), lo = half(x - hi):
// 22 bits, at scales (powers of two, exact) that keep the halves within their normal
// range.  A product of two such matrices is three matrix-instruction products, hi hi + hi
// lo + lo hi, added in float: about float's own accuracy at a third of the 16-bit rate,
// five times the float instructions' rate (2048 x 2048: error 1.9e-6, in float products
// 2.9e-6).  One half would leave 1.3e-3 to 1.6e-3 by its rounding, a pair 3e-7 (96 x 96 to
// 512 x 512, simulated in double).  The Frobenius norm is added in double.
//
// A and B are symmetric: only their lower tiles are computed, and written twice, and both
// operands of every product are read along their rows (of X there is a transposed copy).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <vector>

#include "device_utils.h"
#include "internal.h"
#include "mfma_tiles.h"
#include "orthogonal.h"
#include "value_types.h"

namespace relm_mp {

namespace {

using Half8 = Frag<f16>;
using Half4 = f16 __attribute__((ext_vector_type(4)));

struct Pair {
    f16 hi, lo;
};
__device__ __forceinline__ Pair halves(float x) {
    const f16 hi = static_cast<f16>(x);
    return {hi, static_cast<f16>(x - static_cast<float>(hi))};
}
__device__ __forceinline__ float whole(f16 hi, f16 lo) { return static_cast<float>(hi) + static_cast<float>(lo); }

// One product of pairs; the small terms first.
__device__ __forceinline__ f32x4 mma_pairs(Half8 ah, Half8 al, Half8 bh, Half8 bl, f32x4 c) {
    c = mma<f16>(al, bh, c);
    c = mma<f16>(ah, bl, c);
    return mma<f16>(ah, bh, c);
}

// The contraction values row 4 g + j and 16 + 4 g + j of lds_frag_t, along a row.
__device__ __forceinline__ Half8 lds_frag_split(const f16* tile, int stride, int row, int col) {
    const int g = lane_id() / 16;
    const Half4 a = *reinterpret_cast<const Half4*>(tile + row * stride + col + 4 * g);
    const Half4 b = *reinterpret_cast<const Half4*>(tile + row * stride + col + 16 + 4 * g);
    return Half8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Entry (i, j) of the result; X is the update turned so that it is at least as wide as tall.
template <typename T>
__device__ __forceinline__ void put_entry(const OrthoMatrix& d, int i, int j, float x) {
    T* out = static_cast<T*>(d.out);
    out[d.tall ? static_cast<int64_t>(j) * d.m + i : static_cast<int64_t>(i) * d.n + j] = round_to<T>(x);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o /= 2) v += __shfl_xor(v, o);
    return v;
}

// ---- one workgroup per matrix, everything in LDS ------------------------------------------

constexpr int kSmallThreads = 512;
constexpr int kSmallWaves = kSmallThreads / kWave;
constexpr int kSmallBlocks = 2;  // 32 x 32 blocks of A that a wave keeps: 10 lower blocks of 128 rows on 8 waves

struct OrthoBatch {
    OrthoMatrix mat[kOrthoBatch];
};

// Latency bound (a product of 96 x 96 is 36 matrix instructions to a wave): few barriers
// (4 a step), operands from LDS in blocks of 32 x 32, a step's A kept in the registers
// of the wave that computed it.  14 matrices of 32 x 32 to 96 x 96 take 45 us: 7 a step for
// the largest, the rest outside the steps.  16 waves ran out of registers and spilled.
template <typename T>
__global__ __launch_bounds__(kSmallThreads) void k_ortho_small(OrthoBatch batch, OrthoRule rule) {
    extern __shared__ __align__(16) f16 pool[];
    __shared__ double partial[kSmallWaves];
    const OrthoMatrix& d = batch.mat[blockIdx.x];
    const int m = d.m, n = d.n, mp = d.mp, np = d.np;
    const int sx = np + 8, sa = mp + 8;  // strides: rows spread over the banks
    f16 *xh = pool, *xl = xh + mp * sx, *ah = xl + mp * sx, *al = ah + mp * sa;
    const int tid = static_cast<int>(threadIdx.x), l = lane_id(), g = l / 16, c16 = l % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);

    // X starts as zeros: its padding stays
    for (int u = tid; u < mp * sx / 4; u += kSmallThreads)  // both planes, 8 halves at a time
        *reinterpret_cast<Half8*>(xh + 8 * u) = Half8(static_cast<f16>(0.0f));
    // the update twice, kBatch values of a thread in flight: its norm, then its entries
    constexpr int kBatch = 8;
    const int cols = d.tall ? m : n, total = m * n;
    const T* in = static_cast<const T*>(d.in);
    auto every = [&](auto&& use) {
        for (int u0 = tid; u0 < total; u0 += kBatch * kSmallThreads) {
            float x[kBatch];
            int row[kBatch], col[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int u = min(u0 + k * kSmallThreads, total - 1);
                row[k] = static_cast<int>((static_cast<uint64_t>(u) * d.inv_cols) >> 40);
                col[k] = u - row[k] * cols;
                x[k] = static_cast<float>(in[row[k] * d.in_stride + col[k]]);
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                if (u0 + k * kSmallThreads < total) use(row[k], col[k], x[k]);
        }
    };
    double sum = 0.0;
    every([&](int, int, float x) { sum = fma(static_cast<double>(x), static_cast<double>(x), sum); });
    sum = wave_sum(sum);
    if (l == 0) partial[wave] = sum;
    __syncthreads();
    sum = partial[0];
#pragma unroll
    for (int v = 1; v < kSmallWaves; ++v) sum += partial[v];
    const float scale = static_cast<float>(static_cast<double>(d.scale) / (sqrt(sum) + static_cast<double>(rule.eps)));
    every([&](int row, int col, float x) {
        const Pair p = halves(x * scale);
        const int at = d.tall ? col * sx + row : row * sx + col;
        xh[at] = p.hi;
        xl[at] = p.lo;
    });
    __syncthreads();

    const int blocks = mp / 32, lower = blocks * (blocks + 1) / 2;
    const float to_a = rule.scale_a / (d.scale * d.scale), from_b = 1.0f / rule.scale_b;
    const float b_of_a = rule.b * rule.scale_b / rule.scale_a, b_of_aa = rule.c * rule.scale_b / (rule.scale_a * rule.scale_a);
    for (int step = 0; step < rule.steps; ++step) {
        // A, the lower blocks; then A A over the same blocks
        f32x4 a[kSmallBlocks][2][2];
        auto product = [&](const f16* ph, const f16* pl, int stride, int depth, int r0, int c0, f32x4 (&acc)[2][2]) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < 2; ++c) acc[r][c] = f32x4(0.0f);
            for (int k = 0; k < depth; k += 32) {
                Half8 fh[2], fl[2], gh[2], gl[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    fh[r] = lds_frag<f16>(ph, stride, r0 + 16 * r + c16, k + 8 * g);
                    fl[r] = lds_frag<f16>(pl, stride, r0 + 16 * r + c16, k + 8 * g);
                    gh[r] = lds_frag<f16>(ph, stride, c0 + 16 * r + c16, k + 8 * g);
                    gl[r] = lds_frag<f16>(pl, stride, c0 + 16 * r + c16, k + 8 * g);
                }
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) acc[r][c] = mma_pairs(fh[r], fl[r], gh[c], gl[c], acc[r][c]);
            }
        };
        auto place = [&](int q, int& r0, int& c0) {  // block q of the lower triangle, row by row
            int r = 0;
            while ((r + 1) * (r + 2) / 2 <= q) ++r;
            r0 = 32 * r;
            c0 = 32 * (q - r * (r + 1) / 2);
        };
        auto put = [&](int r0, int c0, const f32x4 (&v)[2][2]) {  // a block and its mirror image
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    Half4 hi, lo;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const Pair p = halves(v[r][c][i]);
                        const int row = r0 + 16 * r + 4 * g + i, col = c0 + 16 * c + c16;
                        hi[i] = p.hi;
                        lo[i] = p.lo;
                        if (r0 != c0) {
                            ah[row * sa + col] = p.hi;
                            al[row * sa + col] = p.lo;
                        }
                    }
                    const int at = (c0 + 16 * c + c16) * sa + r0 + 16 * r + 4 * g;
                    *reinterpret_cast<Half4*>(ah + at) = hi;
                    *reinterpret_cast<Half4*>(al + at) = lo;
                }
        };
#pragma unroll
        for (int q = 0; q < kSmallBlocks; ++q) {
            const int block = wave + q * kSmallWaves;
            if (block >= lower) break;
            int r0, c0;
            place(block, r0, c0);
            product(xh, xl, sx, np, r0, c0, a[q]);
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < 2; ++c) a[q][r][c] *= to_a;
            put(r0, c0, a[q]);
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kSmallBlocks; ++q) {
            const int block = wave + q * kSmallWaves;
            if (block >= lower) break;
            int r0, c0;
            place(block, r0, c0);
            f32x4 aa[2][2];
            product(ah, al, sa, mp, r0, c0, aa);
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < 2; ++c) a[q][r][c] = a[q][r][c] * b_of_a + aa[r][c] * b_of_aa;
        }
        __syncthreads();  // A has been read: B takes its place
#pragma unroll
        for (int q = 0; q < kSmallBlocks; ++q) {
            const int block = wave + q * kSmallWaves;
            if (block >= lower) break;
            int r0, c0;
            place(block, r0, c0);
            put(r0, c0, a[q]);
        }
        __syncthreads();
        // X <- a X + B X: 16 columns of X depend on themselves and B alone, so each is one
        // wave's, in place: all products, then all entries.  The products are transposed (X's
        // columns down), so that a lane holds four neighbours of a row of X.
        const bool last = step + 1 == rule.steps;
        for (int strip = wave; strip < np / 16; strip += kSmallWaves) {
            f32x4 acc[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) acc[r] = f32x4(0.0f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k >= blocks) break;
                const Half8 fh = lds_frag_t<f16>(xh, sx, 32 * k, 16 * strip), fl = lds_frag_t<f16>(xl, sx, 32 * k, 16 * strip);
#pragma unroll
                for (int r = 0; r < 8; r += 2) {
                    if (r >= 2 * blocks) break;
                    const Half8 bh0 = lds_frag_split(ah, sa, 16 * r + c16, 32 * k), bl0 = lds_frag_split(al, sa, 16 * r + c16, 32 * k);
                    const Half8 bh1 = lds_frag_split(ah, sa, 16 * r + 16 + c16, 32 * k),
                                bl1 = lds_frag_split(al, sa, 16 * r + 16 + c16, 32 * k);
                    acc[r] = mma<f16>(fl, bh0, acc[r]);
                    acc[r + 1] = mma<f16>(fl, bh1, acc[r + 1]);
                    acc[r] = mma<f16>(fh, bl0, acc[r]);
                    acc[r + 1] = mma<f16>(fh, bl1, acc[r + 1]);
                    acc[r] = mma<f16>(fh, bh0, acc[r]);
                    acc[r + 1] = mma<f16>(fh, bh1, acc[r + 1]);
                }
            }
            const int col = 16 * strip + 4 * g;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r >= 2 * blocks) break;
                const int row = 16 * r + c16;
                f16 *to_h = xh + row * sx + col, *to_l = xl + row * sx + col;
                Half4 hi = *reinterpret_cast<const Half4*>(to_h), lo = *reinterpret_cast<const Half4*>(to_l);
                f32x4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[i] = fmaf(rule.a, whole(hi[i], lo[i]), acc[r][i] * from_b);
                    const Pair p = halves(y[i]);
                    hi[i] = p.hi;
                    lo[i] = p.lo;
                }
                if (!last) {
                    *reinterpret_cast<Half4*>(to_h) = hi;
                    *reinterpret_cast<Half4*>(to_l) = lo;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (row < m && col + i < n) put_entry<T>(d, row, col + i, y[i] / d.scale);
                }
            }
        }
        __syncthreads();
    }
}

// ---- larger matrices: tiles of all matrices of a launch -------------------------------------

constexpr int kThreads = 256;

// Partial sums of squares, kNormParts to a matrix.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_ortho_norm(OrthoBatch batch, void* ws) {
    __shared__ double lds[kThreads / kWave];
    const OrthoMatrix& d = batch.mat[blockIdx.y];
    const int64_t rows = d.tall ? d.n : d.m;
    const int cols = d.tall ? d.m : d.n;
    const int wave = static_cast<int>(threadIdx.x) / kWave;
    constexpr int V = kLaneValues<T>;  // the last unit's values past the row are zeros
    double sum = 0.0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + wave; r < rows;
         r += kNormParts * (kThreads / kWave)) {
        const T* in = static_cast<const T*>(d.in) + r * d.in_stride;
#pragma unroll 4
        for (int c = lane_id() * V; c < cols; c += kWave * V) {
            const FloatVec<V> x = load_values<T, V>(in, c, cols);
#pragma unroll
            for (int j = 0; j < V; ++j) sum = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), sum);
        }
    }
    sum = wave_sum(sum);
    if (lane_id() == 0) lds[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int v = 1; v < kThreads / kWave; ++v) sum += lds[v];
        reinterpret_cast<double*>(static_cast<char*>(ws) + d.partial)[blockIdx.x] = sum;
    }
}

// Planes of a matrix in the workspace: hi, then lo, row-major over a padded width (zeros).
struct Planes {
    f16* hi;
    f16* lo;
    int64_t stride;
};
__device__ __forceinline__ Planes planes(void* ws, int64_t at, int64_t rows, int64_t stride) {
    f16* hi = reinterpret_cast<f16*>(static_cast<char*>(ws) + at);
    return {hi, hi + rows * stride, stride};
}
__device__ __forceinline__ Planes planes_x(void* ws, const OrthoMatrix& d) { return planes(ws, d.x, d.m, d.np); }
__device__ __forceinline__ Planes planes_xt(void* ws, const OrthoMatrix& d, int which) {
    return planes(ws, d.xt[which], d.n, d.mp);
}
__device__ __forceinline__ Planes planes_a(void* ws, const OrthoMatrix& d) { return planes(ws, d.a, d.m, d.mp); }
__device__ __forceinline__ Planes planes_b(void* ws, const OrthoMatrix& d) { return planes(ws, d.b, d.m, d.mp); }

// X and its transpose as pairs, 32 x 32 entries to a workgroup; the padding of every plane.
// Bound by memory and the launch: 2048 x 2048 floats 14 us.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_ortho_split(OrthoBatch batch, OrthoRule rule, void* ws) {
    __shared__ float tile[32][33];
    __shared__ double total;
    const OrthoMatrix& d = batch.mat[blockIdx.z];
    const int i0 = static_cast<int>(blockIdx.y) * 32, j0 = static_cast<int>(blockIdx.x) * 32;
    if (i0 >= d.mp || j0 >= d.np) return;
    const int tx = static_cast<int>(threadIdx.x) % 32, ty = static_cast<int>(threadIdx.x) / 32;
    if (threadIdx.x < kWave) {
        const double* part = reinterpret_cast<const double*>(static_cast<const char*>(ws) + d.partial);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kNormParts / kWave; ++i) sum += part[i * kWave + threadIdx.x];
        sum = wave_sum(sum);
        if (threadIdx.x == 0) total = sum;
    }
    for (int r = ty; r < 32; r += kThreads / 32) {  // along the update's rows
        const int i = d.tall ? i0 + tx : i0 + r, j = d.tall ? j0 + r : j0 + tx;
        const T* in = static_cast<const T*>(d.in);
        const float x = i >= d.m || j >= d.n ? 0.0f
                                             : static_cast<float>(d.tall ? in[j * d.in_stride + i] : in[i * d.in_stride + j]);
        if (d.tall)
            tile[tx][r] = x;
        else
            tile[r][tx] = x;
    }
    __syncthreads();
    const float scale = static_cast<float>(static_cast<double>(d.scale) / (sqrt(total) + static_cast<double>(rule.eps)));
    const Planes x = planes_x(ws, d), xt = planes_xt(ws, d, 0), xt1 = planes_xt(ws, d, 1), a = planes_a(ws, d),
                 b = planes_b(ws, d);
    for (int r = ty; r < 32; r += kThreads / 32) {
        if (i0 + r < d.m) {
            const Pair p = halves(tile[r][tx] * scale);
            const int64_t at = (i0 + r) * x.stride + j0 + tx;
            x.hi[at] = p.hi;
            x.lo[at] = p.lo;
        }
        if (j0 + r < d.n) {
            const Pair p = halves(tile[tx][r] * scale);
            const int64_t at = (j0 + r) * xt.stride + i0 + tx;
            xt.hi[at] = p.hi;
            xt.lo[at] = p.lo;
            if (i0 + tx >= d.m) xt1.hi[at] = xt1.lo[at] = static_cast<f16>(0.0f);
        }
    }
    // the columns past m of A and B: the workgroups of the last 32 columns of row block
    // 0 of X hold i0 = 0 only, so each workgroup of column 0 takes its 32 rows
    if (j0 == 0 && d.mp > d.m)
        for (int u = static_cast<int>(threadIdx.x); u < 32 * (d.mp - d.m); u += kThreads) {
            const int row = i0 + u / (d.mp - d.m), col = d.m + u % (d.mp - d.m);
            if (row < d.m) {
                const int64_t at = row * a.stride + col;
                a.hi[at] = a.lo[at] = b.hi[at] = b.lo[at] = static_cast<f16>(0.0f);
            }
        }
}

enum Product { kGram, kSquare, kUpdate };

// A tile of one of the three products of a step: BT x BT entries, 4 waves of (BT / 2)^2, a
// stage of depth 32 at a time.  While a stage is multiplied from registers, the next one's
// fragments come from LDS, the one after it goes from registers to LDS and the third is on
// its way from memory: one barrier a stage.  Bound by the matrix instructions: a wave of the
// 128-tile runs 48 of them (768 cycles) a stage beside 16 LDS reads and 8 writes of 1 KB.
// 2048 x 2048, per launch under the profiler: the 136 lower tiles 45 to 49 us (matrix instructions
// are busy for 48% of the waves' cycles), the update's 256 tiles 64 us; as 528 tiles of 64 x 64 the
// lower ones take 68.
template <typename T, int PRODUCT, int BT>
__global__ __launch_bounds__(kThreads, 2) void k_ortho_product(OrthoBatch batch, OrthoRule rule, int count, int step, void* ws) {
    constexpr int MT = BT / 32;
    constexpr int kRounds = BT * 4 / kThreads;  // 16-byte units of a thread per operand and plane
    // [buffer][operand][plane]: rows of 32 halves, their four 16-byte units exchanged by row
    // (unit u of row r lies at u ^ (r / 2 % 4)): eight neighbouring lanes then read or write
    // all banks once, along a row and down the rows
    __shared__ __align__(16) f16 lds[2][2][2][BT * 32];
    // the tile's matrix
    const int64_t flat = xcd_tile(blockIdx.x, gridDim.x);
    int which = 0;
    const int first_of = PRODUCT == kUpdate ? 1 : 0;
    while (which + 1 < count && flat >= batch.mat[which + 1].first_tile[first_of]) ++which;
    const OrthoMatrix& d = batch.mat[which];
    const int t = static_cast<int>(flat - d.first_tile[first_of]);
    int ti, tj;
    if constexpr (PRODUCT == kUpdate) {
        // eight tile rows at a time: the 32 tiles that an XCD has on its CUs then read 8 + 4
        // operand strips, not 16 + 2
        constexpr int kStrip = 8;
        const int rows = (d.m + BT - 1) / BT, cols = (d.n + BT - 1) / BT;
        const int strip = t / (kStrip * cols), in = t - strip * kStrip * cols, high = min(kStrip, rows - strip * kStrip);
        tj = in / high;
        ti = strip * kStrip + in - tj * high;
    } else {  // the lower triangle, row by row
        ti = static_cast<int>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
        while (ti * (ti + 1) / 2 > t) --ti;
        tj = t - ti * (ti + 1) / 2;
    }
    const Planes a = planes_a(ws, d), b = planes_b(ws, d);
    const Planes xt = planes_xt(ws, d, step & 1);
    Planes p, q;
    int depth, q_rows;
    if constexpr (PRODUCT == kGram) {
        p = q = planes_x(ws, d);
        depth = d.np;
        q_rows = d.m;
    } else if constexpr (PRODUCT == kSquare) {
        p = q = a;
        depth = d.mp;
        q_rows = d.m;
    } else {
        p = b;
        q = xt;
        depth = d.mp;
        q_rows = d.n;
    }
    const int r0 = ti * BT, c0 = tj * BT;
    const int tid = static_cast<int>(threadIdx.x), wave = tid / kWave, l = lane_id(), g = l / 16, c16 = l % 16;
    const int wr = (wave / 2) * (BT / 2), wc = (wave % 2) * (BT / 2);

    // rows past the matrix read its last one: their results are not stored
    const f16* const from[2][2] = {{p.hi + r0 * p.stride, p.lo + r0 * p.stride}, {q.hi + c0 * q.stride, q.lo + c0 * q.stride}};
    uint32_t offset[2][kRounds];
    int to[kRounds];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        const int row = (i * kThreads + tid) / 4, unit = tid % 4;
        offset[0][i] = static_cast<uint32_t>(min(row, d.m - 1 - r0) * p.stride + unit * 8);
        offset[1][i] = static_cast<uint32_t>(min(row, q_rows - 1 - c0) * q.stride + unit * 8);
        to[i] = row * 32 + (unit ^ (row / 2 % 4)) * 8;
    }
    // stages on their way: two of the small tile's, whose stage is over before a load arrives
    constexpr int kFlights = BT == 64 ? 2 : 1;
    struct Flight {
        Half8 v[2][2][kRounds];
    } flight[kFlights];
    auto fetch = [&](Flight& f, int k) {
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < kRounds; ++i)
                    f.v[o][h][i] = *reinterpret_cast<const Half8*>(from[o][h] + k + offset[o][i]);
    };
    auto settle = [&](const Flight& f, int buffer) {
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < kRounds; ++i) *reinterpret_cast<Half8*>(&lds[buffer][o][h][to[i]]) = f.v[o][h][i];
    };
    f32x4 acc[MT][MT];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) acc[r][c] = f32x4(0.0f);
    struct Stage {
        Half8 fh[MT], fl[MT], gh[MT], gl[MT];
    } even, odd;
    const int at = c16 * 32 + (g ^ (c16 / 2 % 4)) * 8;  // of the lane's unit within 16 rows
    auto read = [&](Stage& f, int buffer) {
#pragma unroll
        for (int r = 0; r < MT; ++r) {
            f.fh[r] = *reinterpret_cast<const Half8*>(&lds[buffer][0][0][(wr + 16 * r) * 32 + at]);
            f.fl[r] = *reinterpret_cast<const Half8*>(&lds[buffer][0][1][(wr + 16 * r) * 32 + at]);
            f.gh[r] = *reinterpret_cast<const Half8*>(&lds[buffer][1][0][(wc + 16 * r) * 32 + at]);
            f.gl[r] = *reinterpret_cast<const Half8*>(&lds[buffer][1][1][(wc + 16 * r) * 32 + at]);
        }
    };
    auto multiply = [&](const Stage& f) {  // the small terms first
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
            for (int c = 0; c < MT; ++c) acc[r][c] = mma<f16>(f.fl[r], f.gh[c], acc[r][c]);
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
            for (int c = 0; c < MT; ++c) acc[r][c] = mma<f16>(f.fh[r], f.gl[c], acc[r][c]);
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
            for (int c = 0; c < MT; ++c) acc[r][c] = mma<f16>(f.fh[r], f.gh[c], acc[r][c]);
    };
    const int stages = depth / 32;
    // Stage s, whose fragments are in `now`.  Past the last stage the reads, writes and loads
    // repeat it, unused, so that a pass has no branch and its instructions mix: one LDS or
    // memory access to every two matrix instructions, in this order.
    auto pass = [&](int s, const Stage& now, Stage& next_stage, Flight& f) {
        read(next_stage, (s + 1) & 1);
        multiply(now);
        settle(f, s & 1);  // stage s + 2 into the buffer of stage s, which all have read
        fetch(f, 32 * min(s + 2 + kFlights, stages - 1));
#pragma unroll
        for (int i = 0; i < 4 * MT; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);       // LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, MT / 2, 0);  // matrix instructions
        }
#pragma unroll
        for (int i = 0; i < 4 * kRounds; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // load
            __builtin_amdgcn_sched_group_barrier(0x008, MT * MT * 3 / (4 * kRounds) - MT * MT / (2 * kRounds), 0);
        }
        __syncthreads();
    };
    Flight &first = flight[0], &second = flight[kFlights - 1];
    fetch(first, 0);
    settle(first, 0);
    fetch(second, 32 * min(1, stages - 1));
    if constexpr (kFlights == 2) fetch(first, 32 * min(2, stages - 1));
    __syncthreads();
    read(even, 0);
    settle(second, 1);
    fetch(second, 32 * min(1 + kFlights, stages - 1));
    __syncthreads();
    int s = 0;
    for (; s + 1 < stages; s += 2) {
        pass(s, even, odd, first);
        pass(s + 1, odd, even, second);
    }
    if (s < stages) multiply(even);

    const float to_a = rule.scale_a / (d.scale * d.scale), from_b = 1.0f / rule.scale_b;
    const float b_of_a = rule.b * rule.scale_b / rule.scale_a, b_of_aa = rule.c * rule.scale_b / (rule.scale_a * rule.scale_a);
    const Planes x = planes_x(ws, d), xt_new = planes_xt(ws, d, (step & 1) ^ 1);
    const bool last = step + 1 == rule.steps;
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) {
            // entries (row0 .. row0 + 3, col)
            const int row0 = r0 + wr + 16 * r + 4 * g, col = c0 + wc + 16 * c + c16;
            if (row0 >= d.m || col >= q_rows) continue;
            f32x4 v = acc[r][c];
            if constexpr (PRODUCT == kGram) {
                v *= to_a;
            } else {
                const Planes& old = PRODUCT == kSquare ? a : xt;  // A is symmetric
                const Half4 oh = *reinterpret_cast<const Half4*>(old.hi + col * old.stride + row0);
                const Half4 ol = *reinterpret_cast<const Half4*>(old.lo + col * old.stride + row0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (PRODUCT == kSquare)
                        v[i] = whole(oh[i], ol[i]) * b_of_a + v[i] * b_of_aa;
                    else
                        v[i] = fmaf(rule.a, whole(oh[i], ol[i]), v[i] * from_b);
                }
            }
            if constexpr (PRODUCT == kUpdate) {
                if (last) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (row0 + i < d.m) put_entry<T>(d, row0 + i, col, v[i] / d.scale);
                    continue;
                }
            }
            const Planes& direct = PRODUCT == kGram ? a : PRODUCT == kSquare ? b : x;
            const Planes& turned = PRODUCT == kGram ? a : PRODUCT == kSquare ? b : xt_new;
            Half4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Pair pr = row0 + i < d.m ? halves(v[i]) : Pair{static_cast<f16>(0.0f), static_cast<f16>(0.0f)};
                hi[i] = pr.hi;
                lo[i] = pr.lo;
                // a tile on the diagonal is written once, as its own mirror image
                if (row0 + i < d.m && (PRODUCT == kUpdate || ti != tj)) {
                    direct.hi[(row0 + i) * direct.stride + col] = pr.hi;
                    direct.lo[(row0 + i) * direct.stride + col] = pr.lo;
                }
            }
            // the padded width holds all four (zeros past m)
            *reinterpret_cast<Half4*>(turned.hi + col * turned.stride + row0) = hi;
            *reinterpret_cast<Half4*>(turned.lo + col * turned.stride + row0) = lo;
        }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// LDS of k_ortho_small.
size_t small_bytes(int64_t mp, int64_t np) { return static_cast<size_t>(2 * mp * (np + 8) + 2 * mp * (mp + 8)) * sizeof(f16); }

constexpr size_t kSmallLds = 160 * 1024 - 256;  // a CU's, less the kernel's own

bool is_small(const relm_mp_update& u) {
    const int64_t mp = ceil_div(std::min(u.rows, u.cols), 32) * 32, np = ceil_div(std::max(u.rows, u.cols), 32) * 32;
    return mp <= 128 && np <= 16384 && small_bytes(mp, np) <= kSmallLds;
}

// Whether matrices that would fit a workgroup go with the larger ones: where there are some
// and one launch holds them all, their tiles cost nothing beside the others', and the launch
// of their own is saved (two of 398 x 11 beside four of up to 398 x 387: 48 of 190 us).
bool small_join(const relm_mp_update* updates, int32_t count) {
    if (count > kOrthoBatch) return false;
    for (int32_t i = 0; i < count; ++i)
        if (updates[i].rows > 0 && updates[i].cols > 0 && !is_small(updates[i])) return true;
    return false;
}

// Sizes of a matrix; its planes from `at` on in the workspace unless it is `small`.
OrthoMatrix describe(const relm_mp_update& u, bool small, size_t& at) {
    OrthoMatrix d{};
    d.in = u.in;
    d.out = u.out;
    d.in_stride = u.row_stride;
    d.tall = u.rows > u.cols;
    d.m = static_cast<int32_t>(std::min(u.rows, u.cols));
    d.n = static_cast<int32_t>(std::max(u.rows, u.cols));
    d.mp = static_cast<int32_t>(ceil_div(d.m, 32) * 32);
    d.np = static_cast<int32_t>(ceil_div(d.n, 32) * 32);
    // 2^round(log2 sqrt(m n)), at most 2^13: the entries of X are about 1 at first, and
    // no more than twice the scale throughout
    const int e = static_cast<int>(std::lround(0.5 * std::log2(static_cast<double>(d.m) * static_cast<double>(d.n))));
    d.scale = std::ldexp(1.0f, std::min(e, 13));
    d.inv_cols = ((uint64_t{1} << 40) + u.cols - 1) / u.cols;
    if (small) return d;
    const auto take = [&](size_t bytes) {
        const size_t p = at;
        at = align_up(at + bytes, 256);
        return static_cast<int64_t>(p);
    };
    const size_t m = d.m, n = d.n, mp = d.mp, np = d.np;
    d.x = take(4 * m * np);
    d.xt[0] = take(4 * n * mp);
    d.xt[1] = take(4 * n * mp);
    d.a = take(4 * m * mp);
    d.b = take(4 * m * mp);
    d.partial = take(kNormParts * sizeof(double));
    return d;
}

// Numbers the tiles of one kind (0: the lower ones of a symmetric product, 1: the update's)
// of a launch's matrices; their count.
int64_t number_tiles(OrthoBatch& b, int count, int64_t bt, int kind) {
    int64_t at = 0;
    for (int i = 0; i < count; ++i) {
        OrthoMatrix& d = b.mat[i];
        d.first_tile[kind] = at;
        const int64_t r = ceil_div(d.m, bt), c = ceil_div(d.n, bt);
        at += kind == 0 ? r * (r + 1) / 2 : r * c;
    }
    return at;
}

template <typename T, int PRODUCT>
void product(const OrthoBatch& b, const OrthoRule& rule, int count, int step, bool large, int64_t tiles, void* ws,
             hipStream_t st) {
    const auto kernel = large ? k_ortho_product<T, PRODUCT, 128> : k_ortho_product<T, PRODUCT, 64>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles)), dim3(kThreads), 0, st, b, rule, count, step, ws);
}

// Sets the kernel's LDS limit on the current device, if that has not been done there.
template <typename T>
hipError_t allow_small_lds() {
    constexpr int kDevices = 64;
    static std::atomic<bool> done[kDevices];
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const bool known = device >= 0 && device < kDevices;
    if (known && done[device].load(std::memory_order_acquire)) return hipSuccess;
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_ortho_small<T>), hipFuncAttributeMaxDynamicSharedMemorySize, kSmallLds);
    if (e == hipSuccess && known) done[device].store(true, std::memory_order_release);
    return e;
}

template <typename T>
hipError_t run(const std::vector<OrthoMatrix>& small, const std::vector<OrthoMatrix>& large, const OrthoRule& rule, void* ws,
               hipStream_t st) {
    if (!small.empty()) {
        const hipError_t e = allow_small_lds<T>();
        if (e != hipSuccess) return e;
    }
    for (size_t i = 0; i < small.size(); i += kOrthoBatch) {
        OrthoBatch b{};
        const size_t count = std::min<size_t>(kOrthoBatch, small.size() - i);
        size_t lds = 0;
        for (size_t k = 0; k < count; ++k) {
            b.mat[k] = small[i + k];
            lds = std::max(lds, small_bytes(b.mat[k].mp, b.mat[k].np));
        }
        hipLaunchKernelGGL(k_ortho_small<T>, dim3(static_cast<unsigned>(count)), dim3(kSmallThreads), lds, st, b, rule);
    }
    for (size_t i = 0; i < large.size(); i += kOrthoBatch) {
        OrthoBatch b{};
        const int count = static_cast<int>(std::min<size_t>(kOrthoBatch, large.size() - i));
        int mp = 0, np = 0;
        for (int k = 0; k < count; ++k) {
            b.mat[k] = large[i + k];
            mp = std::max(mp, b.mat[k].mp);
            np = std::max(np, b.mat[k].np);
        }
        hipLaunchKernelGGL(k_ortho_norm<T>, dim3(kNormParts, count), dim3(kThreads), 0, st, b, ws);
        hipLaunchKernelGGL(k_ortho_split<T>, dim3(np / 32, mp / 32, count), dim3(kThreads), 0, st, b, rule, ws);
        int64_t tiles[2];
        bool wide[2];
        for (int kind = 0; kind < 2; ++kind) {
            tiles[kind] = number_tiles(b, count, 128, kind);
            wide[kind] = tiles[kind] >= kLargeTiles[kind];
            if (!wide[kind]) tiles[kind] = number_tiles(b, count, 64, kind);
        }
        for (int step = 0; step < rule.steps; ++step) {
            product<T, kGram>(b, rule, count, step, wide[0], tiles[0], ws, st);
            product<T, kSquare>(b, rule, count, step, wide[0], tiles[0], ws, st);
            product<T, kUpdate>(b, rule, count, step, wide[1], tiles[1], ws, st);
        }
    }
    return hipGetLastError();
}

}  // namespace

size_t orthogonalise_workspace(const relm_mp_update* updates, int32_t count) {
    size_t at = 0;
    const bool join = small_join(updates, count);
    for (int32_t i = 0; i < count; ++i)
        if (updates[i].rows > 0 && updates[i].cols > 0) describe(updates[i], !join && is_small(updates[i]), at);
    return at;
}

hipError_t launch_orthogonalise(int dtype, const relm_mp_update* updates, int32_t count, const OrthoRule& rule, void* ws,
                                hipStream_t st) {
    std::vector<OrthoMatrix> small, large;
    size_t at = 0;
    const bool join = small_join(updates, count);
    for (int32_t i = 0; i < count; ++i) {
        if (updates[i].rows == 0 || updates[i].cols == 0) continue;
        const bool fits = !join && is_small(updates[i]);
        (fits ? small : large).push_back(describe(updates[i], fits, at));
    }
    hipError_t e = hipErrorInvalidValue;
    with_value_type(dtype, [&](auto t) { e = run<decltype(t)>(small, large, rule, ws, st); });
    return e;
}

}  // namespace relm_mp
