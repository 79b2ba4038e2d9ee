// Cross attention of per-graph queries to their graph's keys, forward and backward:
//
//   s = scale * q k^T,  p = softmax(s),  out = p v,  lse = log(sum exp s)
//   delta = <grad, out>,  ds = p (grad v^T - delta),
//   dq = scale * ds k,  dk = scale * ds^T q,  dv = p^T grad
//
// One pass over the keys with the running maximum and total of each row's softmax;
// the scores stay in registers.  The scores are computed transposed (keys down,
// queries across): a lane then holds four neighbouring keys of one query, which is
// what the next product wants as an operand, so probabilities go from one matrix
// instruction to the next without leaving the lane, and a query's statistics are one
// value per lane.  Scores, statistics, totals and all accumulators are float.
// Probabilities and ds are rounded to the values' type for the products that read
// them: each such rounding is independent of the others and of the size of the
// outputs' own, so that an output errs by up to 1.5 times that one (two roundings in
// the place of one; 16-bit products are nine times the float ones' rate).  With float
// values nothing is rounded.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention.h"
#include "device_utils.h"
#include "internal.h"
#include "mfma_tiles.h"
#include "value_types.h"

namespace relm_mp {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// An operand [rows, heads, head_dim] by its strides.
template <typename T>
struct Rows {
    const T* data;
    int64_t row_stride, head_stride;
};

template <typename T>
Rows<T> rows_of(const relm_mp_head_rows& r) {
    return {static_cast<const T*>(r.data), r.row_stride, r.head_stride};
}

// Units of 16 bytes of a row of `dim` values, from column `col` on, zero past its end: one
// access each, wherever rows start.  A unit that lies past the row is its first; one that
// ends past it (kCut: 8 does not divide dim) is read ending with the row and moved down
// after (settle_unit: 3 to 6% of a kernel's time, so rows of whole units have kernels without
// it).  Rows of fewer than 8 values (kShort) go value by value.  Nothing branches: loads on
// both sides of a branch would wait for one another.
enum Fit { kShort, kCut, kWhole };

template <typename T>
constexpr int kUnit = 16 / static_cast<int>(sizeof(T));
template <typename T, int N>
using Values = T __attribute__((ext_vector_type(N)));
template <typename T>
using Unit = Values<T, kUnit<T>>;

template <typename T, int FIT>
__device__ __forceinline__ Unit<T> load_unit(const T* p, int col, int dim) {
    constexpr int N = kUnit<T>;
    if constexpr (FIT != kShort) {
        return *reinterpret_cast<const ValueVec<T, N>*>(p + (col < dim ? min(col, dim - N) : 0));
    } else {
        Unit<T> v;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = p[min(col + j, dim - 1)];
        return v;
    }
}

template <typename T, int FIT>
__device__ __forceinline__ Unit<T> settle_unit(Unit<T> v, int col, int dim) {
    constexpr int N = kUnit<T>;
    if constexpr (FIT != kShort) {
        if constexpr (FIT == kCut) {
            const int down = (col < dim ? max(col + N - dim, 0) : 0) * static_cast<int>(8 * sizeof(T));  // bits
            struct Words {
                uint64_t lo, hi;
            } w = __builtin_bit_cast(Words, v);
            const uint64_t carried = down == 0 ? 0 : w.hi << ((64 - down) & 63);
            w.lo = down >= 64 ? w.hi >> (down & 63) : (w.lo >> (down & 63)) | carried;
            w.hi = down >= 64 ? 0 : w.hi >> (down & 63);
            v = __builtin_bit_cast(Unit<T>, w);
        }
        if (col >= dim) v = Unit<T>(static_cast<T>(0.0f));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (col + j >= dim) v[j] = static_cast<T>(0.0f);
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void put4(T* p, int col, int dim, f32x4 x) {
    if (col + 4 <= dim) {
        ValueVec<T, 4> v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = round_to<T>(x[j]);
        *reinterpret_cast<ValueVec<T, 4>*>(p + col) = v;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < dim) p[col + j] = round_to<T>(x[j]);
    }
}

template <typename T>
struct Args {
    Rows<T> q, k, v, grad;
    const uint8_t* key_mask;
    int dim;
    int heads, kv_heads, group;
    int row_tile, key_tile;
    float scale;
    int num_items;
    const AttnItem* items;
    const AttnJoin* joins;
    T* out;
    float* lse;     // forward, may be NULL
    RowStats* stats;  // forward (may be NULL): written; backward: read
    float* delta;
    T *dq, *dk, *dv;
    float* parts;        // sums of the parts, rows of part_stride floats
    float* part_stats;   // forward: their maxima and totals
    int part_stride;
};

// What the forward leaves of row `at` (query and head): its statistics and their logarithm.  A
// row that had no finite score gets probabilities of 0.
template <typename T>
__device__ __forceinline__ void put_stats(const Args<T>& a, int64_t at, float top, float total) {
    const bool none = total == 0.0f;
    if (a.lse != nullptr) a.lse[at] = none ? -kInf : fmaf(top, a.scale, log2f(total) * kLn2);
    if (a.stats != nullptr) a.stats[at] = {none ? 0.0f : top, none ? 0.0f : 1.0f / total};
}

// A workgroup's item and key head.  Neighbouring heads of an item share the lines of
// its rows, and neighbouring items a graph's keys: they run on one XCD.
struct Work {
    AttnItem it;
    int head;
};
__device__ __forceinline__ Work work_of(const AttnItem* items, int num_items, int kv_heads) {
    const int flat = static_cast<int>(xcd_tile(blockIdx.x, static_cast<int64_t>(num_items) * kv_heads));
    const int item = flat / kv_heads;
    return {items[item], flat - item * kv_heads};
}

// Where row r of a graph lies: its query and head (the head counted over all heads).
struct Place {
    int64_t row;
    int head;
};
template <typename T>
__device__ __forceinline__ Place place_of(const Args<T>& a, int q_first, int kv_head, int r) {
    const int q = a.group == 1 ? r : r / a.group;
    return {static_cast<int64_t>(q_first) + q, kv_head * a.group + (r - q * a.group)};
}

// BN rows of an operand in flight from global memory to LDS: a thread holds its share of
// the tile in registers while the tile before it is computed on.  Rows of LDS are padded
// by 16 bytes, which spreads a column's rows over the banks.
template <typename T, int DP>
constexpr int kLdsStride = DP + 16 / static_cast<int>(sizeof(T));

template <typename T, int DP, int BN>
struct TileLoad {
    static constexpr int kUnits = DP / kUnit<T>;         // of a row
    static constexpr int kStep = kThreads / kUnits;      // rows of a round
    static constexpr int kRounds = BN / kStep;
    static_assert(kThreads % kUnits == 0 && BN % kStep == 0, "whole rounds");
    Unit<T> v[kRounds];

    static __device__ __forceinline__ int first_row() { return static_cast<int>(threadIdx.x) / kUnits; }
    static __device__ __forceinline__ int column() { return (static_cast<int>(threadIdx.x) % kUnits) * kUnit<T>; }

    // place(row): where a row of the tile lies (some row that exists for one that does not)
    template <int FIT, typename F>
    __device__ __forceinline__ void fetch(F&& place, int dim) {
#pragma unroll
        for (int i = 0; i < kRounds; ++i) v[i] = load_unit<T, FIT>(place(first_row() + i * kStep), column(), dim);
    }
    // Into LDS; unless `all` rows enter, those that keep(row) leaves out as zeros.
    template <int FIT, typename F>
    __device__ __forceinline__ void store(T* tile, int dim, bool all, F&& keep) const {
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int row = first_row() + i * kStep;
            Unit<T> x = settle_unit<T, FIT>(v[i], column(), dim);
            if (!all && !keep(row)) x = Unit<T>(static_cast<T>(0.0f));
            *reinterpret_cast<Unit<T>*>(tile + row * kLdsStride<T, DP> + column()) = x;
        }
    }
};

// Which of a tile's BN keys are kept: bit k of the words.
template <int BN>
struct KeyBits {
    uint32_t byte[BN / 64];
    uint64_t bits[BN / 64];
    // asks for the mask's bytes of keys [first, first + left), left > 0
    __device__ __forceinline__ void fetch(const uint8_t* mask, int64_t first, int left) {
#pragma unroll
        for (int w = 0; w < BN / 64; ++w) {
            const int k = w * 64 + lane_id();
            byte[w] = mask != nullptr ? mask[first + min(k, left - 1)] : 1u;
            byte[w] = k < left ? byte[w] : 0u;
        }
    }
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int w = 0; w < BN / 64; ++w) bits[w] = __ballot(byte[w] != 0);
    }
    __device__ __forceinline__ bool all() const { return (bits[0] & bits[BN / 64 - 1]) == ~0ull; }
    __device__ __forceinline__ bool none() const { return (bits[0] | bits[BN / 64 - 1]) == 0; }
    __device__ __forceinline__ uint64_t word(int k) const { return BN == 128 && (k & 64) ? bits[BN / 64 - 1] : bits[0]; }
    __device__ __forceinline__ bool has(int k) const { return (word(k) >> (k % 64)) & 1; }
};

// Fragments of 16 rows of q (or grad) that a wave keeps: lane l holds row l % 16.
template <typename T, int DP>
struct RowFrags {
    Frag<T> f[DP / 32];
    template <int FIT>
    __device__ __forceinline__ void fetch(const T* p, int dim) {
        const int g = lane_id() / 16;
        constexpr int N = kUnit<T>;
        Unit<T> u[DP / 32][8 / N];
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
#pragma unroll
            for (int h = 0; h < 8 / N; ++h) u[c][h] = load_unit<T, FIT>(p, c * 32 + g * 8 + h * N, dim);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
#pragma unroll
            for (int h = 0; h < 8 / N; ++h) {
                const Unit<T> x = settle_unit<T, FIT>(u[c][h], c * 32 + g * 8 + h * N, dim);
#pragma unroll
                for (int j = 0; j < N; ++j) f[c][h * N + j] = x[j];
            }
    }
};

// Products of 32 keys (rows of a tile, from key0 on) with RT tiles of 16 rows, keys down:
// two tiles of 16 keys each, on top of `start`.
template <typename T, int DP, int RT>
__device__ __forceinline__ void keys_by_rows(const T* keys, int key0, const RowFrags<T, DP> (&rows)[RT], const f32x4 (&start)[2],
                                             f32x4 (&s)[RT][2]) {
    const int l = lane_id();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r][t] = start[t];
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            const Frag<T> k = lds_frag<T>(keys, kLdsStride<T, DP>, key0 + 16 * t + l % 16, c * 32 + (l / 16) * 8);
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r][t] = mma<T>(k, rows[r].f[c], s[r][t]);
        }
    }
}

// What the scores of the lane's keys start from: 0, or -inf for a key that is not kept
// (whose values are zeros in LDS).  The products then need no selection.
__device__ __forceinline__ void key_starts(const float* starts, int key0, f32x4 (&start)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) start[t] = *reinterpret_cast<const f32x4*>(starts + key0 + 16 * t + 4 * (lane_id() / 16));
}

// Over the four lanes that share a query (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float lanes_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Half values end at 2^-14 (below, they lose bits, and below 2^-25 all of them): the
// probabilities of a query with tens of thousands of keys would, and those of all keys beside
// one that lies 10 above them.  They are at most 1, so products read them in units of 2^-15.
template <typename T>
constexpr float kProbabilityUnit = std::is_same_v<T, f16> ? 32768.0f : 1.0f;

// The exponent of a score s under its row's maximum m, sl2 (s - m).  As fma(s, sl2, -(sl2 m)) it is
// one instruction, and off by the rounding of sl2 m: nothing of a row's own distribution is
// lost, but the largest probability is not 1, and from 2^30 on that rounding passes the
// exponent's range (below the largest float everything was infinite, or 0).
//
// Forward: rows past kFarScore take the difference first, which is exact near the maximum: `off`
// is then m and `base` 0.  Float rows always do (2^-24 is their own accuracy, and matrix
// instructions bound them); 16-bit ones have 2^-17 up to there, a thirtieth of a half's unit.
// The branch that this takes stands behind the tile's maximum, which has read the scores.  One
// between a matrix instruction and the first use of its result would be wrong: this compiler
// leaves out the wait that such a use needs behind a taken branch.
constexpr float kFarScore = 256.0f;

template <typename T>
struct Under {
    float base, off;
    __device__ __forceinline__ Under() = default;
    __device__ __forceinline__ Under(float top, float sl2) {
        const float m = top == -kInf ? 0.0f : top;
        const bool far = sizeof(T) == 4 || fabsf(m * sl2) >= kFarScore;
        base = far ? 0.0f : m * sl2;
        off = far ? m : 0.0f;
    }
    __device__ __forceinline__ bool far() const { return sizeof(T) == 4 || off != 0.0f; }
};
// Takes off from scores where some row of the wave is far.
template <int N>
__device__ __forceinline__ void lower(f32x4 (&s)[N], float off) {
#pragma unroll
    for (int t = 0; t < N; ++t) s[t] -= off;
}

// Backward: the row's statistics are known, so the rounding of its base is too, and goes into the
// factor that divides by the total: p = 2^(slope s - base) * share, without a branch.  Past
// kLastScore scores that are not equal lie 64 and more apart in units of the exponent, so
// only equal ones share the row: there the slope is a power of two, exact on all of them.
constexpr float kLastScore = 1073741824.0f;  // 2^30

struct RowScore {
    float slope, base, share;
    __device__ __forceinline__ RowScore() = default;
    __device__ __forceinline__ RowScore(RowStats r, float sl2) {
        slope = sl2;
        base = r.top * sl2;
        share = r.inv_total * exp2_of(-fmaf(r.top, sl2, -base));
        if (!(fabsf(base) < kLastScore)) {
            const int e = static_cast<int>(__float_as_uint(r.top) >> 23 & 255);  // top * slope in [2^30, 2^31)
            slope = __uint_as_float(static_cast<unsigned>(min(max(284 - e, 1), 254)) << 23);
            base = r.top * slope;
            share = r.inv_total;
        }
    }
};

// Two waves to a SIMD with 16-bit values: one's matrix instructions run beside the other's
// exponentials.  Float rows need the registers of both.
template <typename T>
constexpr int kWavesPerSimd = sizeof(T) == 2 ? 2 : 1;
// Float rows of 32 values, one tile to a wave: LDS holds four workgroups, and so do registers
// when asked to (of themselves they take 130, for three: 512 graphs of 8 x 200 in 16.1 us, not 14.8).
template <typename T, int DP, int RT>
constexpr int kForwardWaves = sizeof(T) == 4 && DP == 32 && RT == 1 ? 4 : kWavesPerSimd<T>;

// Shapes of the row kernels: a wave has RT tiles of 16 rows; WM waves have rows of their
// own and 4 / WM share each row tile, taking different keys of a tile.
template <int RT, int WM>
struct RowShape {
    static constexpr int kRows = 16 * RT * WM;             // of a workgroup
    static constexpr int kSharers = kWaves / WM;           // waves on one row tile
    static constexpr int kKeys = kSharers == 4 ? 128 : 64; // of a tile in LDS
    static constexpr int kChunks = kKeys / (32 * kSharers);  // 32-key chunks of a wave per tile
};

// Forward.  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m) with the running maximum m:
// when a key tile raises it, what has been added up is scaled by exp(m_old - m_new).
// Long rows of work are bound by the exponentials and conversions beside the matrix
// instructions: 4 x 2048 queries x 4096 keys,
// 16 heads of 128 over 4 key heads, bfloat16, 338 us (815 TFLOP/s).  Few rows are bound by
// the reads of keys and values: one query over 262,147 keys, 2 key heads of 64 in half
// precision, in 512 parts 31 us (4.3 TB/s); 2048 graphs of 64 to 512 keys, up to 32 queries,
// 4 heads of 32 in bfloat16 95 us (3.4 TB/s).
template <typename T, int DP, int RT, int WM, int FIT>
__global__ __launch_bounds__(kThreads, (kForwardWaves<T, DP, RT>)) void k_attention(Args<T> a) {
    using S = RowShape<RT, WM>;
    constexpr int BN = S::kKeys, ST = kLdsStride<T, DP>, ND = DP / 16;
    constexpr int kTileBytes = 2 * BN * ST * static_cast<int>(sizeof(T));
    constexpr int kMergeBytes = S::kSharers > 1 ? kWaves * 16 * RT * (DP + 2) * 4 : 0;
    __shared__ __align__(16) char lds[kTileBytes > kMergeBytes ? kTileBytes : kMergeBytes];
    __shared__ __align__(16) float starts[BN];
    T* kt = reinterpret_cast<T*>(lds);
    T* vt = kt + BN * ST;
    const Work w = work_of(a.items, a.num_items, a.kv_heads);
    const int l = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave, g = l / 16;
    const int row_wave = wave / S::kSharers, key_wave = wave % S::kSharers;
    const float sl2 = a.scale * kLog2e;

    RowFrags<T, DP> qf[RT];
    Place at[RT];
    bool real[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = (row_wave * RT + r) * 16 + l % 16;
        real[r] = row < w.it.rows;
        at[r] = place_of(a, w.it.q_first, w.head, w.it.row0 + (real[r] ? row : 0));
        // a row past the item reads its first: a column of the scores, used by no other
        qf[r].template fetch<FIT>(a.q.data + at[r].row * a.q.row_stride + at[r].head * a.q.head_stride, a.dim);
    }
    f32x4 o[RT][ND];
    float m[RT], total[RT];
    Under<T> under[RT];
    bool far = false;  // whether some row of the wave is
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        m[r] = -kInf;
        total[r] = 0.0f;
        under[r] = Under<T>(m[r], sl2);
#pragma unroll
        for (int n = 0; n < ND; ++n) o[r][n] = f32x4(0.0f);
    }

    TileLoad<T, DP, BN> kl, vl;
    KeyBits<BN> bits;
    const auto fetch = [&](int k0) {
        const int left = w.it.keys - k0;
        const int64_t first = static_cast<int64_t>(w.it.key_first) + k0;
        const T* kp = a.k.data + first * a.k.row_stride + w.head * a.k.head_stride;
        const T* vp = a.v.data + first * a.v.row_stride + w.head * a.v.head_stride;
        kl.template fetch<FIT>([&](int row) { return kp + min(row, left - 1) * a.k.row_stride; }, a.dim);
        vl.template fetch<FIT>([&](int row) { return vp + min(row, left - 1) * a.v.row_stride; }, a.dim);
        bits.fetch(a.key_mask, first, left);
    };
    bool any = false;  // whether some key of the item is kept (the same for all waves)
    if (w.it.keys > 0) fetch(0);
    for (int k0 = 0; k0 < w.it.keys; k0 += BN) {
        bits.settle();
        any = any || !bits.none();
        __syncthreads();
        kl.template store<FIT>(kt, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        vl.template store<FIT>(vt, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        if (threadIdx.x < BN) starts[threadIdx.x] = bits.has(threadIdx.x) ? 0.0f : -kInf;
        __syncthreads();
        if (k0 + BN < w.it.keys) fetch(k0 + BN);
        f32x4 s[S::kChunks][RT][2];
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int key0 = (key_wave * S::kChunks + c) * 32;
            f32x4 start[2];
            key_starts(starts, key0, start);
            keys_by_rows<T, DP, RT>(kt, key0, qf, start, s[c]);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float top = -kInf;  // the scale is positive: also the scaled scores' maximum
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[c][r][t][i]);
            const float most = fmaxf(m[r], lanes_max(top));
            if (__any(most > m[r])) {
                const float shrink = exp2_of((m[r] - (most == -kInf ? 0.0f : most)) * sl2);
                total[r] *= shrink;
#pragma unroll
                for (int n = 0; n < ND; ++n) o[r][n] *= shrink;
                m[r] = most;
                if constexpr (sizeof(T) == 2) {
                    under[r] = Under<T>(most, sl2);
                    far = far || __any(under[r].far());
                }
            }
            // (of float rows from m: a register more to a row cost a wave to a SIMD)
            const Under<T> now = sizeof(T) == 2 ? under[r] : Under<T>(m[r], sl2);
            if (sizeof(T) == 4 || far) {
#pragma unroll
                for (int c = 0; c < S::kChunks; ++c) lower(s[c][r], now.off);
            }
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = exp2_of(fmaf(s[c][r][t][i], sl2, -now.base));
                        s[c][r][t][i] = p * kProbabilityUnit<T>;
                        total[r] += p;
                    }
        }
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int key0 = (key_wave * S::kChunks + c) * 32;
            Frag<T> p[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) p[r] = frag_of<T>(s[c][r][0], s[c][r][1]);
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                const Frag<T> vf = lds_frag_t<T>(vt, ST, key0, n * 16);
#pragma unroll
                for (int r = 0; r < RT; ++r) o[r][n] = mma<T>(vf, p[r], o[r][n]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        total[r] = lanes_sum(total[r]);
#pragma unroll
        for (int n = 0; n < ND; ++n) o[r][n] *= 1.0f / kProbabilityUnit<T>;
        if (!any) {  // nothing to read: zeros, whatever an infinite query made of it
            m[r] = -kInf;
            total[r] = 0.0f;
#pragma unroll
            for (int n = 0; n < ND; ++n) o[r][n] = f32x4(0.0f);
        }
    }

    const auto finish = [&](int row, Place p, int col, f32x4 sum, float top, float sum_p) {
        if (w.it.part < 0) {
            const float inv = sum_p == 0.0f ? 0.0f : 1.0f / sum_p;
            put4<T>(a.out + (p.row * a.heads + p.head) * a.dim, col, a.dim, sum * inv);
            if (col == 0) put_stats(a, p.row * a.heads + p.head, top, sum_p);
        } else {
            const int64_t slot = (static_cast<int64_t>(w.it.part) * a.kv_heads + w.head) * a.row_tile + row;
            if (col < a.part_stride) *reinterpret_cast<f32x4*>(a.parts + slot * a.part_stride + col) = sum;
            if (col == 0) {
                a.part_stats[2 * slot] = top;
                a.part_stats[2 * slot + 1] = sum_p;
            }
        }
    };
    if constexpr (S::kSharers == 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
            if (real[r])
#pragma unroll
                for (int n = 0; n < ND; ++n)
                    finish((row_wave * RT + r) * 16 + l % 16, at[r], n * 16 + g * 4, o[r][n], m[r], total[r]);
    } else {
        // the sharers' sums, brought to the largest of their maxima, meet in LDS
        constexpr int R = 16 * RT;
        float* tops = reinterpret_cast<float*>(lds);  // [kWaves][R]
        float* totals = tops + kWaves * R;
        float* sums = totals + kWaves * R;            // [kWaves][R][DP]
        __syncthreads();
        if (g == 0) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                tops[wave * R + r * 16 + l] = m[r];
                totals[wave * R + r * 16 + l] = total[r];
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < ND; ++n)
                *reinterpret_cast<f32x4*>(sums + (wave * R + r * 16 + l % 16) * DP + n * 16 + g * 4) = o[r][n];
        __syncthreads();
        for (int u = static_cast<int>(threadIdx.x); u < w.it.rows * (DP / 4); u += kThreads) {
            const int row = u / (DP / 4), col = (u % (DP / 4)) * 4;
            if (col >= a.dim) continue;
            const int slot = (row / R) * S::kSharers * R + row % R;  // the first sharer's
            float top = -kInf, sum_p = 0.0f;
#pragma unroll
            for (int v = 0; v < S::kSharers; ++v) top = fmaxf(top, tops[v * R + slot]);
            const float most = top == -kInf ? 0.0f : top;
            f32x4 sum = f32x4(0.0f);
#pragma unroll
            for (int v = 0; v < S::kSharers; ++v) {
                const float share = exp2_of((tops[v * R + slot] - most) * sl2);
                sum_p = fmaf(totals[v * R + slot], share, sum_p);
                sum += *reinterpret_cast<const f32x4*>(sums + (v * R + slot) * DP + col) * share;
            }
            finish(row, place_of(a, w.it.q_first, w.head, w.it.row0 + row), col, sum, top, sum_p);
        }
    }
}

// Joins the parts of a row: out = sum_p e^(m_p - m) sum_p / sum_p e^(m_p - m) total_p, or
// dq = sum of the parts (DQ).  Thread groups of DP / 4 threads hold a row's sums.  MANY: a
// workgroup per row and key head, its groups taking every kJoinGroups-th part; else a row
// to each group.  Latency bound: 512 parts are 32 rounds of loads of a group, four at a time
// (7 us for 4 rows of 2 key heads; 55 us with a thread to a value and no rounds in flight).
template <int DP>
constexpr int kJoinGroups = kThreads / (DP / 4);

template <typename T, int DP, bool MANY, bool DQ>
__global__ __launch_bounds__(kThreads) void k_attention_join(Args<T> a) {
    constexpr int G = kJoinGroups<DP>, W = DP / 4;
    __shared__ float lds_top[kThreads / kWave], lds_total[G];
    __shared__ __align__(16) f32x4 lds_sum[MANY ? G * W : 1];
    const int t = static_cast<int>(threadIdx.x), col = (t % W) * 4, grp = t / W, head = static_cast<int>(blockIdx.y);
    const int per = MANY ? a.row_tile : a.row_tile / G;  // workgroups of a join
    const AttnJoin j = a.joins[blockIdx.x / per];
    const int row = static_cast<int>(blockIdx.x % per) * (MANY ? 1 : G) + (MANY ? 0 : grp);
    if (MANY && row >= j.rows) return;
    const int64_t slot0 = (static_cast<int64_t>(j.part0) * a.kv_heads + head) * a.row_tile + row;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * a.row_tile;
    const bool mine = row < j.rows && col < a.part_stride;
    float top = -kInf;
    if constexpr (!DQ) {
        if constexpr (MANY) {
            for (int p = t; p < j.parts; p += kThreads) top = fmaxf(top, a.part_stats[2 * (slot0 + p * step)]);
#pragma unroll
            for (int o = kWave / 2; o > 0; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
            if (lane_id() == 0) lds_top[t / kWave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kThreads / kWave; ++w) top = fmaxf(top, lds_top[w]);
        } else if (row < j.rows) {
            for (int p = 0; p < j.parts; ++p) top = fmaxf(top, a.part_stats[2 * (slot0 + p * step)]);
        }
    }
    const float sl2 = a.scale * kLog2e, most = top == -kInf ? 0.0f : top;
    f32x4 sum = f32x4(0.0f);
    float total = 0.0f;
    if (mine) {
#pragma unroll 4
        for (int p = MANY ? grp : 0; p < j.parts; p += MANY ? G : 1) {
            const int64_t slot = slot0 + p * step;
            const f32x4 x = *reinterpret_cast<const f32x4*>(a.parts + slot * a.part_stride + col);
            if constexpr (DQ) {
                sum += x;
            } else {
                const float share = exp2_of((a.part_stats[2 * slot] - most) * sl2);
                total = fmaf(a.part_stats[2 * slot + 1], share, total);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fmaf(x[i], share, sum[i]);
            }
        }
    }
    if constexpr (MANY) {
        lds_sum[t] = sum;
        if (col == 0) lds_total[grp] = total;
        __syncthreads();
        if (grp != 0) return;
        for (int i = 1; i < G; ++i) {
            sum += lds_sum[i * W + t];
            total += lds_total[i];
        }
    }
    if (!mine) return;
    const Place p = place_of(a, j.q_first, head, j.row0 + row);
    T* to = (DQ ? a.dq : a.out) + (p.row * a.heads + p.head) * a.dim;
    if constexpr (DQ) {
        put4<T>(to, col, a.dim, sum * a.scale);
    } else {
        put4<T>(to, col, a.dim, sum * (total == 0.0f ? 0.0f : 1.0f / total));
        if (col == 0) put_stats(a, p.row * a.heads + p.head, top, total);
    }
}

// The probabilities of the backward are the forward's: 2^(sl2 (s - top)) / total with the row's
// maximum and total as they were (the logarithm of the total would enter the exponent
// rounded at its own size).  dp of a query's keys becomes ds but for the query's share, which
// dq takes at the end.
//
// delta comes from the output as it was stored.  With few keys ds is a small difference, and the
// rounding of a 16-bit output made dq and dk err 2.2 times as much (two keys; 1.6 with nine, nothing
// to speak of from 32 on).  Where all keys of a graph are these 32, what a row's ds add up to, which
// should be nothing, shows that rounding: row_rest is added to delta before the walk.
__device__ __forceinline__ void backward_scores(const f32x4 (&s)[2], f32x4 (&dp)[2], float slope, float base, float delta) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[t][i] = exp2_of(fmaf(s[t][i], slope, -base)) * (dp[t][i] - delta);
}

__device__ __forceinline__ float row_rest(const f32x4 (&s)[2], f32x4 (&dp)[2], float slope, float base, float share, float delta) {
    backward_scores(s, dp, slope, base, delta);
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += dp[t][i];
    return lanes_sum(sum) * share;
}

// Whether an item's keys are its graph's and one wave's 32, and their outputs rounded.
template <typename T>
__device__ __forceinline__ bool few_keys(const AttnItem& it) {
    return sizeof(T) == 2 && it.part < 0 && it.keys > 0 && it.keys <= 32;
}

// <grad, out> of a wave's 16 rows, each in the four lanes that share its row: the diagonal of a
// matrix product of the rows, whose sums run in the same order as those of <grad, v>.  A row
// whose softmax is one key then has <grad, v> - delta = 0, not what is left when two
// roundings are subtracted; and what is no number stays none.
template <typename T, int DP>
__device__ __forceinline__ float row_delta_of(const RowFrags<T, DP>& out, const RowFrags<T, DP>& grad) {
    f32x4 d = f32x4(0.0f);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) d = mma<T>(out.f[c], grad.f[c], d);
    // entry i of lane l is <out of row 4 (l / 16) + i, grad of row l % 16>
    const int l = lane_id(), i = l % 4, row = l % 16;
    const float mine = i == 0 ? d[0] : i == 1 ? d[1] : i == 2 ? d[2] : d[3];
    return __shfl(mine, (row / 4) * 16 + row);
}

// Rows past an item's end are zeros in a tile, and 0 against a key that holds an infinity is NaN:
// entries from `rows` on of a lane's four leave their sums.
__device__ __forceinline__ void clear_rows(f32x4& p, f32x4& ds, int rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p[i] = i < rows ? p[i] : 0.0f;
        ds[i] = i < rows ? ds[i] : 0.0f;
    }
}

// Half values lose bits below 2^-14, where ds of keys with small probabilities lies.  A lane
// holds ds of one query (key) and the sum over keys (queries) that it enters: both are kept
// in units of a power of two, which falls as the largest ds seen so far rises (like the
// forward's running maximum), so that that one is held as 2^14 to 2^15.  Other types have
// float's range: unit 1.
constexpr float kFirstUnit = 1152921504606846976.0f;  // 2^60

template <typename T>
constexpr float kStartUnit = std::is_same_v<T, f16> ? kFirstUnit : 1.0f;

template <typename T, int N>
__device__ __forceinline__ void into_unit(f32x4 (&ds)[2], float& unit, f32x4 (&sum)[N]) {
    if constexpr (std::is_same_v<T, f16>) {
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(ds[t][i]));
        most = lanes_max(most);
        if (__any(most * unit > 32768.0f)) {
            const int e = static_cast<int>(__float_as_uint(most) >> 23);  // 127 + floor(log2(most))
            const float fresh = fminf(unit, __uint_as_float(static_cast<unsigned>(min(268 - e, 187)) << 23));
            const float change = fresh * (1.0f / unit);
#pragma unroll
            for (int n = 0; n < N; ++n) sum[n] *= change;
            unit = fresh;
        }
        ds[0] *= unit;
        ds[1] *= unit;
    }
}

// dq of a row item: like the forward, with the probabilities recomputed from its statistics.  A row's
// delta is left for the key kernel (parts of one row leave the same).  Three products to the
// forward's two, bound alike: 8 graphs of 500 to 1500 queries x 900 to 2100 keys, 8 heads
// of 64 in bfloat16, 73 us (470 TFLOP/s).
template <typename T, int DP, int RT, int WM, int FIT>
__global__ __launch_bounds__(kThreads, kWavesPerSimd<T>) void k_attention_dq(Args<T> a) {
    using S = RowShape<RT, WM>;
    constexpr int BN = S::kKeys, ST = kLdsStride<T, DP>, ND = DP / 16;
    constexpr int kTileBytes = 2 * BN * ST * static_cast<int>(sizeof(T));
    constexpr int kMergeBytes = S::kSharers > 1 ? kWaves * 16 * RT * DP * 4 : 0;
    __shared__ __align__(16) char lds[kTileBytes > kMergeBytes ? kTileBytes : kMergeBytes];
    __shared__ __align__(16) float starts[BN];
    T* kt = reinterpret_cast<T*>(lds);
    T* vt = kt + BN * ST;
    const Work w = work_of(a.items, a.num_items, a.kv_heads);
    const int l = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave, g = l / 16;
    const int row_wave = wave / S::kSharers, key_wave = wave % S::kSharers;
    const float sl2 = a.scale * kLog2e;

    RowFrags<T, DP> qf[RT], gf[RT];
    Place at[RT];
    bool real[RT];
    RowScore score[RT];
    float delta[RT], unit[RT];
    f32x4 dq[RT][ND];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = (row_wave * RT + r) * 16 + l % 16;
        real[r] = row < w.it.rows;
        at[r] = place_of(a, w.it.q_first, w.head, w.it.row0 + (real[r] ? row : 0));
        qf[r].template fetch<FIT>(a.q.data + at[r].row * a.q.row_stride + at[r].head * a.q.head_stride, a.dim);
        gf[r].template fetch<FIT>(a.grad.data + at[r].row * a.grad.row_stride + at[r].head * a.grad.head_stride, a.dim);
        RowFrags<T, DP> of;
        of.template fetch<FIT>(a.out + (at[r].row * a.heads + at[r].head) * a.dim, a.dim);
        delta[r] = row_delta_of<T, DP>(of, gf[r]);
        score[r] = RowScore(a.stats[at[r].row * a.heads + at[r].head], sl2);
        unit[r] = kStartUnit<T>;
#pragma unroll
        for (int n = 0; n < ND; ++n) dq[r][n] = f32x4(0.0f);
    }

    TileLoad<T, DP, BN> kl, vl;
    KeyBits<BN> bits;
    const auto fetch = [&](int k0) {
        const int left = w.it.keys - k0;
        const int64_t first = static_cast<int64_t>(w.it.key_first) + k0;
        const T* kp = a.k.data + first * a.k.row_stride + w.head * a.k.head_stride;
        const T* vp = a.v.data + first * a.v.row_stride + w.head * a.v.head_stride;
        kl.template fetch<FIT>([&](int row) { return kp + min(row, left - 1) * a.k.row_stride; }, a.dim);
        vl.template fetch<FIT>([&](int row) { return vp + min(row, left - 1) * a.v.row_stride; }, a.dim);
        bits.fetch(a.key_mask, first, left);
    };
    if (w.it.keys > 0) fetch(0);
    if (few_keys<T>(w.it)) {
        bits.settle();
        kl.template store<FIT>(kt, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        vl.template store<FIT>(vt, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        if (threadIdx.x < BN) starts[threadIdx.x] = bits.has(threadIdx.x) ? 0.0f : -kInf;
        __syncthreads();
        if (key_wave == 0) {  // the one that has the keys
            const f32x4 zero[2] = {f32x4(0.0f), f32x4(0.0f)};
            f32x4 start[2], s[RT][2], dp[RT][2];
            key_starts(starts, 0, start);
            keys_by_rows<T, DP, RT>(kt, 0, qf, start, s);
            keys_by_rows<T, DP, RT>(vt, 0, gf, zero, dp);
#pragma unroll
            for (int r = 0; r < RT; ++r)
                delta[r] += row_rest(s[r], dp[r], score[r].slope, score[r].base, score[r].share, delta[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
        if (real[r] && key_wave == 0 && g == 0) a.delta[at[r].row * a.heads + at[r].head] = delta[r];
    bool any = false;  // whether some key of the item is kept (the same for all waves)
    for (int k0 = 0; k0 < w.it.keys; k0 += BN) {
        bits.settle();
        any = any || !bits.none();
        __syncthreads();
        kl.template store<FIT>(kt, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        vl.template store<FIT>(vt, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        if (threadIdx.x < BN) starts[threadIdx.x] = bits.has(threadIdx.x) ? 0.0f : -kInf;
        __syncthreads();
        if (k0 + BN < w.it.keys) fetch(k0 + BN);
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const int key0 = (key_wave * S::kChunks + c) * 32;
            const f32x4 zero[2] = {f32x4(0.0f), f32x4(0.0f)};
            f32x4 start[2], s[RT][2], dp[RT][2];
            key_starts(starts, key0, start);
            keys_by_rows<T, DP, RT>(kt, key0, qf, start, s);
            keys_by_rows<T, DP, RT>(vt, key0, gf, zero, dp);
            Frag<T> ds[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                backward_scores(s[r], dp[r], score[r].slope, score[r].base, delta[r]);
                into_unit<T>(dp[r], unit[r], dq[r]);
                ds[r] = frag_of<T>(dp[r][0], dp[r][1]);
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                const Frag<T> kf = lds_frag_t<T>(kt, ST, key0, n * 16);
#pragma unroll
                for (int r = 0; r < RT; ++r) dq[r][n] = mma<T>(kf, ds[r], dq[r][n]);
            }
        }
    }

#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < ND; ++n) dq[r][n] = any ? dq[r][n] * (score[r].share / unit[r]) : f32x4(0.0f);
    const auto finish = [&](int row, Place p, int col, f32x4 sum) {
        if (w.it.part < 0) {
            put4<T>(a.dq + (p.row * a.heads + p.head) * a.dim, col, a.dim, sum * a.scale);
        } else {
            const int64_t slot = (static_cast<int64_t>(w.it.part) * a.kv_heads + w.head) * a.row_tile + row;
            if (col < a.part_stride) *reinterpret_cast<f32x4*>(a.parts + slot * a.part_stride + col) = sum;
        }
    };
    if constexpr (S::kSharers == 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
            if (real[r])
#pragma unroll
                for (int n = 0; n < ND; ++n) finish((row_wave * RT + r) * 16 + l % 16, at[r], n * 16 + g * 4, dq[r][n]);
    } else {
        constexpr int R = 16 * RT;
        float* sums = reinterpret_cast<float*>(lds);  // [kWaves][R][DP]
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < ND; ++n)
                *reinterpret_cast<f32x4*>(sums + (wave * R + r * 16 + l % 16) * DP + n * 16 + g * 4) = dq[r][n];
        __syncthreads();
        for (int u = static_cast<int>(threadIdx.x); u < w.it.rows * (DP / 4); u += kThreads) {
            const int row = u / (DP / 4), col = (u % (DP / 4)) * 4;
            const int slot = (row / R) * S::kSharers * R + row % R;  // the first sharer's
            f32x4 sum = *reinterpret_cast<const f32x4*>(sums + slot * DP + col);
#pragma unroll
            for (int v = 1; v < S::kSharers; ++v) sum += *reinterpret_cast<const f32x4*>(sums + (v * R + slot) * DP + col);
            if (col < a.dim) finish(row, place_of(a, w.it.q_first, w.head, w.it.row0 + row), col, sum);
        }
    }
}

// dk and dv of a key item: a wave keeps KT tiles of 16 keys and walks the graph's rows
// (rows down, keys across, so that a lane's probabilities are the operand of the products
// over rows).  Four products, bound by LDS reads (each of a wave's products reads its
// operand for 16 KT keys) and the exponentials: the batch above 89 us (510 TFLOP/s).
template <typename T, int DP, int KT, int FIT>
__global__ __launch_bounds__(kThreads, kWavesPerSimd<T>) void k_attention_dkv(Args<T> a) {
    constexpr int BR = 64, ST = kLdsStride<T, DP>, ND = DP / 16;
    __shared__ __align__(16) T qt[BR * ST];
    __shared__ __align__(16) T gt[BR * ST];
    __shared__ __align__(16) float row_base[BR];
    __shared__ __align__(16) float row_slope[BR];
    __shared__ __align__(16) float row_share[BR];
    __shared__ __align__(16) float row_delta[BR];
    // an item's keys are taken by key_tile / (64 KT) workgroups
    const int slices = a.key_tile / (64 * KT);
    const Work w = work_of(a.items, a.num_items, a.kv_heads * slices);
    const int head = w.head / slices;
    const int l = lane_id(), g = l / 16, wave = (w.head % slices) * kWaves + static_cast<int>(threadIdx.x) / kWave;
    const float sl2 = a.scale * kLog2e;

    RowFrags<T, DP> kf[KT], vf[KT];
    bool real[KT];
    float unit[KT];
    f32x4 start[KT];  // of the scores: -inf for a key that is not kept
    f32x4 dk[KT][ND], dv[KT][ND];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int key = (wave * KT + t) * 16 + l % 16;
        // a key past the item reads its last: a column of the scores, used by no other
        real[t] = key < w.it.keys;
        const int64_t at = static_cast<int64_t>(w.it.key_first) + min(key, w.it.keys - 1);
        const bool kept = real[t] && (a.key_mask == nullptr || a.key_mask[at] != 0);
        kf[t].template fetch<FIT>(a.k.data + at * a.k.row_stride + head * a.k.head_stride, a.dim);
        vf[t].template fetch<FIT>(a.v.data + at * a.v.row_stride + head * a.v.head_stride, a.dim);
        if (!kept) {
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) kf[t].f[c] = vf[t].f[c] = Frag<T>(static_cast<T>(0.0f));
        }
        start[t] = f32x4(kept ? 0.0f : -kInf);
#pragma unroll
        for (int n = 0; n < ND; ++n) dk[t][n] = dv[t][n] = f32x4(0.0f);
        unit[t] = kStartUnit<T>;
    }

    TileLoad<T, DP, BR> ql, gl;
    RowScore score_in;
    float delta_in = 0.0f;
    const auto fetch = [&](int r0) {
        const int left = w.it.rows - r0;
        const auto place = [&](int row) { return place_of(a, w.it.q_first, head, w.it.row0 + r0 + min(row, left - 1)); };
        ql.template fetch<FIT>([&](int row) {
            const Place p = place(row);
            return a.q.data + p.row * a.q.row_stride + p.head * a.q.head_stride;
        }, a.dim);
        gl.template fetch<FIT>([&](int row) {
            const Place p = place(row);
            return a.grad.data + p.row * a.grad.row_stride + p.head * a.grad.head_stride;
        }, a.dim);
        const int row = static_cast<int>(threadIdx.x) % BR;
        const Place p = place(row);
        score_in = RowScore(a.stats[p.row * a.heads + p.head], sl2);
        delta_in = a.delta[p.row * a.heads + p.head];
    };
    if (w.it.rows > 0) fetch(0);
    for (int r0 = 0; r0 < w.it.rows; r0 += BR) {
        __syncthreads();
        const int left = w.it.rows - r0;
        ql.template store<FIT>(qt, a.dim, left >= BR, [&](int row) { return row < left; });
        gl.template store<FIT>(gt, a.dim, left >= BR, [&](int row) { return row < left; });
        if (threadIdx.x < BR) {
            row_slope[threadIdx.x] = score_in.slope;
            row_base[threadIdx.x] = score_in.base;
            row_share[threadIdx.x] = score_in.share;
            row_delta[threadIdx.x] = delta_in;
        }
        __syncthreads();
        if (left > BR) fetch(r0 + BR);
#pragma unroll
        for (int c = 0; c < BR / 32; ++c) {
            if (c * 32 >= left) break;
            f32x4 s[KT][2], dp[KT][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = c * 32 + h * 16;
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    s[t][h] = start[t];
                    dp[t][h] = f32x4(0.0f);
                }
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) {
                    const Frag<T> qr = lds_frag<T>(qt, ST, row + l % 16, i * 32 + g * 8);
                    const Frag<T> gr = lds_frag<T>(gt, ST, row + l % 16, i * 32 + g * 8);
#pragma unroll
                    for (int t = 0; t < KT; ++t) {
                        s[t][h] = mma<T>(qr, kf[t].f[i], s[t][h]);
                        dp[t][h] = mma<T>(gr, vf[t].f[i], dp[t][h]);
                    }
                }
            }
            Frag<T> pf[KT], dsf[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 slope = *reinterpret_cast<const f32x4*>(row_slope + c * 32 + h * 16 + g * 4);
                    const f32x4 base = *reinterpret_cast<const f32x4*>(row_base + c * 32 + h * 16 + g * 4);
                    const f32x4 share = *reinterpret_cast<const f32x4*>(row_share + c * 32 + h * 16 + g * 4);
                    const f32x4 delta = *reinterpret_cast<const f32x4*>(row_delta + c * 32 + h * 16 + g * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = exp2_of(fmaf(s[t][h][i], slope[i], -base[i])) * share[i];
                        s[t][h][i] = p;
                        dp[t][h][i] = p * (dp[t][h][i] - delta[i]);
                    }
                }
                if (left < c * 32 + 32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) clear_rows(s[t][h], dp[t][h], left - (c * 32 + h * 16 + g * 4));
                }
                pf[t] = frag_of<T>(s[t][0] * kProbabilityUnit<T>, s[t][1] * kProbabilityUnit<T>);
                into_unit<T>(dp[t], unit[t], dk[t]);
                dsf[t] = frag_of<T>(dp[t][0], dp[t][1]);
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                const Frag<T> gf = lds_frag_t<T>(gt, ST, c * 32, n * 16);
                const Frag<T> qf = lds_frag_t<T>(qt, ST, c * 32, n * 16);
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    dv[t][n] = mma<T>(gf, pf[t], dv[t][n]);
                    dk[t][n] = mma<T>(qf, dsf[t], dk[t][n]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        if (!real[t]) continue;
        const int key = (wave * KT + t) * 16 + l % 16;
        const int64_t at = (static_cast<int64_t>(w.it.key_first) + key) * a.kv_heads + head;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            const int col = n * 16 + g * 4;
            dk[t][n] *= 1.0f / unit[t];
            if (start[t][0] != 0.0f) dk[t][n] = dv[t][n] = f32x4(0.0f);  // whatever an infinite query made of it
            if (w.it.part < 0) {
                put4<T>(a.dk + at * a.dim, col, a.dim, dk[t][n] * a.scale);
                put4<T>(a.dv + at * a.dim, col, a.dim, dv[t][n] * (1.0f / kProbabilityUnit<T>));
            } else {
                float* to = a.parts + ((static_cast<int64_t>(w.it.part) * a.kv_heads + head) * a.key_tile + key) *
                                          (2 * a.part_stride) + col;
                if (col < a.part_stride) {
                    *reinterpret_cast<f32x4*>(to) = dk[t][n];
                    *reinterpret_cast<f32x4*>(to + a.part_stride) = dv[t][n] * (1.0f / kProbabilityUnit<T>);
                }
            }
        }
    }
}

// Joins the parts of a key item: a thread group per key, its dk and dv side by side.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void k_attention_dkv_join(Args<T> a) {
    constexpr int W = DP / 4, G = kThreads / (2 * W);
    const int t = static_cast<int>(threadIdx.x), per = a.key_tile / G;
    const AttnJoin j = a.joins[blockIdx.x / per];
    const int key = static_cast<int>(blockIdx.x % per) * G + t / (2 * W), head = static_cast<int>(blockIdx.y);
    const int which = t / W % 2, col = (t % W) * 4;
    if (key >= j.keys || col >= a.part_stride) return;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * a.key_tile * 2 * a.part_stride;
    const float* part = a.parts + (((static_cast<int64_t>(j.part0) * a.kv_heads + head) * a.key_tile + key) * 2 + which) *
                                      a.part_stride + col;
    f32x4 sum = f32x4(0.0f);
#pragma unroll 4
    for (int p = 0; p < j.parts; ++p) sum += *reinterpret_cast<const f32x4*>(part + p * step);
    const int64_t at = ((static_cast<int64_t>(j.key_first) + key) * a.kv_heads + head) * a.dim;
    if (which == 0)
        put4<T>(a.dk + at, col, a.dim, sum * a.scale);
    else
        put4<T>(a.dv + at, col, a.dim, sum);
}

// The whole backward of a batch whose graphs have at most 32 rows: a workgroup has all of a
// graph's rows, so a key tile's dk and dv are complete when it has been walked, dq when
// all have, and keys and values are read once.  A wave takes 32 keys of a tile.  dq sums over
// keys and wants them down (as in the forward), dk and dv over rows and want those down: the
// scores are computed both ways, from the same fragments with the operands exchanged, and
// their exponentials twice.  Bound by latency, then by the reads and writes
// (keys, values and their gradients once each): 2048 graphs of 64 to 512 keys, up to 32
// queries, 4 heads of 32 in bfloat16 214 us (291 before the items were dealt by length, then
// 318 for the two kernels of longer rows, when this one took 192).
template <typename T, int DP>
struct FewRows {
    static constexpr int kKeys = 128, kStride = kLdsStride<T, DP>;
    // float rows of 128 values leave LDS for 16 rows
    static constexpr int kRows = sizeof(T) * DP < 512 ? 32 : 16;
    __align__(16) T k[kKeys * kStride];
    __align__(16) T v[kKeys * kStride];
    __align__(16) T q[kRows * kStride];
    __align__(16) T g[kRows * kStride];
    __align__(16) float starts[kKeys];
    __align__(16) float slope[32];
    __align__(16) float base[32];
    __align__(16) float share[32];
    __align__(16) float delta[32];
};

template <typename T, int DP, int RT, int FIT>
__device__ __forceinline__ void few_rows_backward(const Args<T>& a, const Work& w, FewRows<T, DP>& m) {
    using M = FewRows<T, DP>;
    constexpr int BN = M::kKeys, ST = M::kStride, ND = DP / 16;
    const int l = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave, g = l / 16;
    const float sl2 = a.scale * kLog2e;

    TileLoad<T, DP, BN> kl, vl;
    KeyBits<BN> bits;
    const auto fetch = [&](int k0) {
        const int left = w.it.keys - k0;
        const int64_t first = static_cast<int64_t>(w.it.key_first) + k0;
        const T* kp = a.k.data + first * a.k.row_stride + w.head * a.k.head_stride;
        const T* vp = a.v.data + first * a.v.row_stride + w.head * a.v.head_stride;
        kl.template fetch<FIT>([&](int row) { return kp + min(row, left - 1) * a.k.row_stride; }, a.dim);
        vl.template fetch<FIT>([&](int row) { return vp + min(row, left - 1) * a.v.row_stride; }, a.dim);
        bits.fetch(a.key_mask, first, left);
    };
    if (w.it.keys > 0) fetch(0);

    RowFrags<T, DP> qf[RT], gf[RT];
    Place at[RT];
    bool real[RT];
    float unit[RT];
    f32x4 dq[RT][ND];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = r * 16 + l % 16;
        real[r] = row < w.it.rows;
        at[r] = place_of(a, w.it.q_first, w.head, w.it.row0 + (real[r] ? row : 0));
        qf[r].template fetch<FIT>(a.q.data + at[r].row * a.q.row_stride + at[r].head * a.q.head_stride, a.dim);
        gf[r].template fetch<FIT>(a.grad.data + at[r].row * a.grad.row_stride + at[r].head * a.grad.head_stride, a.dim);
        RowFrags<T, DP> of;
        of.template fetch<FIT>(a.out + (at[r].row * a.heads + at[r].head) * a.dim, a.dim);
        const float delta = row_delta_of<T, DP>(of, gf[r]);
        const RowScore score(a.stats[at[r].row * a.heads + at[r].head], sl2);
        if (!real[r]) {  // a sum over rows must not see it
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) qf[r].f[c] = gf[r].f[c] = Frag<T>(static_cast<T>(0.0f));
        }
        unit[r] = kStartUnit<T>;
#pragma unroll
        for (int n = 0; n < ND; ++n) dq[r][n] = f32x4(0.0f);
        if (wave == 0) {
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                lds_put<T>(m.q + row * ST + c * 32 + g * 8, qf[r].f[c]);
                lds_put<T>(m.g + row * ST + c * 32 + g * 8, gf[r].f[c]);
            }
            if (g == 0) {
                m.slope[row] = score.slope;
                m.base[row] = score.base;
                m.share[row] = score.share;
                m.delta[row] = delta;
            }
        }
    }

    if (few_keys<T>(w.it)) {
        bits.settle();
        kl.template store<FIT>(m.k, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        vl.template store<FIT>(m.v, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        if (threadIdx.x < BN) m.starts[threadIdx.x] = bits.has(threadIdx.x) ? 0.0f : -kInf;
        __syncthreads();
        if (wave == 0) {  // the one that has the keys, and wrote the rows
            const f32x4 zero[2] = {f32x4(0.0f), f32x4(0.0f)};
            f32x4 start[2], s[RT][2], dp[RT][2];
            key_starts(m.starts, 0, start);
            keys_by_rows<T, DP, RT>(m.k, 0, qf, start, s);
            keys_by_rows<T, DP, RT>(m.v, 0, gf, zero, dp);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int row = r * 16 + l % 16;
                const float rest = row_rest(s[r], dp[r], m.slope[row], m.base[row], m.share[row], m.delta[row]);
                if (g == 0) m.delta[row] += rest;
            }
        }
    }
    bool any = false;  // whether some key of the item is kept (the same for all waves)
    for (int k0 = 0; k0 < w.it.keys; k0 += BN) {
        bits.settle();
        any = any || !bits.none();
        __syncthreads();
        kl.template store<FIT>(m.k, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        vl.template store<FIT>(m.v, a.dim, bits.all(), [&](int row) { return bits.has(row); });
        if (threadIdx.x < BN) m.starts[threadIdx.x] = bits.has(threadIdx.x) ? 0.0f : -kInf;
        __syncthreads();
        if (k0 + BN < w.it.keys) fetch(k0 + BN);
        const int key0 = wave * 32;
        if (k0 + key0 >= w.it.keys) continue;

        // keys down, for dq
        f32x4 start[2], s[RT][2], dp[RT][2];
        const f32x4 zero[2] = {f32x4(0.0f), f32x4(0.0f)};
        key_starts(m.starts, key0, start);
        keys_by_rows<T, DP, RT>(m.k, key0, qf, start, s);
        keys_by_rows<T, DP, RT>(m.v, key0, gf, zero, dp);
        Frag<T> ds[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = r * 16 + l % 16;  // its statistics from LDS: in registers they spilled others
            backward_scores(s[r], dp[r], m.slope[row], m.base[row], m.delta[row]);
            into_unit<T>(dp[r], unit[r], dq[r]);
            ds[r] = frag_of<T>(dp[r][0], dp[r][1]);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            const Frag<T> kf = lds_frag_t<T>(m.k, ST, key0, n * 16);
#pragma unroll
            for (int r = 0; r < RT; ++r) dq[r][n] = mma<T>(kf, ds[r], dq[r][n]);
        }
        // rows down, for dk and dv
        Frag<T> pf[2], dsf[2];
        float unit2[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 s2[RT], dp2[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                s2[r] = f32x4(m.starts[key0 + 16 * t + l % 16]);
                dp2[r] = f32x4(0.0f);
            }
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                const Frag<T> k = lds_frag<T>(m.k, ST, key0 + 16 * t + l % 16, c * 32 + g * 8);
                const Frag<T> v = lds_frag<T>(m.v, ST, key0 + 16 * t + l % 16, c * 32 + g * 8);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    s2[r] = mma<T>(qf[r].f[c], k, s2[r]);
                    dp2[r] = mma<T>(gf[r].f[c], v, dp2[r]);
                }
            }
            f32x4 pr[2] = {f32x4(0.0f), f32x4(0.0f)}, dr[2] = {f32x4(0.0f), f32x4(0.0f)}, none[1] = {f32x4(0.0f)};
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const f32x4 row_slope = *reinterpret_cast<const f32x4*>(m.slope + r * 16 + g * 4);
                const f32x4 row_base = *reinterpret_cast<const f32x4*>(m.base + r * 16 + g * 4);
                const f32x4 row_share = *reinterpret_cast<const f32x4*>(m.share + r * 16 + g * 4);
                const f32x4 row_delta = *reinterpret_cast<const f32x4*>(m.delta + r * 16 + g * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    pr[r][i] = exp2_of(fmaf(s2[r][i], row_slope[i], -row_base[i])) * row_share[i];
                    dr[r][i] = pr[r][i] * (dp2[r][i] - row_delta[i]);
                }
                if (w.it.rows < 16 * RT) clear_rows(pr[r], dr[r], w.it.rows - (r * 16 + g * 4));
            }
            pf[t] = frag_of<T>(pr[0] * kProbabilityUnit<T>, pr[1] * kProbabilityUnit<T>);
            unit2[t] = kStartUnit<T>;
            into_unit<T>(dr, unit2[t], none);
            dsf[t] = frag_of<T>(dr[0], dr[1]);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            const Frag<T> gt = rows_frag_t<T, RT>(m.g, ST, n * 16);
            const Frag<T> qt = rows_frag_t<T, RT>(m.q, ST, n * 16);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 dv = mma<T>(gt, pf[t], f32x4(0.0f));
                f32x4 dk = mma<T>(qt, dsf[t], f32x4(0.0f));
                // a key that is not kept gets 0, whatever an infinite query made of it
                if (m.starts[key0 + 16 * t + l % 16] != 0.0f) dk = dv = f32x4(0.0f);
                const int key = k0 + key0 + 16 * t + l % 16;
                if (key < w.it.keys) {
                    const int64_t to = ((static_cast<int64_t>(w.it.key_first) + key) * a.kv_heads + w.head) * a.dim;
                    put4<T>(a.dk + to, n * 16 + g * 4, a.dim, dk * (a.scale / unit2[t]));
                    put4<T>(a.dv + to, n * 16 + g * 4, a.dim, dv * (1.0f / kProbabilityUnit<T>));
                }
            }
        }
    }

    // the waves' shares of dq meet in LDS
    constexpr int R = 16 * RT;
    static_assert(sizeof(m.k) + sizeof(m.v) >= sizeof(float) * kWaves * R * DP, "room for the shares");
    float* sums = reinterpret_cast<float*>(m.k);  // [kWaves][R][DP]
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < ND; ++n)
            *reinterpret_cast<f32x4*>(sums + (wave * R + r * 16 + l % 16) * DP + n * 16 + g * 4) =
                any ? dq[r][n] * (m.share[r * 16 + l % 16] / unit[r]) : f32x4(0.0f);
    __syncthreads();
    for (int u = static_cast<int>(threadIdx.x); u < w.it.rows * (DP / 4); u += kThreads) {
        const int row = u / (DP / 4), col = (u % (DP / 4)) * 4;
        f32x4 sum = *reinterpret_cast<const f32x4*>(sums + row * DP + col);
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += *reinterpret_cast<const f32x4*>(sums + (v * R + row) * DP + col);
        if (w.it.part < 0) {
            const Place p = place_of(a, w.it.q_first, w.head, w.it.row0 + row);
            put4<T>(a.dq + (p.row * a.heads + p.head) * a.dim, col, a.dim, sum * a.scale);
        } else if (col < a.part_stride) {
            const int64_t slot = (static_cast<int64_t>(w.it.part) * a.kv_heads + w.head) * a.row_tile + row;
            *reinterpret_cast<f32x4*>(a.parts + slot * a.part_stride + col) = sum;
        }
    }
}

// Waves to a SIMD that the kernel's registers are held to.
template <typename T, int DP>
constexpr int kFewRowsWaves = sizeof(T) == 2 ? (DP == 32 ? 3 : DP == 64 ? 2 : 1) : (DP == 32 ? 2 : 1);

// Items of graphs without queries have no rows: their keys get zeros.
template <typename T, int DP, int FIT>
__global__ __launch_bounds__(kThreads, (kFewRowsWaves<T, DP>)) void k_attention_few_rows_backward(Args<T> a) {
    __shared__ FewRows<T, DP> m;
    const Work w = work_of(a.items, a.num_items, a.kv_heads);
    if (w.it.rows == 0) {
        for (int u = static_cast<int>(threadIdx.x); u < w.it.keys * (DP / 4); u += kThreads) {
            const int col = (u % (DP / 4)) * 4;
            const int64_t to = ((static_cast<int64_t>(w.it.key_first) + u / (DP / 4)) * a.kv_heads + w.head) * a.dim;
            put4<T>(a.dk + to, col, a.dim, f32x4(0.0f));
            put4<T>(a.dv + to, col, a.dim, f32x4(0.0f));
        }
        return;
    }
    if constexpr (FewRows<T, DP>::kRows == 32) {
        if (w.it.rows > 16) {
            few_rows_backward<T, DP, 2, FIT>(a, w, m);
            return;
        }
    }
    few_rows_backward<T, DP, 1, FIT>(a, w, m);
}

// The statistics of rows of which only the logarithm of the total was kept: those of a single
// score of that size.
__global__ __launch_bounds__(kThreads) void k_attention_stats(const float* lse, int64_t rows, float scale, RowStats* stats) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; at < rows; at += step) {
        const float x = lse[at];
        stats[at] = {x == -kInf ? 0.0f : x / scale, x == -kInf ? 0.0f : 1.0f};
    }
}

// ---- launches -----------------------------------------------------------------------

template <typename T>
Args<T> args_of(const relm_mp_attention_plan& p, const AttnOperands& o) {
    Args<T> a{};
    a.q = rows_of<T>(o.q);
    a.k = rows_of<T>(o.k);
    a.v = rows_of<T>(o.v);
    a.grad = rows_of<T>(o.grad);
    a.key_mask = o.key_mask;
    a.dim = static_cast<int>(o.head_dim);
    a.heads = p.heads;
    a.kv_heads = p.kv_heads;
    a.group = p.heads / p.kv_heads;
    a.row_tile = p.row_tile;
    a.key_tile = p.key_tile;
    a.scale = o.scale;
    a.num_items = p.num_items;
    a.items = plan_items(p);
    a.joins = plan_joins(p);
    a.out = static_cast<T*>(o.out);
    a.lse = o.lse;
    a.stats = o.stats;
    a.delta = o.delta;
    a.dq = static_cast<T*>(o.dq);
    a.dk = static_cast<T*>(o.dk);
    a.dv = static_cast<T*>(o.dv);
    a.parts = o.parts;
    a.part_stride = static_cast<int>(attention_part_stride(o.head_dim));
    a.part_stats = o.parts + attention_part_rows(p) * a.part_stride;
    return a;
}

// f with the padded head size (32, 64 or 128), FIT, and the rows' shape of the plan.
template <typename F>
void with_dim(int64_t dim, F&& f) {
    const auto with = [&](auto dp) {
        if (dim % 8 == 0)
            f(dp, std::integral_constant<int, kWhole>{});
        else if (decltype(dp)::value > 32 || dim > 8)
            f(dp, std::integral_constant<int, kCut>{});
        else if constexpr (decltype(dp)::value == 32)
            f(dp, std::integral_constant<int, kShort>{});
    };
    if (dim <= 32)
        with(std::integral_constant<int, 32>{});
    else if (dim <= 64)
        with(std::integral_constant<int, 64>{});
    else
        with(std::integral_constant<int, 128>{});
}
template <typename T, int DP, typename F>
void with_rows(int row_tile, F&& f) {
    using std::integral_constant;
    // rows of 128 values: tiles of 128 keys and of 32 rows to a wave leave it too few
    // registers
    constexpr bool kLarge = DP == 128;
    switch (row_tile) {
        case 16: f(integral_constant<int, 1>{}, integral_constant<int, 1>{}); break;
        case 32: f(integral_constant<int, kLarge ? 1 : 2>{}, integral_constant<int, kLarge ? 2 : 1>{}); break;
        case 64: f(integral_constant<int, 1>{}, integral_constant<int, 4>{}); break;
        default: f(integral_constant<int, 2>{}, integral_constant<int, 4>{}); break;
    }
}

// Rows of up to kFewParts parts on average are joined a thread group to a row; with more, a
// workgroup to a row.  4 heads of 64 in bfloat16, forward, us: 60 queries x 3000 keys in 6 parts
// 17.0 and 15.8, x 5000 in 10 18.4 and 15.6; 128 x 9000 in 18 25.0 and 20.5; 500 x 9000 in 18 29.7 and
// 28.1.  (At 5 to 6 parts the second form is already a microsecond faster.)
constexpr int kFewParts = 8;

template <typename T, int DP, bool DQ>
void join_rows(const relm_mp_attention_plan& p, const Args<T>& a, hipStream_t st) {
    if (p.num_joins == 0) return;
    if (p.num_parts > kFewParts * p.num_joins || p.row_tile < kJoinGroups<DP>)
        hipLaunchKernelGGL((k_attention_join<T, DP, true, DQ>),
                           dim3(static_cast<unsigned>(p.num_joins) * p.row_tile, p.kv_heads), dim3(kThreads), 0, st, a);
    else
        hipLaunchKernelGGL((k_attention_join<T, DP, false, DQ>),
                           dim3(static_cast<unsigned>(p.num_joins) * (p.row_tile / kJoinGroups<DP>), p.kv_heads),
                           dim3(kThreads), 0, st, a);
}

template <typename T>
hipError_t forward(const relm_mp_attention_plan& p, const AttnOperands& o, hipStream_t st) {
    const Args<T> a = args_of<T>(p, o);
    if (p.num_items == 0) return hipSuccess;
    with_dim(o.head_dim, [&](auto dp, auto whole) {
        constexpr int DP = decltype(dp)::value;
        constexpr int W = decltype(whole)::value;
        with_rows<T, DP>(p.row_tile, [&](auto rt, auto wm) {
            hipLaunchKernelGGL((k_attention<T, DP, decltype(rt)::value, decltype(wm)::value, W>),
                               dim3(static_cast<unsigned>(p.num_items) * p.kv_heads), dim3(kThreads), 0, st, a);
        });
        join_rows<T, DP, false>(p, a, st);
    });
    return hipGetLastError();
}

template <typename T>
hipError_t backward(const relm_mp_attention_plan& p, const AttnOperands& o, hipStream_t st) {
    Args<T> a = args_of<T>(p, o);
    with_dim(o.head_dim, [&](auto dp, auto whole) {
        constexpr int DP = decltype(dp)::value;
        constexpr int W = decltype(whole)::value;
        if (p.row_tile <= FewRows<T, DP>::kRows) {
            a.num_items = p.num_items + p.num_idle_items;
            if (a.num_items > 0)
                hipLaunchKernelGGL((k_attention_few_rows_backward<T, DP, W>),
                                   dim3(static_cast<unsigned>(a.num_items) * p.kv_heads), dim3(kThreads), 0, st, a);
            join_rows<T, DP, true>(p, a, st);
            return;
        }
        if (p.num_items > 0)
            with_rows<T, DP>(p.row_tile, [&](auto rt, auto wm) {
                hipLaunchKernelGGL((k_attention_dq<T, DP, decltype(rt)::value, decltype(wm)::value, W>),
                                   dim3(static_cast<unsigned>(p.num_items) * p.kv_heads), dim3(kThreads), 0, st, a);
            });
        join_rows<T, DP, true>(p, a, st);
        if (p.num_key_items > 0) {
            Args<T> b = a;
            b.items = plan_key_items(p);
            b.joins = plan_key_joins(p);
            b.num_items = p.num_key_items;
            // two tiles of keys to a wave halve its reads of the rows; rows of 128 values
            // leave no registers for the second
            constexpr int KT = DP < 128 ? 2 : 1;
            const unsigned wgs = static_cast<unsigned>(p.num_key_items) * p.kv_heads;
            if (p.key_tile == 64 * KT)
                hipLaunchKernelGGL((k_attention_dkv<T, DP, KT, W>), dim3(wgs), dim3(kThreads), 0, st, b);
            else
                hipLaunchKernelGGL((k_attention_dkv<T, DP, 1, W>), dim3(wgs * (p.key_tile / 64)), dim3(kThreads), 0, st, b);
            if (p.num_key_joins > 0)
                hipLaunchKernelGGL((k_attention_dkv_join<T, DP>),
                                   dim3(static_cast<unsigned>(p.num_key_joins) * (p.key_tile / (kThreads / (DP / 2))), p.kv_heads),
                                   dim3(kThreads), 0, st, b);
        }
    });
    return hipGetLastError();
}

}  // namespace

hipError_t launch_cross_attention(int dtype, const relm_mp_attention_plan& p, const AttnOperands& o, hipStream_t st) {
    hipError_t e = hipErrorInvalidValue;
    with_value_type(dtype, [&](auto t) { e = forward<decltype(t)>(p, o, st); });
    return e;
}

hipError_t launch_attention_stats(const relm_mp_attention_plan& p, const float* lse, float scale, RowStats* stats, hipStream_t st) {
    const int64_t rows = p.q_rows * p.heads;
    const int64_t blocks = std::min<int64_t>((rows + kThreads - 1) / kThreads, 256 * 32);
    if (rows > 0)
        hipLaunchKernelGGL(k_attention_stats, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, lse, rows, scale, stats);
    return hipGetLastError();
}

hipError_t launch_cross_attention_backward(int dtype, const relm_mp_attention_plan& p, const AttnOperands& o,
                                           hipStream_t st) {
    hipError_t e = hipErrorInvalidValue;
    with_value_type(dtype, [&](auto t) { e = backward<decltype(t)>(p, o, st); });
    return e;
}

}  // namespace relm_mp
