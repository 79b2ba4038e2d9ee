// Root-mean-square norm of a residual stream, fused with the residual's addition:
//
//   h = x + r,   y = h * rstd * w,   rstd = 1 / sqrt(mean(h^2) + eps)   per row,
//
// with y in the values' type or in 8 bits (e4m3) under a scale per row, and its
// backward
//
//   dx = dr = rstd * (dn - n * mean(dn * n)) + dh,   n = h * rstd,  dn = dy * w,
//   dw = sum over the rows of dy * n.
//
// Sums, statistics and h inside a pass are float; h is rounded only as it is
// stored, and the norm is that of the unrounded sum.  The backward reads the stored h (a
// second stream of x and r would be a quarter more bytes): of 16-bit values n is then off
// by one rounding, and dw errs by two in the place of one.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device_utils.h"
#include "internal.h"
#include "value_types.h"

namespace relm_mp {

namespace {

constexpr int kThreads = 256;
constexpr float kFp8Max = 448.0f;  // largest finite e4m3 value

// A row belongs to a group of L lanes (part of a wave up to 64, else the
// workgroup); each lane holds NV units of V neighbouring values, V a divisor of the
// width, unit i of lane l at column (i * L + l) * V, so a group reads L * V values side
// by side.  Lanes past the row read its first unit as zeros: a load under a branch
// would wait for the one before it.  NV = 0: rows of any width, walked in units that
// are read again for the second pass (from the caches: the first pass has just read
// them).
template <typename T, int V>
__device__ __forceinline__ FloatVec<V> load_unit(const T* __restrict__ row, int64_t col, int64_t width) {
    const bool live = col < width;
    const ValueVec<T, V> v = *reinterpret_cast<const ValueVec<T, V>*>(row + (live ? col : 0));
    FloatVec<V> x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = live ? static_cast<float>(v[i]) : 0.0f;
    return x;
}

template <typename T, int V>
__device__ __forceinline__ void store_unit(T* __restrict__ row, int64_t col, int64_t width, FloatVec<V> x) {
    ValueVec<T, V> v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = round_to<T>(x[i]);
    if (col < width) *reinterpret_cast<ValueVec<T, V>*>(row + col) = v;
}

template <int L>
constexpr int kGroups = kThreads / L;

template <int L>
__device__ __forceinline__ float group_sum(float v, float* lds) {
#pragma unroll
    for (int o = (L < kWave ? L : kWave) / 2; o > 0; o /= 2) v += __shfl_xor(v, o);
    if constexpr (L > kWave) {
        if (lane_id() == 0) lds[threadIdx.x / kWave] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int i = 1; i < L / kWave; ++i) v += lds[i];
        __syncthreads();
    }
    return v;
}

// The larger of two magnitudes; NaN wins, so that a row with one has a NaN scale.
__device__ __forceinline__ float max_or_nan(float a, float b) { return a > b || a != a ? a : b; }

template <int L>
__device__ __forceinline__ float group_max(float v, float* lds) {
#pragma unroll
    for (int o = (L < kWave ? L : kWave) / 2; o > 0; o /= 2) v = max_or_nan(v, __shfl_xor(v, o));
    if constexpr (L > kWave) {
        if (lane_id() == 0) lds[threadIdx.x / kWave] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int i = 1; i < L / kWave; ++i) v = max_or_nan(v, lds[i]);
        __syncthreads();
    }
    return v;
}

template <int V>
__device__ __forceinline__ float square_sum(FloatVec<V> v, float sum) {
#pragma unroll
    for (int j = 0; j < V; ++j) sum = fmaf(v[j], v[j], sum);
    return sum;
}

// V values rounded to e4m3 (nearest even; the row's scale keeps them within range).  A
// row's bytes start anywhere: units of 4 and 8 are stored whole where they lie on dwords.
template <int V>
__device__ __forceinline__ void store_fp8(uint8_t* row, int64_t col, int64_t width, FloatVec<V> v) {
    if (col >= width) return;
    if constexpr (V % 4 == 0) {
        uint32_t word[V / 4];
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j], v[4 * j + 1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2], v[4 * j + 3], w, true);
            word[j] = static_cast<uint32_t>(w);
        }
        if (((reinterpret_cast<uintptr_t>(row) + col) & 3) == 0) {
#pragma unroll
            for (int j = 0; j < V / 4; ++j) reinterpret_cast<uint32_t*>(row + col)[j] = word[j];
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        row[col + j] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[j], 0.0f, 0, false) & 0xff);
}

struct NormArgs {
    const void* x;
    const void* r;  // may be NULL
    const void* w;
    void* y;        // values, or e4m3 bytes
    void* h;        // may be NULL
    float* scale;   // 8-bit output: per row
    float* rstd;    // may be NULL
    int64_t rows;
    int64_t width;
    float eps;
};

// Bound by memory: x, r, y and h move once (the weight stays in registers over
// the rows of a group).  589,825 x 128 floats 222 us (5.4 TB/s, as a large copy); 3,001 x
// 1,280 bfloat16 to e4m3 9 us, of which the bytes take 5; 200 x 128 floats 3 us.
template <typename T, int V, int NV, int L, bool FP8, bool RESIDUAL>
__global__ __launch_bounds__(kThreads) void k_norm(NormArgs a) {
    __shared__ float lds[kThreads / kWave];
    constexpr int NR = NV == 0 ? 1 : NV;
    const int lane = static_cast<int>(threadIdx.x) % L;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups<L> + threadIdx.x / L;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups<L>;
    const T* w = static_cast<const T*>(a.w);
    const int64_t units = NV == 0 ? (a.width + V * L - 1) / (V * L) : NV;
    FloatVec<V> wv[NR];
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) wv[i] = load_unit<T, V>(w, static_cast<int64_t>(i * L + lane) * V, a.width);
    }
    // groups of a workgroup walk the same number of rows: the barriers inside the
    // sums of whole-workgroup groups (L == kThreads: one group) stay together
    for (int64_t row = group; row < a.rows; row += step) {
        const T* x = static_cast<const T*>(a.x) + row * a.width;
        const T* r = static_cast<const T*>(a.r) + (RESIDUAL ? row * a.width : 0);
        T* h = a.h != nullptr ? static_cast<T*>(a.h) + row * a.width : nullptr;
        FloatVec<V> v[NR];
        float sum = 0.0f;
        auto take = [&](int64_t col) {
            FloatVec<V> s = load_unit<T, V>(x, col, a.width);
            if constexpr (RESIDUAL) s += load_unit<T, V>(r, col, a.width);
            return s;
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = take(static_cast<int64_t>(i * L + lane) * V);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (h != nullptr) store_unit<T, V>(h, static_cast<int64_t>(i * L + lane) * V, a.width, v[i]);
                sum = square_sum<V>(v[i], sum);
            }
        } else {
            for (int64_t i = 0; i < units; ++i) {
                const int64_t col = (i * L + lane) * V;
                const FloatVec<V> s = take(col);
                if (h != nullptr) store_unit<T, V>(h, col, a.width, s);
                sum = square_sum<V>(s, sum);
            }
        }
        sum = group_sum<L>(sum, lds);
        const float rstd = 1.0f / sqrtf(sum / static_cast<float>(a.width) + a.eps);
        if (a.rstd != nullptr && lane == 0) a.rstd[row] = rstd;
        auto result = [&](int64_t i) {  // unit i of y
            const int64_t col = (i * L + lane) * V;
            if constexpr (NV > 0) return v[i] * rstd * wv[i];
            return take(col) * rstd * load_unit<T, V>(w, col, a.width);
        };
        if constexpr (!FP8) {
            T* y = static_cast<T*>(a.y) + row * a.width;
            if constexpr (NV > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    store_unit<T, V>(y, static_cast<int64_t>(i * L + lane) * V, a.width, result(i));
            } else {
                for (int64_t i = 0; i < units; ++i) store_unit<T, V>(y, (i * L + lane) * V, a.width, result(i));
            }
        } else {
            uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.width;
            float most = 0.0f;
            auto magnitude = [&](FloatVec<V> u) {
#pragma unroll
                for (int j = 0; j < V; ++j) most = max_or_nan(most, fabsf(u[j]));
            };
            if constexpr (NV > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    v[i] = result(i);
                    magnitude(v[i]);
                }
            } else {
                for (int64_t i = 0; i < units; ++i) magnitude(result(i));
            }
            most = group_max<L>(most, lds);
            float scale = most / kFp8Max;
            if (scale == 0.0f) scale = 1.0f;  // zeros, or too small to have a scale
            if (lane == 0) a.scale[row] = scale;
            // a scale below the smallest normal float may round up to 9% off: the
            // quotient is held to the type's range
            auto scaled = [&](FloatVec<V> u) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float q = u[j] / scale;
                    u[j] = q > kFp8Max ? kFp8Max : q < -kFp8Max ? -kFp8Max : q;
                }
                return u;
            };
            if constexpr (NV > 0) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    store_fp8<V>(y, static_cast<int64_t>(i * L + lane) * V, a.width, scaled(v[i]));
            } else {
                for (int64_t i = 0; i < units; ++i)
                    store_fp8<V>(y, (i * L + lane) * V, a.width, scaled(result(i)));
            }
        }
    }
}

struct NormBackwardArgs {
    const void* dy;
    const void* dh;  // may be NULL
    const void* h;
    const void* w;
    const float* rstd;
    void* dx;
    float* partial;  // [blocks][width] sums of dy * n (NV > 0)
    int64_t rows;
    int64_t width;
};

// Bound by memory: dy, dh, h and dx move once.  A lane adds its columns' share of
// the weight gradient over the rows of its group in registers; the groups of a
// workgroup add theirs through LDS in group order, the workgroups in
// k_norm_fold: no atomics, the same result every time.  589,825 x 128 floats 230 us
// (5.3 TB/s).
template <typename T, int V, int NV, int L, bool DH>
__global__ __launch_bounds__(kThreads) void k_norm_backward(NormBackwardArgs a) {
    __shared__ float lds[kThreads / kWave];
    constexpr int NR = NV == 0 ? 1 : NV;
    const int lane = static_cast<int>(threadIdx.x) % L;
    const int group = static_cast<int>(threadIdx.x) / L;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups<L>;
    const T* w = static_cast<const T*>(a.w);
    const int64_t units = NV == 0 ? (a.width + V * L - 1) / (V * L) : NV;
    const float share = 1.0f / static_cast<float>(a.width);
    FloatVec<V> wv[NR], sum_w[NR];
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            wv[i] = load_unit<T, V>(w, static_cast<int64_t>(i * L + lane) * V, a.width);
            sum_w[i] = FloatVec<V>(0.0f);
        }
    }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups<L> + group; row < a.rows; row += step) {
        const T* dy = static_cast<const T*>(a.dy) + row * a.width;
        const T* dh = static_cast<const T*>(a.dh) + (DH ? row * a.width : 0);
        const T* h = static_cast<const T*>(a.h) + row * a.width;
        T* dx = static_cast<T*>(a.dx) + row * a.width;
        const float rstd = a.rstd[row];
        float dot = 0.0f;
        auto dots = [&](FloatVec<V> dn, FloatVec<V> n) {
#pragma unroll
            for (int j = 0; j < V; ++j) dot = fmaf(dn[j], n[j], dot);
        };
        auto finish = [&](int64_t col, FloatVec<V> dn, FloatVec<V> n, FloatVec<V> g) {
            FloatVec<V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = fmaf(rstd, dn[j] - n[j] * dot, g[j]);
            store_unit<T, V>(dx, col, a.width, o);
        };
        if constexpr (NV > 0) {
            FloatVec<V> d[NV], n[NV], g[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t col = static_cast<int64_t>(i * L + lane) * V;
                d[i] = load_unit<T, V>(dy, col, a.width);
                n[i] = load_unit<T, V>(h, col, a.width);
                if constexpr (DH)
                    g[i] = load_unit<T, V>(dh, col, a.width);
                else
                    g[i] = FloatVec<V>(0.0f);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                n[i] *= rstd;
#pragma unroll
                for (int j = 0; j < V; ++j) sum_w[i][j] = fmaf(d[i][j], n[i][j], sum_w[i][j]);
                d[i] *= wv[i];
                dots(d[i], n[i]);
            }
            dot = group_sum<L>(dot, lds) * share;
#pragma unroll
            for (int i = 0; i < NV; ++i) finish(static_cast<int64_t>(i * L + lane) * V, d[i], n[i], g[i]);
        } else {
            for (int64_t i = 0; i < units; ++i) {
                const int64_t col = (i * L + lane) * V;
                dots(load_unit<T, V>(dy, col, a.width) * load_unit<T, V>(w, col, a.width),
                     load_unit<T, V>(h, col, a.width) * rstd);
            }
            dot = group_sum<L>(dot, lds) * share;
            for (int64_t i = 0; i < units; ++i) {
                const int64_t col = (i * L + lane) * V;
                FloatVec<V> g = FloatVec<V>(0.0f);
                if constexpr (DH) g = load_unit<T, V>(dh, col, a.width);
                finish(col, load_unit<T, V>(dy, col, a.width) * load_unit<T, V>(w, col, a.width),
                       load_unit<T, V>(h, col, a.width) * rstd, g);
            }
        }
    }
    if constexpr (NV > 0) {
        if constexpr (L == kThreads) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                store_unit<float, V>(a.partial + blockIdx.x * a.width, static_cast<int64_t>(i * L + lane) * V, a.width,
                                       sum_w[i]);
        } else {
            __shared__ float part[kThreads * NV * V];
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) part[(group * NV + i) * (L * V) + lane * V + j] = sum_w[i][j];
            __syncthreads();
            for (int c = static_cast<int>(threadIdx.x); c < L * V * NV && c < a.width; c += kThreads) {
                float s = 0.0f;
                for (int g = 0; g < kGroups<L>; ++g) s += part[g * (L * V * NV) + c];
                a.partial[blockIdx.x * a.width + c] = s;
            }
        }
    }
}

// The weight gradient's partial sums of rows too wide for k_norm_backward's
// registers: a thread per column, a block of rows per workgroup row.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_norm_weight_partial(NormBackwardArgs a, int64_t rows_per_block) {
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (col >= a.width) return;
    const int64_t r0 = blockIdx.y * rows_per_block, r1 = min(r0 + rows_per_block, a.rows);
    const T* dy = static_cast<const T*>(a.dy);
    const T* h = static_cast<const T*>(a.h);
    float sum = 0.0f;
    for (int64_t r = r0; r < r1; ++r)
        sum = fmaf(static_cast<float>(dy[r * a.width + col]), static_cast<float>(h[r * a.width + col]) * a.rstd[r], sum);
    a.partial[blockIdx.y * a.width + col] = sum;
}

// dw[col] = the blocks' partial sums added up: kFoldRows partial chains per column, then
// those in order.  Latency bound: 7 us after 589,825 rows of 128 floats.
constexpr int kFoldCols = 16;
constexpr int kFoldRows = 64;

template <typename T>
__global__ __launch_bounds__(kFoldCols * kFoldRows) void k_norm_fold(const float* __restrict__ partial, int64_t blocks,
                                                                     int64_t width, T* __restrict__ dw) {
    __shared__ float lds[kFoldRows][kFoldCols];
    const int c = static_cast<int>(threadIdx.x) % kFoldCols, q = static_cast<int>(threadIdx.x) / kFoldCols;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kFoldCols + c;
    float sum = 0.0f;
    if (col < width)
        for (int64_t b = q; b < blocks; b += kFoldRows) sum += partial[b * width + col];
    lds[q][c] = sum;
    __syncthreads();
    if (q == 0 && col < width) {
        for (int i = 1; i < kFoldRows; ++i) sum += lds[i][c];
        dw[col] = round_to<T>(sum);
    }
}

// Most workgroups of the backward: each leaves a row of partial sums.
constexpr int64_t kMaxBlocks = 1024;
constexpr int64_t kLongRows = 64;  // rows of a workgroup of k_norm_weight_partial, at least

// Values of a lane's unit: 16 bytes where they divide the row, else a dword, else one
// value.
template <typename T>
int unit_values(int64_t width) {
    constexpr int kDword = 4 / static_cast<int>(sizeof(T));
    return width % kLaneValues<T> == 0 ? kLaneValues<T> : width % kDword == 0 ? kDword : 1;
}
template <typename T, typename F>
void with_unit(int values, F&& f) {
    if (values == kLaneValues<T>)
        f(std::integral_constant<int, kLaneValues<T>>{});
    else if (sizeof(T) < 4 && values == 2)
        f(std::integral_constant<int, sizeof(T) < 4 ? 2 : 1>{});
    else
        f(std::integral_constant<int, 1>{});
}

// Lanes of a row and units of a lane for `units` units: the fewest lanes that
// hold a row in one unit each, up to a wave (then two to four units, and the
// workgroup's lanes from 257 units on, four of each at most).  nv = 0: walked.  Three units
// spare a quarter of the registers' work of four: 60,000 rows of 160 of them (1280 in bfloat16) in
// training 249 us and 312, to 8 bits 104 and 107; of 640 floats 231 and 248.
struct NormShape {
    int lanes;
    int nv;
};
NormShape norm_shape(int64_t units) {
    if (units <= 8) return {8, 1};
    if (units <= 16) return {16, 1};
    if (units <= 32) return {32, 1};
    if (units <= 64) return {64, 1};
    if (units <= 128) return {64, 2};
    if (units <= 192) return {64, 3};
    if (units <= 256) return {64, 4};
    if (units <= 512) return {kThreads, 2};
    if (units <= 1024) return {kThreads, 4};
    return {kThreads, 0};
}

template <typename F>
void with_shape(NormShape s, F&& f) {
    using std::integral_constant;
#define RELM_SHAPE(l, n)              \
    if (s.lanes == l && s.nv == n) {  \
        f(integral_constant<int, l>{}, integral_constant<int, n>{}); \
        return;                       \
    }
    RELM_SHAPE(8, 1)
    RELM_SHAPE(16, 1)
    RELM_SHAPE(32, 1)
    RELM_SHAPE(64, 1)
    RELM_SHAPE(64, 2)
    RELM_SHAPE(64, 3)
    RELM_SHAPE(64, 4)
    RELM_SHAPE(kThreads, 2)
    RELM_SHAPE(kThreads, 4)
    f(integral_constant<int, kThreads>{}, integral_constant<int, 0>{});
#undef RELM_SHAPE
}

template <typename T, int V>
hipError_t norm_forward(const NormArgs& a, bool fp8, hipStream_t st) {
    const NormShape s = norm_shape((a.width + V - 1) / V);
    const int64_t groups = kThreads / s.lanes;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((a.rows + groups - 1) / groups, 256 * 32)));
    with_shape(s, [&](auto l, auto n) {
        constexpr int L = decltype(l)::value, NV = decltype(n)::value;
        const auto kernel = a.r != nullptr ? (fp8 ? k_norm<T, V, NV, L, true, true> : k_norm<T, V, NV, L, false, true>)
                                           : (fp8 ? k_norm<T, V, NV, L, true, false> : k_norm<T, V, NV, L, false, false>);
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, a);
    });
    return hipGetLastError();
}

int64_t backward_blocks(int64_t rows, int64_t units) {
    const NormShape s = norm_shape(units);
    if (s.nv == 0) return std::min<int64_t>((rows + kLongRows - 1) / kLongRows, kMaxBlocks);
    const int64_t groups = kThreads / s.lanes;
    return std::min<int64_t>((rows + groups - 1) / groups, kMaxBlocks);
}

template <typename T, int V>
hipError_t norm_backward(NormBackwardArgs a, void* dw, hipStream_t st) {
    const int64_t units = (a.width + V - 1) / V;
    const NormShape s = norm_shape(units);
    const int64_t blocks = backward_blocks(a.rows, units);
    with_shape(s, [&](auto l, auto n) {
        constexpr int L = decltype(l)::value, NV = decltype(n)::value;
        const int64_t grid = NV > 0 ? blocks : std::min<int64_t>(a.rows, 256 * 8);
        const auto kernel = a.dh != nullptr ? k_norm_backward<T, V, NV, L, true> : k_norm_backward<T, V, NV, L, false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, st, a);
    });
    if (s.nv == 0) {
        const int64_t per_block = (a.rows + blocks - 1) / blocks;
        hipLaunchKernelGGL(k_norm_weight_partial<T>,
                           dim3(static_cast<unsigned>((a.width + kThreads - 1) / kThreads), static_cast<unsigned>(blocks)),
                           dim3(kThreads), 0, st, a, per_block);
    }
    hipLaunchKernelGGL(k_norm_fold<T>, dim3(static_cast<unsigned>((a.width + kFoldCols - 1) / kFoldCols)),
                       dim3(kFoldCols * kFoldRows), 0, st, a.partial, blocks, a.width, static_cast<T*>(dw));
    return hipGetLastError();
}

}  // namespace

hipError_t launch_add_rms_norm(int dtype, const void* x, const void* r, const void* w, int64_t rows, int64_t width,
                               float eps, void* y, void* h, float* rstd, float* scale, hipStream_t st) {
    if (rows == 0 || width == 0) return hipSuccess;
    hipError_t e = hipErrorInvalidValue;
    const NormArgs a{x, r, w, y, h, scale, rstd, rows, width, eps};
    with_value_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_unit<T>(unit_values<T>(width),
                     [&](auto v) { e = norm_forward<T, decltype(v)::value>(a, scale != nullptr, st); });
    });
    return e;
}

size_t add_rms_norm_backward_workspace(int dtype, int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    int64_t blocks = 0;
    with_value_type(dtype, [&](auto t) {
        blocks = backward_blocks(rows, width / unit_values<decltype(t)>(width));
    });
    return static_cast<size_t>(blocks * width) * sizeof(float);
}

hipError_t launch_add_rms_norm_backward(int dtype, const void* dy, const void* dh, const void* h, const void* w,
                                        const float* rstd, int64_t rows, int64_t width, void* dx, void* dw, float* partial,
                                        hipStream_t st) {
    if (width == 0) return hipSuccess;
    hipError_t e = hipErrorInvalidValue;
    const NormBackwardArgs a{dy, dh, h, w, rstd, dx, partial, rows, width};
    with_value_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (rows == 0) {
            hipLaunchKernelGGL(k_norm_fold<T>, dim3(static_cast<unsigned>((width + kFoldCols - 1) / kFoldCols)),
                               dim3(kFoldCols * kFoldRows), 0, st, nullptr, int64_t{0}, width, static_cast<T*>(dw));
            e = hipGetLastError();
            return;
        }
        with_unit<T>(unit_values<T>(width),
                     [&](auto v) { e = norm_backward<T, decltype(v)::value>(a, dw, st); });
    });
    return e;
}

}  // namespace relm_mp
