// Value types of the readout kernels (float, bfloat16, half): vectors of them,
// their loads and stores at the alignment that strided rows leave, and the
// rounding to fewer bits.  All arithmetic on them is in float.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "relm_mp.h"

namespace relm_mp {

using bf16 = __bf16;
using f16 = _Float16;

// N values of T wherever they start: the target's global memory takes accesses of up to
// 16 bytes at any address, and the compiler makes one of each.
template <typename T, int N>
using ValueVec = T __attribute__((ext_vector_type(N), aligned(sizeof(T))));
template <int N>
using FloatVec = float __attribute__((ext_vector_type(N)));

// Values of a 16-byte access.
template <typename T>
constexpr int kLaneValues = 16 / static_cast<int>(sizeof(T));

// Rounds to nearest even, as every conversion to T here.
template <typename T>
__device__ __forceinline__ T round_to(float x) {
    return static_cast<T>(x);
}

// Values [col, col + N) of a row of `width`, zero past its end; one access where
// all of them exist.
template <typename T, int N>
__device__ __forceinline__ FloatVec<N> load_values(const T* __restrict__ row, int64_t col, int64_t width) {
    FloatVec<N> x;
    if constexpr (N == 1) {
        x[0] = col < width ? static_cast<float>(row[col]) : 0.0f;
    } else if (col + N <= width) {
        const ValueVec<T, N> v = *reinterpret_cast<const ValueVec<T, N>*>(row + col);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = static_cast<float>(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = col + i < width ? static_cast<float>(row[col + i]) : 0.0f;
    }
    return x;
}

// Calls f with a value of the type that a dtype code stands for; false where it
// stands for none of them.
template <typename F>
bool with_value_type(int dtype, F&& f) {
    switch (dtype) {
        case RELM_MP_F32: f(float{}); return true;
        case RELM_MP_BF16: f(bf16{}); return true;
        case RELM_MP_F16: f(f16{}); return true;
        default: return false;
    }
}

inline size_t value_bytes(int dtype) { return dtype == RELM_MP_F32 ? 4 : 2; }

}  // namespace relm_mp
