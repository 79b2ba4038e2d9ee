// Matrix-instruction fragments of the readout kernels, the same for 16-bit and
// float values: a lane holds 8 neighbouring values of a row's contraction axis.
//
// Product of A [16 x 32] and B [32 x 16] in a wave: lane l holds A[l % 16][8 (l / 16)
// .. + 8] and B[8 (l / 16) .. + 8][l % 16]; entry i of the result is C[4 (l / 16) +
// i][l % 16].  16-bit values take one instruction of depth 32; float values eight
// of depth 4, the j-th over the lanes' j-th values.  Only the pairing of A and B
// matters for the sum, so any order of the contraction axis serves that both
// fragments share.
#pragma once

#include <hip/hip_runtime.h>

#include "value_types.h"

namespace relm_mp {

using f32x4 = float __attribute__((ext_vector_type(4)));
template <typename T>
using Frag = T __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x4 mma(const Frag<T>& a, const Frag<T>& b, f32x4 c) {
    if constexpr (std::is_same_v<T, bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, f16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
}

// The fragment of a row-major tile in LDS (rows of `stride` values, 16-byte aligned):
// row `row`, values [col, col + 8).
template <typename T>
__device__ __forceinline__ Frag<T> lds_frag(const T* tile, int stride, int row, int col) {
    using Half = T __attribute__((ext_vector_type(16 / sizeof(T))));
    const T* p = tile + row * stride + col;
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        f = *reinterpret_cast<const Half*>(p);
    } else {
        const Half lo = *reinterpret_cast<const Half*>(p), hi = *reinterpret_cast<const Half*>(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = lo[j];
            f[4 + j] = hi[j];
        }
    }
    return f;
}

// The fragment of the tile's transpose that pairs with a result of two products
// (rows 16 t + 4 g + i of lane group g, t = 0, 1): for column `col0 + l % 16` of the
// tile the rows row0 + 4 g + j (j < 4) and row0 + 16 + 4 g + (j - 4).  16-bit values
// through the transposing LDS read: within 16 lanes, lane i reads 4 values of row i /
// 4 and receives column i.
template <typename T>
__device__ __forceinline__ Frag<T> lds_frag_t(const T* tile, int stride, int row0, int col0) {
    const int l = static_cast<int>(threadIdx.x) & 63, g = l / 16, i = l % 16;
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        using Bits = short __attribute__((ext_vector_type(4)));
        using Quad = T __attribute__((ext_vector_type(4)));
        const T* p = tile + (row0 + 4 * g + i / 4) * stride + col0 + (i % 4) * 4;
        const auto* q = reinterpret_cast<const Bits*>(p);
        const Bits lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) Bits*)(const_cast<Bits*>(q)));
        const auto* r = reinterpret_cast<const Bits*>(p + 16 * stride);
        const Bits hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) Bits*)(const_cast<Bits*>(r)));
        const Quad a = __builtin_bit_cast(Quad, lo), b = __builtin_bit_cast(Quad, hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = a[j];
            f[4 + j] = b[j];
        }
    } else {
        const T* p = tile + (row0 + 4 * g) * stride + col0 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = p[j * stride];
            f[4 + j] = p[(16 + j) * stride];
        }
    }
    return f;
}

// lds_frag_t of the first 16 RT rows of a tile (RT = 1: the other 16 are zeros).
template <typename T, int RT>
__device__ __forceinline__ Frag<T> rows_frag_t(const T* tile, int stride, int col0) {
    if constexpr (RT == 2) return lds_frag_t<T>(tile, stride, 0, col0);
    const int l = static_cast<int>(threadIdx.x) & 63, g = l / 16, i = l % 16;
    Frag<T> f = Frag<T>(static_cast<T>(0.0f));
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = tile[(4 * g + j) * stride + col0 + i];
    return f;
}

// 8 values to LDS, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void lds_put(T* to, const Frag<T>& f) {
    using Part = T __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int p = 0; p < 8 / N; ++p) {
        Part x;
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = f[p * N + j];
        *reinterpret_cast<Part*>(to + p * N) = x;
    }
}

// Two results of neighbouring 16-row tiles as the fragment that pairs with
// lds_frag_t, rounded to T.
template <typename T>
__device__ __forceinline__ Frag<T> frag_of(f32x4 lo, f32x4 hi) {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = round_to<T>(lo[j]);
        f[4 + j] = round_to<T>(hi[j]);
    }
    return f;
}

}  // namespace relm_mp
