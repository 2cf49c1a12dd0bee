// svsx_mfma.h -- fragments and products of the matrix units as the attention kernels use them, the same for every row type.
//
// A fragment is 8 consecutive elements of a row (16 bytes of a 16-bit type).  product16(a, b, c): c[16 x 16] += A[16 x 32] B[32 x 16]; lane l holds row (a) or
// column (b) l % 16, elements 8 (l / 16) .. + 7 of the 32; of c it holds column l % 16, rows 4 (l / 16) .. + 3.  float32 rows take eight 16x16x4 products,
// the j-th of the j-th elements: which elements meet does not matter as long as both sides agree, so the layout is that of the 16-bit types.
#pragma once

#include "svsx_paged.h"

namespace svsx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct FragOf;
template <> struct FragOf<float> { typedef f32x8 type; };
template <> struct FragOf<_Float16> { typedef f16x8 type; };
template <> struct FragOf<bf16_t> { typedef bf16x8 type; };
template <typename T> using Frag = typename FragOf<T>::type;

__device__ __forceinline__ f32x4 product16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 product16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 product16(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// elements [col, col + 8) of a row of `dim`; zero beyond it.  Wide: rows begin at 16-byte boundaries and dim is a multiple of 8.
template <typename T, bool Wide> __device__ __forceinline__ Frag<T> load_frag(const T* row, uint32_t col, uint32_t dim) {
    Frag<T> f = {};
    if constexpr (Wide) {
        if (col < dim) f = *reinterpret_cast<const Frag<T>*>(row + col);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (col + j < dim) f[j] = row[col + j];
    }
    return f;
}

// n / d for n < 2^31, with inverse = (2^32 - 1) / d: the product's high half is the quotient or one less.
struct Divider {
    uint32_t d, inverse;
    __device__ __forceinline__ uint32_t operator()(uint32_t n, uint32_t* rest) const {
        uint32_t q = __umulhi(n, inverse), r = n - q * d;
        if (r >= d) {
            ++q;
            r -= d;
        }
        *rest = r;
        return q;
    }
};
inline Divider divider(uint32_t d) { return Divider{d, 0xFFFFFFFFu / d}; }

} // namespace svsx
