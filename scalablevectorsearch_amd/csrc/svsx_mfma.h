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

// product32(a, b, c): c[32 x 32] += A[32 x 16] B[16 x 32]; lane l holds row / column l % 32, elements 8 (l / 32) .. + 7 of the 16; of c column l % 32, and in register
// 4 i + j row 8 i + 4 (l / 32) + j.
typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16 product32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 product32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 product32(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
// Which of 32 rows a lane of product32 reads so that registers 8 i .. 8 i + 7 of the result are rows 16 i + 8 (l / 32) .. + 7, eight consecutive ones: a fragment of the
// next product as they are, and one 16-byte word of a 16-bit type.
__device__ __forceinline__ uint32_t row32(uint32_t lane) { return (lane & 0x13) | (lane & 8) >> 1 | (lane & 4) << 1; }

// 2^x; the hardware's instruction, denormal results are zero
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// The running maximum of a softmax is raised only when a score exceeds it by more than kSlack powers of two.
constexpr float kSlack = 4.0f;
// Probabilities are rounded to the row type before they meet the values; float16 gets them 2^8 up, so that small ones stay normal numbers (at most 2^12 with the slack).
template <typename T> inline constexpr float kLift = 0.0f;
template <> inline constexpr float kLift<_Float16> = 8.0f;

#pragma clang diagnostic ignored "-Winline-asm" // m0 is a reserved register; the compiler is told that it changes
// 16 bytes per lane from base + offset to LDS at `to` + 16 * lane; not waited for (direct_wait).
__device__ __forceinline__ void direct_load(const void* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void direct_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// a barrier for what went through LDS: loads from HBM stay in flight over it
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
typedef __attribute__((address_space(3))) unsigned char lds_byte;

// Orders the block that it stands in: LDS reads Ahead fragments ahead of the products that use them (N fragments and N products in all; reads and instructions
// per fragment and product by type).  Left to itself the compiler reads each fragment right before its product and waits for it.
template <typename T, int N, int Ahead> __device__ __forceinline__ void reads_ahead() {
    constexpr int kReads = sizeof(T) == 2 ? 1 : 2, kProducts = sizeof(T) == 2 ? 1 : 8;
    __builtin_amdgcn_sched_group_barrier(0x100, Ahead * kReads, 0);
#pragma unroll
    for (int i = 0; i < N - Ahead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, kProducts, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, Ahead * kProducts, 0);
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
