// svsx_paged.h -- what the translation units of the operators over paged rows share (svsx_cache.hip, svsx_attention.hip, svsx_latent.hip).
#pragma once

#include "../../include/svsx.h"
#include <hip/hip_runtime.h>
#include <atomic>
#include <stddef.h>
#include <stdint.h>

namespace svsx {

// bytes of a row element; 0 = not a type these operators take (the 8-bit row types of the indexes have no meaning here)
inline size_t paged_dtype_size(int dtype) { return dtype == SVSX_F32 ? 4 : dtype == SVSX_F16 || dtype == SVSX_BF16 ? 2 : 0; }

// The device of a call, and the caller's own device again afterwards.
struct DeviceScope {
    int before = -1;
    hipError_t error;
    explicit DeviceScope(int device) {
        error = hipGetDevice(&before);
        if (error == hipSuccess && before != device) error = hipSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

// A kernel that uses more than 64 KB of LDS asks for it, once on each device (bit d of *granted: device d).
inline hipError_t grant_lds(const void* kernel, int bytes, std::atomic<uint64_t>* granted) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
    if (e != hipSuccess || (granted->load(std::memory_order_relaxed) & bit)) return e;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) granted->fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// 16-bit and 32-bit row elements; sums are float32 everywhere
typedef __bf16 bf16_t;
template <typename T> __device__ __forceinline__ float to_f32(T x) { return static_cast<float>(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x) { return static_cast<T>(x); } // to nearest, ties to even

constexpr int kMaxDim = 1024; // columns of a key or value row that attention takes

// One workgroup of four waves, one query head: softmax(scale * q . k) . v over rows [0, n) in float32, the rows dealt to the waves in turn and each wave's lanes
// across the columns.  `q` in LDS; key_of(r) / value_of(r): row r, or NULL where it is left out.  Result in sm.out[0..dv), normalised.  Every row is read once
// and nothing is shared between heads: right for any size, type and alignment, and the form that the faster kernels are checked against.
struct RowsShared {
    float q[kMaxDim];
    float out[4][kMaxDim];
    float top[4], sum[4];
};
template <typename T, typename K, typename V>
__device__ __forceinline__ float attend_rows(RowsShared& sm, uint32_t n, uint32_t dk, uint32_t dv, float scale, K key_of, V value_of) {
    constexpr int kPer = kMaxDim / 64;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float o[kPer], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = 0.0f;
    for (uint32_t r = wave; r < n; r += 4) {
        const T* k = key_of(r);
        if (k == nullptr) continue;
        float s = 0.0f;
        for (uint32_t c = lane; c < dk; c += 64) s = fmaf(sm.q[c], to_f32(k[c]), s);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off);
        s *= scale;
        if (s == -INFINITY) continue; // no weight; it must not become the difference of two infinities
        const float t = s > top || s != s ? s : top, was = expf(top - t), p = expf(s - t);
        top = t;
        sum = fmaf(sum, was, p);
        const T* v = value_of(r);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t c = lane + 64 * i;
            if (c < dv) o[i] = fmaf(p, to_f32(v[c]), o[i] * was);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (lane + 64 * i < dv) sm.out[wave][lane + 64 * i] = o[i];
    if (lane == 0) {
        sm.top[wave] = top;
        sm.sum[wave] = sum;
    }
    __syncthreads();
    float all = -INFINITY, total = 0.0f, w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) all = sm.top[i] > all || sm.top[i] != sm.top[i] ? sm.top[i] : all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = sm.top[i] == -INFINITY ? 0.0f : expf(sm.top[i] - all);
        total = fmaf(sm.sum[i], w[i], total);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    for (uint32_t c = threadIdx.x; c < dv; c += 256) {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) x = fmaf(sm.out[i][c], w[i], x);
        sm.out[0][c] = x * inv;
    }
    __syncthreads();
    return total == 0.0f ? -INFINITY : all + logf(total);
}

} // namespace svsx
