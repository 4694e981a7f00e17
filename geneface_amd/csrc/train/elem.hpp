// Element types of the training-step kernels: 32-bit, bfloat16 and binary16 values, all computed on in 32 bits.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gf {

enum { F32 = 0, BF16 = 1, F16 = 2 };

// Four consecutive values at any address that their type allows: the memory pipeline takes 16- and 8-byte accesses at any of them.
template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Vec4<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Vec4<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4), aligned(2))); };

template <typename T>
__device__ __forceinline__ void load4(const T* src, float out[4]) {
    const typename Vec4<T>::type v = *reinterpret_cast<const typename Vec4<T>::type*>(src);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (float)v[i];
}
template <typename T>
__device__ __forceinline__ void store4(T* dst, const float in[4]) {
    typename Vec4<T>::type v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)in[i];      // one rounding to nearest even
    *reinterpret_cast<typename Vec4<T>::type*>(dst) = v;
}

// four values of which the first `left` exist (0 for the others)
template <typename T>
__device__ __forceinline__ void load4_of(const T* src, int left, float out[4]) {
    if (left >= 4) { load4(src, out); return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = i < left ? (float)src[i] : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store4_of(T* dst, int left, const float in[4]) {
    if (left >= 4) { store4(dst, in); return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < left) dst[i] = (T)in[i];
}

// largest of a value over the 16 lanes of a row, by rotations inside it
__device__ __forceinline__ uint32_t row_max_u32(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false));   // row_ror:8
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false));
    return x;
}

// largest magnitude; NaN where either is (v_maximum3_f32)
__device__ __forceinline__ float max_abs(float a, float x) { return __builtin_elementwise_maximum(a, __builtin_fabsf(x)); }

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

}  // namespace gf
