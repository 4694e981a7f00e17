// Block-scaled 8-bit values: e4m3 with a power-of-two scale for each block of 128, held as the byte e + 127 of its exponent e.
#pragma once
#include "elem.hpp"

namespace gf {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr uint32_t kScaleNone = 255;      // the scale of a block that holds an infinity or a NaN

// Bits of the largest magnitude of a block -> the byte of the smallest exponent e >= -127 with it <= 448 * 2^e.
// 448 = 1.75 * 2^8: e = exponent - 8, one more where the significand is above 1.75 (0x600000), which is what the addition carries.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
    if (amax >= 0x7f800000u) return kScaleNone;
    const uint32_t e = (amax + 0x1fffffu) >> 23;
    return e > 8 ? e - 8 : 0;
}

// 2^-(byte - 127), by which a block's values are multiplied (exactly); not a number where the block is none, so that all its codes are none too
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
    return byte == kScaleNone ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - byte) << 23);
}

// four values to four codes, each rounded to nearest even once; |x * inverse| <= 448, so nothing saturates
__device__ __forceinline__ uint32_t encode4(const float x[4], float inverse) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inverse, x[1] * inverse, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inverse, x[3] * inverse, w, true);
}

}  // namespace gf
