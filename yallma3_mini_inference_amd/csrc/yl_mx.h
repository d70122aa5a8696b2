// yl_mx.h -- MXFP4 values: blocks of 32 elements of 4 bits (sign, two bits of
// exponent, one of mantissa: 0, 1/2, 1, 3/2, 2, 3, 4, 6) under one scale byte E
// that stands for 2^(E - 127); 255: the whole block is NaN.
//
// Every such value with E from 2 to 252 is a normal bf16 (at most two bits of
// mantissa), so nothing is lost where products take bf16.
#pragma once

#include "yl_device.h"

namespace yl {

// An element of such pages as the attention's products see it.
struct Mx4 { __bf16 value; };

// The scale byte of a block whose largest |element| has the bits `amax` (of f32,
// sign cleared; all of 0x7f800000 or above: an infinity or NaN among them).
// The largest element is below 7 units, so that it is rounded to 6 by at most
// half a step (the next unit would cost all others a bit; a unit by the exponent
// alone would cut off up to a quarter of the largest).
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax) {
    const int e = (int)((amax + 0x200000u) >> 23) - 2;
    return amax >= 0x7f800000u ? 255u : (uint32_t)min(max(e, 2), 252);
}

__device__ __forceinline__ float mx_unit(uint32_t scale) { return __uint_as_float(scale << 23); }

// Four elements' codes, the first in the low bits: to nearest, ties to even codes, saturating at 6 units.
__device__ __forceinline__ uint32_t mx_codes(float a, float b, float c, float d, float unit) {
    const uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, unit, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c, d, unit, 1) & 0xffffu;
}

// Byte `I`'s two elements as packed bf16.
template <int I>
__device__ __forceinline__ uint32_t mx_pair(uint32_t codes, float unit) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, unit, I);
    return __builtin_bit_cast(uint32_t, v);
}

// The largest of 4 or 8 neighbouring lanes (the whole group active).
template <int LANES>
__device__ __forceinline__ uint32_t mx_group_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
    if (LANES == 8) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
    return v;
}

}  // namespace yl
