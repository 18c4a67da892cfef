// The 4-bit format on the device: e2m1 codes in groups of 32 with a
// power-of-two scale byte, and the layout of a page of a 4-bit cache.
//
// gfx950 converts both ways in one instruction for two values, scale included
// (v_cvt_scalef32_pk_f16_fp4 and v_cvt_scalef32_pk_fp4_f32: 4 cycles a wave,
// as any other VALU instruction). Both are exact as the format is defined in
// the header: checked for all 256 scale bytes times all codes one way
// (subnormal f16 results, infinities and the NaN scale among them), and at
// every border between two codes and beside it for all scales the other way.
#pragma once

#include "device.hpp"
#include "ember_hip.h"
#include "paged_device.hpp"

namespace ember::hip {

constexpr int kMxGroup = EMBER_MX_GROUP;
constexpr int kMxLowest = 104, kMxHighest = 140;  // scale bytes that are written: 2^-23 .. 2^13

constexpr int kKv4Page = EMBER_KV4_PAGE_BYTES;
constexpr int kKv4Values = kPage * kHeadDim / 2;                     // bytes: where the V codes start,
constexpr int kKv4KeyScales = 2 * kKv4Values;                        // the K scales
constexpr int kKv4ValueScales = kKv4KeyScales + kPage * kHeadDim / kMxGroup;  // and the V scales
static_assert(kKv4ValueScales + kPage * kHeadDim / kMxGroup == kKv4Page);

// The scale of a group of largest magnitude m >= 0 (finite): the lowest of the
// written ones with m <= 7 scale. 7 is 1.75 * 2^2, so a mantissa above 1.75
// (0x600000) carries into the exponent.
__device__ __forceinline__ int mx_scale_byte(float m) {
    const int e = static_cast<int>((__float_as_uint(m) + 0x1fffffu) >> 23);
    return min(max(e - 2, kMxLowest), kMxHighest);
}

// Scale byte i of a word where the conversions look for it, at an f32's exponent (255 there is the scale NaN). They
// look at the exponent alone (checked for all scales and codes), so the word's other bytes may stay in the other bits.
// (`i` is known where loops are unrolled: one shift.)
__device__ __forceinline__ float mx_scale(uint32_t word, int i = 0) {
    return __uint_as_float(i < 3 ? word << (23 - 8 * i) : word >> 1);
}

// Eight values' codes, the first in the lowest four bits.
__device__ __forceinline__ uint32_t mx_encode8(const float (&x)[8], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

__device__ __forceinline__ u32x4 mx_decode8(uint32_t w, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
}

}  // namespace ember::hip
