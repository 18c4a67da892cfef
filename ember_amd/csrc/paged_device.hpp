// Device-side pieces shared by the kernels that read KV pages with a wave per
// page: scalar loads, page loads through buffer descriptors, and the MFMA
// layouts' cross-lane steps (lane l = 16 g + c serves query column c).
#pragma once

#include "device.hpp"

namespace ember::hip {

// A load through the constant address space: with a wave-uniform address the
// compiler emits s_load (scalar cache, lgkmcnt), which never waits for the
// vector page loads in flight. Only for data the kernel does not write.
template <class T>
__device__ __forceinline__ T uniform_load(const T *p) {
    return *(const __attribute__((address_space(4))) T *)(p);  // an address-space cast
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kDescWord3 = 0x00020000;  // gfx9 raw buffer: 32-bit data format, no swizzle
constexpr int kNonTemporal = 2;         // cache-policy bit nt of a gfx950 buffer load

__device__ __forceinline__ u32x4 load_desc(__amdgpu_buffer_rsrc_t d, uint32_t off) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(d, off, 0, kNonTemporal));
}

// 2^x by the hardware instruction (v_exp_f32): exact powers of two at
// integers, 0 at -inf; results below 2^-126 may flush to 0, which only drops
// weights that cannot move an f32 sum.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// f16 pages: max and sum over the four lane groups of a query column (lanes
// c, c + 16, c + 32, c + 48). Groups 0 and 1, and 2 and 3, meet through
// v_permlane16_swap, then the pairs through v_permlane32_swap. Both operations
// are commutative, so every lane of the column gets the same bits; the sum is
// (x0 + x1) + (x2 + x3).
__device__ __forceinline__ float groups_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// f16 pages: the A operand of the value products' dim tile TILE, dim
// 8 c + TILE of this lane's keys 4 g .. 4 g + 3 (its four 8-dim slices of V,
// one per key): two v_perm, each pairing one half of a word of two keys.
template <int TILE>
__device__ __forceinline__ f16x4 value_tile(const u32x4 (&v)[4]) {
    constexpr uint32_t sel = (TILE & 1) ? 0x07060302u : 0x05040100u;  // high or low halves of (b, a)
    constexpr int w = TILE / 2;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 pair = {__builtin_amdgcn_perm(v[1][w], v[0][w], sel),   // keys 4g, 4g + 1
                        __builtin_amdgcn_perm(v[3][w], v[2][w], sel)};  // keys 4g + 2, 4g + 3
    return __builtin_bit_cast(f16x4, pair);
}

__device__ __forceinline__ f16x8 as_f16x8(const u32x4 &x) { return __builtin_bit_cast(f16x8, x); }

// The running max of a row before any visible key: finite and far below any
// score (|q.k| * scale of f16 vectors is below 1e12), so a row's first visible
// key gives corr = 2^(kNoMax - max) = 0 exactly, as -inf would, while an empty
// row keeps l = 0 and O = 0; the merges below treat it like -inf (weight 0
// against any real max, and zeros when every part is empty).
constexpr float kNoMax = -1.0e30f;

}  // namespace ember::hip
