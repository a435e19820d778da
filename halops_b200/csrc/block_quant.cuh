// e4m3 codes with a float32 scale per block of 128: what the kernels that quantise in that form share.
//
//   amax = max(max |x| over the block, 1e-10),   scale = amax / 448,   code = e4m3(x * 448 / amax)
//
// nearest code, ties to even.  The quotient is computed as x * r with r = 448 / amax, whose error of up to 2 units of the
// last place could carry a value that lies midway between two codes to either side.  A 16-bit x has 11 significant bits at most
// and so has amax; a midpoint has 5 at most and 448 = 7 * 64.  x * 448 / amax therefore either is a midpoint or differs from
// it by 2^-16 of its value at least, and rounding the product to a multiple of 8 units of its last place (2^-20 of the
// value at most) puts it back on the midpoint where it belongs there and moves nothing else across: the codes are those of the
// exact quotient.  (Below the floor amax has 24 bits, and no quotient is a midpoint; that none is near enough to one to be moved onto
// it was tried for all 11996 bf16 magnitudes there.)
// A NaN or an infinity in a block makes its scale NaN or infinite (as maximum of the bit patterns, where NaN is
// above infinity and infinity above the rest), so that every product with the block is NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "common.cuh"

namespace hq {
namespace {

constexpr int kQBlock = 128;            // values of a row per scale
constexpr uint32_t kAmaxFloorBits = 0x2edbe6ffu;  // 1e-10f
constexpr uint32_t kInfF32 = 0x7f800000u;

// Kernel pointers are not __restrict__ and not read through __ldg: what they point to changes, in the preceding kernel, while this one
// waits for it, and a load of constant data may be moved to before the wait.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Two 16-bit values of a word as float32.
template <typename T>
__device__ __forceinline__ float2 two_floats(uint32_t w);
template <>
__device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 two_floats<__half>(uint32_t w) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}

// Magnitude of a 16-bit value's bit pattern (without its sign) as the bit pattern of a float32.
template <typename T>
__device__ __forceinline__ uint32_t magnitude_f32(uint32_t bits16);
template <>
__device__ __forceinline__ uint32_t magnitude_f32<__nv_bfloat16>(uint32_t b) {
    return b << 16;
}
template <>
__device__ __forceinline__ uint32_t magnitude_f32<__half>(uint32_t b) {
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(b))));  // (NaN stays NaN)
}

// Largest bit pattern of |x| over 8 values.
__device__ __forceinline__ uint32_t amax16(const uint4& v) {
    const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}

struct BlockScale {
    float scale;    // amax / 448
    float inverse;  // 448 / amax
    uint32_t add, mask;  // rounding of the products to multiples of 8 units (finite blocks of 16-bit values)
};

__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits, bool snap) {
    const float amax = __uint_as_float(max(amax_bits, kAmaxFloorBits));
    BlockScale s;
    s.scale = __fdiv_rn(amax, 448.0f);
    s.inverse = __fdiv_rn(448.0f, amax);
    const bool on = snap && amax_bits < kInfF32;
    s.add = on ? 4u : 0u;
    s.mask = on ? ~7u : ~0u;
    return s;
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t code2(float2 v, const BlockScale& s) {
    const float a = __uint_as_float((__float_as_uint(v.x * s.inverse) + s.add) & s.mask);
    const float b = __uint_as_float((__float_as_uint(v.y * s.inverse) + s.add) & s.mask);
    return e4m3x2(a, b);
}

// 8 values -> 8 codes.
template <typename T>
__device__ __forceinline__ uint2 codes8(const uint4& v, const BlockScale& s) {
    return make_uint2(code2(two_floats<T>(v.x), s) | code2(two_floats<T>(v.y), s) << 16,
                      code2(two_floats<T>(v.z), s) | code2(two_floats<T>(v.w), s) << 16);
}

}  // namespace
}  // namespace hq
