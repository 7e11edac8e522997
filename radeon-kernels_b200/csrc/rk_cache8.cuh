// rk_cache8.cuh -- the two 8-bit element types of the quantised K/V cache, on the device.
//
// E4m3: 4 exponent and 3 mantissa bits, largest value 448.  Int8: -127..127.  A stored value
// stands for itself times the fp32 scale of its block and head.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>

#include "rk_device.cuh"

namespace rk {

// The least power of two s with amax <= LARGEST * s, never below 2^-126 (so that 1 / s is
// finite): the exponent of amax less that of LARGEST, one more where amax's mantissa exceeds
// LARGEST's.
template <int LARGEST_EXPONENT, uint32_t LARGEST_MANTISSA>
__device__ __forceinline__ float power_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - LARGEST_EXPONENT + ((bits & 0x7FFFFFu) > LARGEST_MANTISSA ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}

struct E4m3 {
  static __device__ __forceinline__ float scale_for(float amax) { return power_scale<8, 0x600000u>(amax); }  // 1.75 * 2^8
  // Four values to four bytes, nearest even, saturating; NaN stays NaN.
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  }
  // Bytes 0, 1 (lo) and 2, 3 (hi) as pairs of halves; exact.
  static __device__ __forceinline__ void halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
};

struct Int8 {
  static __device__ __forceinline__ float scale_for(float amax) { return power_scale<6, 0x7E0000u>(amax); }  // 1.984375 * 2^6
  // NaN becomes 0, infinities the largest value.
  static __device__ __forceinline__ uint32_t byte(float v) {
    return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(v)))) & 0xFFu;
  }
  static __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    return byte(a) | (byte(b) << 8) | (byte(c) << 16) | (byte(d) << 24);
  }
  // With its sign bit flipped a byte is the value plus 128; as the low byte of the half
  // 0x6400 it stands for 1024 + that, so subtracting 1152 gives the value, exactly.
  static __device__ __forceinline__ void halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 k = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), k), y = __hsub2(*reinterpret_cast<__half2*>(&b), k);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
};

}  // namespace rk
