// A cache row in 8 bits: one token's key (or value) of one kv head as codes of 1 sign, 4 exponent and 3 mantissa bits
// (e4m3: largest 448, smallest 2^-9, no infinities) and one byte e for the row, its numbers being code * 2^(e - 127).
//
// The scale is the smallest power of two with which the row's largest magnitude is at most 448, not below 2^-110, and 1 for
// a row of zeros.  A power of two, because a code has four significant bits: code * scale is then a bfloat16 exactly (down to
// 2^-9 * 2^-110, still a normal number), so that reading back rounds nothing, and a tensor core's product of codes needs only
// an exponent added.  A row that holds a number which is not finite in 32 bits gets e = 255 and codes 0, and reads as NaN
// everywhere: what a reader does with a NaN is then decided by the byte alone, and no code ever is one.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

constexpr int Q8_LEAST_POWER = -110;
constexpr int Q8_NAN_BYTE = 255;

// A 64-bit number to 32 bits, rounded to odd: the last bit is set where bits were lost, so that rounding the result to fewer
// bits gives what rounding the 64-bit number would, and comparing it with such a number too.
__device__ __forceinline__ float q8_to_odd(double x) {
  if (fabs(x) >= 3.4028235677973366e38) return (float)x;      // rounds to an infinity (and infinities)
  float f = __double2float_rz(x);
  if ((double)f != x) f = __uint_as_float(__float_as_uint(f) | 1u);
  return f;
}

// The scale byte of a row whose largest magnitude has these bits (as an integer: NaN is above infinity, infinity above the rest).
__device__ __forceinline__ int q8_byte(uint32_t top) {
  if (top >= 0x7f800000u) return Q8_NAN_BYTE;
  if (top == 0) return 127;
  const int power = (int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);      // 1.75 * 2^8 = 448
  return max(power, Q8_LEAST_POWER) + 127;
}
// What codes of a row with this byte are made from: x * q8_inverse(byte).  NaN rows give 0 (and 0 * NaN is caught by q8_pair).
__device__ __forceinline__ float q8_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
// 2^(byte - 127), NaN for 255.
__device__ __forceinline__ float q8_scale(uint32_t byte) {
  return byte == Q8_NAN_BYTE ? __uint_as_float(0x7fffffffu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// Two numbers to codes, rounded to nearest even; the first in the low byte.
__device__ __forceinline__ uint32_t q8_encode2(float first, float second) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(second), "f"(first));
  return r;
}
__device__ __forceinline__ uint32_t q8_encode4(float a, float b, float c, float d) {
  return q8_encode2(a, b) | q8_encode2(c, d) << 16;
}
// Two codes to numbers (16 bits hold them exactly).
__device__ __forceinline__ float2 q8_decode2(uint16_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(codes));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float4 q8_decode4(uint32_t codes) {
  const float2 lo = q8_decode2((uint16_t)codes), hi = q8_decode2((uint16_t)(codes >> 16));
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ float q8_decode(uint8_t code) { return q8_decode2(code).x; }
