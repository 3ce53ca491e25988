// 8-bit page codes: conversion between codes and values, and the exponent
// rule of a page's scale.  Scales are powers of two, so code * scale is exact
// in 32 bits, and raising a scale rounds a held code once more to the new unit
// and nothing else.
#pragma once

#include "common.cuh"

namespace ic {
namespace q8 {

constexpr int PAGE = 16;              // tokens per page
constexpr int E_MIN = -60, E_MAX = 60;

// CODE is IC_E4M3 or IC_I8.  amax <= QMAX * 2^e with amax = m * 2^x, m in
// [0.5, 1): QMAX = 448 = 0.875 * 2^9 or 127 = (127/128) * 2^7, so
// e = x - BITS, one more when m exceeds the factor (compared as the 23
// fraction bits below the leading one).
template <int CODE> struct Fmt;
template <> struct Fmt<IC_E4M3> {
  static constexpr float QMAX = 448.f;
  static constexpr int BITS = 9;
  static constexpr uint32_t TOP_FRAC = 0x600000u;
};
template <> struct Fmt<IC_I8> {
  static constexpr float QMAX = 127.f;
  static constexpr int BITS = 7;
  static constexpr uint32_t TOP_FRAC = 0x7E0000u;
};

__device__ __forceinline__ int clamp_exp(int e) { return max(E_MIN, min(E_MAX, e)); }

// amax_bits: the bits of a finite non-negative float.
template <int CODE>
__device__ __forceinline__ int exponent_for(uint32_t amax_bits) {
  const int x = static_cast<int>(amax_bits >> 23) - 126;
  return clamp_exp(x - Fmt<CODE>::BITS + ((amax_bits & 0x7FFFFFu) > Fmt<CODE>::TOP_FRAC ? 1 : 0));
}
__device__ __forceinline__ int exponent_of(float scale) {
  return clamp_exp(static_cast<int>((__float_as_uint(scale) >> 23) & 255u) - 127);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Four values (already divided by the scale) to four codes, round to nearest
// even, saturating; NaN gives 0.
template <int CODE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  a = a != a ? 0.f : a;
  b = b != b ? 0.f : b;
  c = c != c ? 0.f : c;
  d = d != d ? 0.f : d;
  if (CODE == IC_E4M3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
  }
  const auto one = [](float x) {
    return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x, -127.f), 127.f))) & 255u;
  };
  return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
}

// Four codes to four fp16 values (exact), two per register in byte order.
// int8: byte b with its sign bit flipped is b + 128; under the fp16 exponent
// of 1024 it reads as 1024 + (b + 128), and subtracting 1152 is exact.
template <int CODE>
__device__ __forceinline__ void decode4_h2(uint32_t v, uint32_t& lo, uint32_t& hi) {
  if (CODE == IC_E4M3) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(v));
  } else {
    const uint32_t x = v ^ 0x80808080u;
    const __half2 off = __float2half2_rn(1152.f);
    uint32_t l = __byte_perm(x, 0x64646464u, 0x4140), h = __byte_perm(x, 0x64646464u, 0x4342);
    __half2 l2 = __hsub2(*reinterpret_cast<__half2*>(&l), off), h2 = __hsub2(*reinterpret_cast<__half2*>(&h), off);
    lo = *reinterpret_cast<uint32_t*>(&l2);
    hi = *reinterpret_cast<uint32_t*>(&h2);
  }
}
template <int CODE>
__device__ __forceinline__ void decode4(uint32_t v, float* o) {
  uint32_t lo, hi;
  decode4_h2<CODE>(v, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}

}  // namespace q8
}  // namespace ic
