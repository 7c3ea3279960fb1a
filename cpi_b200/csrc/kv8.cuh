// The cache in 8 bits: what a block of 64 positions of one key/value head is held as.
//
// A block that is complete is 64 x D codes of 8 bits and one scale s, a power of two; an element stands for code * s.
//   int8   s = the smallest power of two with max |x| <= 127 s, code = x / s rounded to the nearest integer (ties to even)
//   e4m3   max |x| / s lies in [128, 256), code = x / s rounded to the nearest e4m3 number (ties to even)
// With a power of two x / s is exact, so the codes are the same in any arithmetic, and code * s (at most 7 significant bits) is
// exact in bfloat16: the rounding to a code is the only one.  It costs int8 half a bit on average beside a scale of max / 127;
// e4m3 nothing.  s lies between 2^-60 and 2^60 (a block of zeros has 2^-60).  Numbers that are not finite do not enter the
// maximum: an infinity is held as the largest code, a NaN as e4m3's NaN or int8's 0 (its own query met it in bfloat16).
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace cpi {
namespace kv8 {

constexpr int PAGE = 64;                  // positions of a block, and of a page of the cache
enum Format : int { kInt8 = 0, kE4m3 = 1 };

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127
// Exponent of the scale for a block whose largest finite magnitude is `top` (a bfloat16 number).
template <int FMT> __device__ __forceinline__ int scale_exponent(float top) {
  if (!(top > 0.f)) return -60;
  const int e = ilogbf(top) + 1;                            // top < 2^e, top >= 2^(e - 1)
  int r;
  if (FMT == kInt8) r = e - 7 + (top > 127.f * power_of_two(max(e - 7, -120)) ? 1 : 0);
  else r = e - 8;
  return min(60, max(-60, r));
}

// Largest finite magnitude among the eight bfloat16 numbers of a vector, as bits (they order like the magnitudes).
__device__ __forceinline__ uint32_t top_of(uint4 v) {
  uint32_t m = 0;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
    m = max(m, lo < 0x7f80u ? lo : 0u);
    m = max(m, hi < 0x7f80u ? hi : 0u);
  }
  return m;
}
__device__ __forceinline__ float lo_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f32(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Two numbers, already divided by the scale, as two codes (the first in the low byte).
template <int FMT> __device__ __forceinline__ uint32_t codes2(float a, float b) {
  if (FMT == kInt8) {
    const int x = min(127, max(-127, __float2int_rn(a))), y = min(127, max(-127, __float2int_rn(b)));
    return (uint32_t)(x & 0xff) | ((uint32_t)(y & 0xff) << 8);
  }
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));      // (the second operand is the low byte)
  return r;
}
// Two e4m3 codes (low half of `w`) as two float16 numbers, exactly.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint16_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
  return r;
}
// Eight bfloat16 numbers as eight codes.
template <int FMT> __device__ __forceinline__ uint2 codes8(uint4 v, float inv) {
  const uint32_t a = codes2<FMT>(lo_f32(v.x) * inv, hi_f32(v.x) * inv), b = codes2<FMT>(lo_f32(v.y) * inv, hi_f32(v.y) * inv);
  const uint32_t c = codes2<FMT>(lo_f32(v.z) * inv, hi_f32(v.z) * inv), d = codes2<FMT>(lo_f32(v.w) * inv, hi_f32(v.w) * inv);
  return make_uint2(a | (b << 16), c | (d << 16));
}
// Four codes as the four numbers they stand for, in bfloat16 (exact).
template <int FMT> __device__ __forceinline__ uint2 values4(uint32_t w, float s) {
  float x[4];
  if (FMT == kInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i)) * s;
  } else {
    const uint32_t a = e4m3x2_f16x2((uint16_t)w), b = e4m3x2_f16x2((uint16_t)(w >> 16));
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&a)), q = __half22float2(*reinterpret_cast<const __half2*>(&b));
    x[0] = p.x * s; x[1] = p.y * s; x[2] = q.x * s; x[3] = q.y * s;
  }
  __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
  return make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
}

}  // namespace kv8
}  // namespace cpi
