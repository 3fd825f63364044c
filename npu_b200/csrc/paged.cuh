// What the kernels over packed tokens and a paged cache share: the sequence of a
// token, and the 8-bit form of a cached row.
//
// 8-bit rows (one token's k or v of one KV head): with a = max |y_i|,
//   s = max(a / 448, 2^-100),  c_i = e4m3(y_i r), r = 1 / s,  read back as c_i s,
// s and r rounded to fp32 (a product for each value and one quotient a row; y_i / s
// would differ where it lies within 2^-23 of the middle of two codes).
// 448 is the largest e4m3 value, and what r's rounding adds to it is rounded away, so
// nothing saturates; e4m3 keeps 4 significant bits of c_i >= 2^-6 and steps of 2^-9
// below, so a value is off by at most 2^-4 of itself or 2^-10 s (and 2^-23 of that). One scale a row and not one a page: rows are
// written one by one, and a page's scale would change under those already
// there. The floor 2^-100 keeps 1 / s finite for rows of (nearly) zeros. A row
// with an infinity or a NaN has the scale NaN and reads back as NaN throughout.
#pragma once

#include "common.cuh"

namespace b2a {

constexpr float kE4m3Max = 448.f;
constexpr float kE4m3SmallestScale = 7.888609052210118e-31f;  // 2^-100
constexpr float kE4m3LargestVScale = 1.2379400392853803e+27f;  // 2^90

// The sequence that owns token n: the largest b with cu[b] <= n (0 when there
// is none), by a search that narrows 32-fold per step. Warp-collective.
__device__ __forceinline__ int find_sequence(const int* cu, int B, long long n) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = B;
  while (len > 1) {
    const int step = (len + 31) / 32;
    const int at = lo + lane * step;
    const bool before = lane * step < len && (lane == 0 || cu[at] <= n);
    const unsigned m = __ballot_sync(0xffffffffu, before);
    const int hit = 31 - __clz(m);
    len = min(step, len - hit * step);
    lo += hit * step;
  }
  return lo;
}

// Whether offsets c0 and c1 are a stretch of N tokens.
__device__ __forceinline__ bool is_stretch(int c0, int c1, long long N) { return c0 >= 0 && c1 >= c0 && c1 <= N; }

// Four floats as e4m3, rounded to nearest even, the first in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Two e4m3 numbers as f16, which holds them all: the low byte's in the low half.
__device__ __forceinline__ uint32_t f16_of_e4m3(uint16_t x) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
  return r;
}
__device__ __forceinline__ float2 unpack_f16x2(uint32_t x) {
  float2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(x));
  return r;
}

// |x| as an integer of the same order, in which infinities and NaN are largest.
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of a row whose largest magnitude is m.
__device__ __forceinline__ float e4m3_scale(unsigned m) {
  if (m >= 0x7f800000u) return __uint_as_float(0x7fffffffu);  // NaN
  const float s = __fdiv_rn(__uint_as_float(m), kE4m3Max);
  return s < kE4m3SmallestScale ? kE4m3SmallestScale : s;
}

// A scale of V as attention takes it: none below the smallest, and NaN in place of
// one whose reciprocal its sums have no room for (values above 5e29).
__device__ __forceinline__ float e4m3_scale_in_range(float s) {
  s = s > kE4m3LargestVScale ? __uint_as_float(0x7fffffffu) : s;
  return s < kE4m3SmallestScale ? kE4m3SmallestScale : s;  // NaN stays
}

}  // namespace b2a
