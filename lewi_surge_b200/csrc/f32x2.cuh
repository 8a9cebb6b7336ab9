// Pairs of floats in one instruction (sm_100 works on two with one issue).
#pragma once

#include "common.cuh"

namespace lewi {

// Two floats side by side (fma.rn.f32x2: each half rounded as a single fma).
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_split(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ uint32_t f2_bf16(F2 a) {
  float lo, hi;
  f2_split(a, lo, hi);
  return pack_bf16(lo, hi);
}

// 2^x by the special function unit (relative error below 2^-22; results below 2^-126 are zero)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x of both halves by fused multiply-adds, for x < 128: n = x rounded to the nearest integer (it falls out of the low bits of x + 1.5 2^23),
// 2^(x - n) by the polynomial of degree 4 with the smallest largest relative error on [-1/2, 1/2] (2.6e-6; found by linear programming
// on the Chebyshev points), 2^n from its bits.  Below -126.5 zero, also for -inf; NaN stays NaN.
__device__ __forceinline__ F2 ex2_poly(F2 x) {
  constexpr float kShift = 12582912.f + 127.f;   // (low bits: n + 127, the exponent field of 2^n)
  float lo, hi;
  f2_split(x, lo, hi);
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(lo));   // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(hi));
  x = f2(lo, hi);
  const F2 t = add2(x, f2(kShift, kShift));
  const F2 f = fma2(add2(t, f2(-kShift, -kShift)), f2(-1.f, -1.f), x);
  F2 p = fma2(f, f2(0.009570531136513637f, 0.009570531136513637f), f2(0.05591866219782843f, 0.05591866219782843f));
  p = fma2(f, p, f2(0.24024735557044632f, 0.24024735557044632f));
  p = fma2(f, p, f2(0.6931216461644981f, 0.6931216461644981f));
  p = fma2(f, p, f2(0.9999992631127679f, 0.9999992631127679f));
  f2_split(t, lo, hi);
  return mul2(p, f2(__uint_as_float(__float_as_uint(lo) << 23), __uint_as_float(__float_as_uint(hi) << 23)));
}

}  // namespace lewi
