// Sigmoids of pairs of fp32 values in packed arithmetic.
#pragma once
#include "common.cuh"
#include "tma.cuh"

namespace mega {

// NaN stays NaN
__device__ __forceinline__ float within(float v, float most) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(most));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(-most));
  return v;
}

// e^(kSign v), for minus_over_one_and.
// 16-bit types: as 2^(v / ln 2) with the product rounded once, relative error (2 + |v|) 2^-23.  fp32: the product's rounding error
// r and the constant's own are taken along, 2^(p + r) = 2^p (1 + r ln 2), which leaves the approximation's 2^-22 whatever v is;
// expf and the division cost three times as many instructions (gates are most of what a step of the recurrence computes: B = 16,
// L = 2048, D = 1024 forward 82 us with them, 67 without).  There v is held within 88, where e^v is finite and r means something.
template <typename T, int kSign>
__device__ __forceinline__ f32x2 exp_pair(f32x2 v) {
  constexpr float kLog = kSign * 1.4426950408889634f;   // 1 / ln 2 in fp32; what is missing of it times ln 2 below
  constexpr float kRest = kSign * (float)((1.4426950408889634074 - (double)1.4426950408889634f) * 0.69314718055994530942);
  float a, b;
  f32x2 u = 0;
  if (sizeof(T) == 4) {
    unpack2(v, a, b);
    v = pack2(within(a, 88.f), within(b, 88.f));
    const f32x2 r = fma2(v, pack2(kLog, kLog), mul2(v, pack2(-kLog, -kLog)));
    u = fma2(v, pack2(kRest, kRest), mul2(r, pack2(0.6931471805599453f, 0.6931471805599453f)));
  }
  unpack2(mul2(v, pack2(kLog, kLog)), a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  return sizeof(T) == 4 ? fma2(pack2(a, b), u, pack2(a, b)) : pack2(a, b);
}

// -1 / (1 + e), by the approximate reciprocal (relative 2^-23; 0 where the result is below 2^-126)
__device__ __forceinline__ f32x2 minus_over_one_and(f32x2 e) {
  float a, b;
  unpack2(fma2(e, pack2(-1.f, -1.f), pack2(-1.f, -1.f)), a, b);
  return pack2(rcp_approx(a), rcp_approx(b));
}

// minus the sigmoid of -kSign v
template <typename T, int kSign>
__device__ __forceinline__ f32x2 minus_sigmoid2(f32x2 v) {
  return minus_over_one_and(exp_pair<T, kSign>(v));
}

// The sides of a gate, sigmoid(v) and sigmoid(-v), are held as the smaller of them, g <= 1/2, to its last places: the other is
// 1 - g to its own.  v >= 0: c = -g = -sigmoid(-v); v < 0: c = g = sigmoid(v).
template <typename T>
__device__ __forceinline__ f32x2 gate_side2(f32x2 v) {
  const f32x2 e = exp_pair<T, 1>(v | 0x8000000080000000ull);   // e^-|v|
  return mul2(e, minus_over_one_and(e)) ^ (v & 0x8000000080000000ull);
}
// all bits where c says v >= 0 (by its sign: g may be 0)
__device__ __forceinline__ f32x2 open_bits(f32x2 c) {
  float a, b;
  unpack2(c, a, b);
  return pack2(__int_as_float(__float_as_int(a) >> 31), __int_as_float(__float_as_int(b) >> 31));
}
__device__ __forceinline__ f32x2 either(f32x2 bits, f32x2 a, f32x2 b) { return (a & bits) | (b & ~bits); }
// u sigmoid(v) and u sigmoid(-v): u + c u and c u, or c u and u + c u
__device__ __forceinline__ f32x2 pass(f32x2 c, f32x2 open, f32x2 u) { return fma2(c, u, u & open); }
__device__ __forceinline__ f32x2 hold_back(f32x2 c, f32x2 open, f32x2 u) { return fma2(c ^ 0x8000000080000000ull, u, u & ~open); }

}  // namespace mega
