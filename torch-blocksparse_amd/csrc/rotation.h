// Angles of rotated positions (rotation.hip, and the caches that rotate what they are given: cache.hip, latent_cache.hip).
//
// Pair p of a row at position t is turned by the angle t * f_p.  A frequency is held as the fraction f / (2 pi) of a turn, less its whole turns, in units of
// 2^-64: position times fraction, where whole turns leave the 64 bits by themselves, is the fraction of the angle.  It is off by |t| 2^-65 of a turn, 2^-34 for
// the farthest position of 32 bits, so no angle is ever large and none is reduced.  What is left is a quarter turn's number and an angle of at most pi / 4, whose sine and
// cosine are the first terms of their series: the terms left out are below 2^-29 (angles in fp32) and 2^-54 (fp64).
#ifndef BSP_ROTATION_H
#define BSP_ROTATION_H
#include "bsp_common.h"

namespace bsp {

struct Turn { float cos, sin; };
struct TurnF64 { double cos, sin; };

// sine and cosine of x, |x| <= pi / 4, and `quarters` quarter turns
template <typename F> __device__ __forceinline__ void quarter_turns(uint32_t quarters, F s, F c, F &cos, F &sin) {
  const F x = quarters & 1 ? s : c, y = quarters & 1 ? c : s;
  cos = (quarters + 1) & 2 ? -x : x;
  sin = quarters & 2 ? -y : y;
}

__device__ __forceinline__ Turn turn_of(int32_t position, uint64_t fraction) {
  const uint64_t turns = (uint64_t)(int64_t)position * fraction;
  const uint32_t t = (uint32_t)((turns + 0x80000000u) >> 32), quarters = (t + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(t - (quarters << 30)) * (6.283185307179586f * 0x1p-32f), z = x * x;
  float s = fmaf(z, 1.f / 362880.f, -1.f / 5040.f), c = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  s = fmaf(z, s, 1.f / 120.f);
  c = fmaf(z, c, -1.f / 720.f);
  s = fmaf(z, s, -1.f / 6.f);
  c = fmaf(z, c, 1.f / 24.f);
  c = fmaf(z, c, -0.5f);
  Turn r;
  quarter_turns(quarters, fmaf(x * z, s, x), fmaf(z, c, 1.f), r.cos, r.sin);
  return r;
}

__device__ __forceinline__ TurnF64 turn_of_f64(int32_t position, uint64_t fraction) {
  const uint64_t turns = (uint64_t)(int64_t)position * fraction, quarters = (turns + ((uint64_t)1 << 61)) >> 62;
  const double x = (double)(int64_t)(turns - (quarters << 62)) * (6.283185307179586476925 * 0x1p-64), z = x * x;
  // 1 / 3!, 1 / 5!, .. 1 / 17! and 1 / 2!, .. 1 / 16!, alternating
  double s = 1. / 355687428096000., c = 1. / 20922789888000.;
  constexpr double sines[] = {-1. / 1307674368000., 1. / 6227020800., -1. / 39916800., 1. / 362880., -1. / 5040., 1. / 120., -1. / 6.};
  constexpr double cosines[] = {-1. / 87178291200., 1. / 479001600., -1. / 3628800., 1. / 40320., -1. / 720., 1. / 24., -0.5};
#pragma unroll
  for (int i = 0; i < 7; i++) {
    s = fma(z, s, sines[i]);
    c = fma(z, c, cosines[i]);
  }
  TurnF64 r;
  quarter_turns((uint32_t)quarters, fma(x * z, s, x), fma(z, c, 1.), r.cos, r.sin);
  return r;
}

// (a, b) turned, in fp32 and rounded once to T.  (The compiler may take a multiply-add and the conversion to float16 as one operation, which rounds once less, here and
// not there: all kernels are to give the same numbers.)
template <typename T> __device__ __forceinline__ void turn_pair(float a, float b, float cos, float sin, T &x, T &y) {
  float u = fmaf(a, cos, -b * sin), v = fmaf(a, sin, b * cos);
  if constexpr (__is_same(T, f16)) asm("" : "+v"(u), "+v"(v));
  x = from_float<T>(u);
  y = from_float<T>(v);
}

// what a rotation is given as: pairs 2 i and 2 i + 1 (neighbours) or i and pairs + i
inline bool rotation_ok(const void *fractions, int pairs, int D) { return fractions && !(reinterpret_cast<uintptr_t>(fractions) & 7) && pairs > 0 && pairs % 8 == 0 && 2 * pairs <= D; }

}  // namespace bsp
#endif
