// What becomes of a score, shared by the attention kernels of a text stage.
//   s = scale q.k;  s = cap tanh(s / cap);  s += -slope |away|  or  distance[clamp(away, -R, R) + R],  away = key - query position
// Everything is kept in units of log2: x = s log2(e), so that a probability is one exp2 of a difference.
#pragma once

#include "attn_common.h"

namespace odit {

constexpr float kLog2e = 1.4426950408889634f;

// The tanh is 1 - 2 / (1 + e^(2y)): one exp2 and one reciprocal, of 1 ulp each, for any y (infinite ones give -1 and 1). Its error is up to
// 2^-21 (3/2 ulp of the quotient near 1, twice), and a capped score's that of the cap, whatever the score: up to kPlainCap it is half of what
// a probability's rounding to fp16 loses, 2^-11.
// For |y| <= 1/2, where a cap leaves most scores, y times a polynomial in y^2 does, the best one in the largest error (a linear
// programme over 4000 places; 2^-22.9): four instructions at full rate where those two alone take as long as eight.
// Larger caps leave common scores where the difference has lost most of its digits. There y times a polynomial of relative error 2^-26 has them up to 1/2
// (the best such one, likewise), and 1 - 2 e / (1 + e) with e = e^(-2|y|) beyond, so that the error is 2^-21 of the score: what a sum of products has too.
constexpr float kMaxCap = 8192.f, kPlainCap = 512.f;
constexpr float kMinScale = 1e-9f, kMaxScale = 1e9f;  // of scales (and the least cap): their quotients and products with log2(e) are fp32 numbers
struct Cap {
  float in, out;     // of the exact form: 2 log2(e) scale / cap and cap log2(e)
  float few;         // products below this in size are small enough for the polynomial (0: none)
  float c0, c1, c2, c3;  // the capped score in units of log2 is s (c0 + c1 s^2 + c2 s^4 + c3 s^6)
  float y;           // scale / cap
  bool large;        // past kPlainCap
  // product -> capped score in units of log2
  __device__ __forceinline__ float operator()(float s) const {
    const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * in));
    return fmaf(-2.f * out, r, out);
  }
  __device__ __forceinline__ float of_large(float s) const {
    const float e = __builtin_amdgcn_exp2f(-fabsf(s * in)), t = s * y, z = t * t;
    const float beyond = copysignf(fmaf(-2.f * e, __builtin_amdgcn_rcpf(1.f + e), 1.f), t);
    const float near = t * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 0.01713485492f, -0.05298604946f), 0.1332477994f), -0.3333306951f), 0.9999999869f);
    return out * (fabsf(t) >= 0.5f ? beyond : near);  // (NaN stays NaN)
  }
  __device__ __forceinline__ float of_any(float s) const { return large ? of_large(s) : (*this)(s); }
};
inline Cap make_cap(float cap, float scale) {
  Cap c{};
  if (!(cap > 0.f)) return c;
  const double y = static_cast<double>(scale) / cap, out = static_cast<double>(cap) * kLog2e;  // y: of a product of 1
  c.in = static_cast<float>(2.0 * kLog2e * y);
  c.out = static_cast<float>(out);
  c.y = static_cast<float>(y);
  c.large = cap > kPlainCap;
  c.few = y > 1e-4 && y < 1e4 && !c.large ? static_cast<float>(0.5 / y) : 0.f;  // (the polynomial's terms stay far from both ends of fp32)
  c.c0 = static_cast<float>(out * y * 0.9999976762);
  c.c1 = static_cast<float>(out * y * y * y * -0.3332065521);
  c.c2 = static_cast<float>(out * y * y * y * y * y * 0.1314514561);
  c.c3 = static_cast<float>(out * y * y * y * y * y * y * y * -0.04337248238);
  return c;
}

// A bias (or a slope) in the units that it is added in: a finite one stays finite, as the least float32 forbids a key beside others and no more
__device__ __forceinline__ float in_units(float x, float unit) {
  const float y = x * unit;
  return fabsf(y) == INFINITY && fabsf(x) < INFINITY ? copysignf(3.402823466e38f, y) : y;
}

constexpr int kMaxRadius = 1024;  // distances with a bias of their own, either way

}  // namespace odit
