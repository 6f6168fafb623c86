// What becomes of a score, shared by the attention kernels of a text stage.
//   s = scale q.k;  s = cap tanh(s / cap);  s += -slope |away|  or  distance[clamp(away, -R, R) + R],  away = key - query position
// Everything is kept in units of log2: x = s log2(e), so that a probability is one exp2 of a difference.
#pragma once

#include "attn_common.h"

namespace odit {

constexpr float kLog2e = 1.4426950408889634f;

// The tanh is 1 - 2 / (1 + e^(2y)): one exp2 and one reciprocal, of 1 ulp each, for any y (infinite ones give -1 and 1). Its error is about
// 2^-23, so a capped score's is 2^-23 of the cap: kMaxCap keeps that below what a probability's rounding to 16 bits loses.
constexpr float kMaxCap = 8192.f;
struct Cap {
  float in, out;  // 2 log2(e) scale / cap and cap log2(e)
  __device__ __forceinline__ float operator()(float s) const {
    const float r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * in));
    return fmaf(-2.f * out, r, out);
  }
};

constexpr int kMaxRadius = 1024;  // distances with a bias of their own, either way

}  // namespace odit
