// Activations of the dense operators and their derivatives, in fp32.
//
// With s(t) = 1 / (1 + e^-t):
//   silu(z) = z s(z)                        silu' = s + z s (1 - s)
//   gelu_tanh(z) = z s(2q),  q = sqrt(2/pi) (z + a z^3), a = 0.044715: the tanh form
//   0.5 z (1 + tanh q) rewritten so that its negative tail keeps its relative accuracy
//                                           gelu' = s + z s (1 - s) 2 sqrt(2/pi) (1 + 3 a z^2)
//   era(z) = gelu_tanh(z) + gamma softplus(z)     (softplus is z above 20, as torch's)
//   era' = gelu' + gamma s(z)
// kFast is for results that are rounded to bf16: the hardware's approximate exponential,
// reciprocal and logarithm, relative errors of 2^-21 or so.  Near 1 the logarithm's error is
// absolute, 2^-22: softplus below 2^-14 has fewer correct bits than bf16, by less than 2^-22.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "dense.h"

namespace vmoe {

__device__ __forceinline__ float ex2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kGeluC2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

template <bool kFast>
__device__ __forceinline__ float act_sigmoid(float t) {
  if constexpr (kFast) return rcp_fast(1.f + ex2_fast(-kLog2e * t));
  return 1.f / (1.f + expf(-t));
}

// s(2q) from z and z^2
template <bool kFast>
__device__ __forceinline__ float gelu_gate(float z, float z2) {
  if constexpr (kFast)
    return rcp_fast(1.f + ex2_fast(z * fmaf(-kLog2e * kGeluC2 * kGeluA, z2, -kLog2e * kGeluC2)));
  return 1.f / (1.f + expf(-(z * (kGeluC2 + kGeluC2 * kGeluA * z2))));
}

template <bool kFast, int ACT>
__device__ __forceinline__ float act_value(float z, float gamma) {
  if constexpr (ACT == kActRelu) {
    return z < 0.f ? 0.f : z;  // NaN stays NaN
  } else if constexpr (ACT == kActSilu) {
    return z * act_sigmoid<kFast>(z);
  } else if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    const float g = z * gelu_gate<kFast>(z, z * z);
    if constexpr (ACT == kActGeluTanh) {
      return g;
    } else if constexpr (kFast) {
      const float sp = kLn2 * lg2_fast(1.f + ex2_fast(kLog2e * fminf(z, 20.f)));
      return fmaf(gamma, z > 20.f ? z : sp, g);
    } else {
      return g + gamma * (z > 20.f ? z : log1pf(expf(z)));
    }
  } else {
    return z;
  }
}

// act(z) and act'(z)
template <bool kFast, int ACT>
__device__ __forceinline__ void act_grad(float z, float gamma, float& a, float& d) {
  if constexpr (ACT == kActRelu) {
    a = z < 0.f ? 0.f : z;
    d = z > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == kActSilu) {
    const float s = act_sigmoid<kFast>(z);
    a = z * s;
    d = fmaf(a, 1.f - s, s);
  } else if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    // far out s (1 - s) is 0: the bound keeps 0 * z^2 from becoming 0 * infinity
    const float z2 = fminf(z * z, 1e30f);
    const float s = gelu_gate<kFast>(z, z2);
    a = z * s;
    d = fmaf(a * (1.f - s), fmaf(3.f * kGeluA * kGeluC2, z2, kGeluC2), s);
    if constexpr (ACT == kActEra) {
      if constexpr (kFast) {  // e^z / (1 + e^z) is 1 in fp32 from 20 on
        const float e = ex2_fast(kLog2e * fminf(z, 20.f));
        const float sp = kLn2 * lg2_fast(1.f + e);
        a = fmaf(gamma, z > 20.f ? z : sp, a);
        d = fmaf(gamma, e * rcp_fast(1.f + e), d);
      } else {
        a += gamma * (z > 20.f ? z : log1pf(expf(z)));
        d += gamma * (z > 20.f ? 1.f : act_sigmoid<false>(z));
      }
    }
  } else {
    a = z;
    d = 1.f;
  }
}

// Calls f with the activation as a compile-time constant (one uniform branch per chunk).
template <typename F>
__device__ __forceinline__ void act_switch(int act, F&& f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActEra: f(std::integral_constant<int, kActEra>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
  }
}

// N consecutive elements of a row from p, `valid` of them inside (the rest read as 0);
// 16-byte accesses where `vec` allows them.
template <int N, typename T>
__device__ __forceinline__ void load_row(const T* p, float (&v)[N], int64_t valid, bool vec) {
  constexpr int V = Vec16<T>::N;
#pragma unroll
  for (int i = 0; i < N; i += V) {
    if (vec && valid >= i + V) {
      load16_to_f(p + i, v + i);
    } else {
#pragma unroll
      for (int j = i; j < i + V; ++j) v[j] = j < valid ? Elt<T>::to_f(p[j]) : 0.f;
    }
  }
}

template <int N, typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[N], int64_t valid, bool vec) {
  constexpr int V = Vec16<T>::N;
#pragma unroll
  for (int i = 0; i < N; i += V) {
    if (vec && valid >= i + V) {
      store16_from_f(p + i, v + i);
    } else {
#pragma unroll
      for (int j = i; j < i + V; ++j)
        if (j < valid) p[j] = Elt<T>::from_f(v[j]);
    }
  }
}

}  // namespace vmoe
