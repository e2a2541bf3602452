// Activations of the dense operators and their derivatives, in fp32.
//
// With s(t) = 1 / (1 + e^-t):
//   silu(z) = z s(z)                        silu' = s + z s (1 - s)
//   gelu_tanh(z) = z s(2q),  q = sqrt(2/pi) (z + a z^3), a = 0.044715: the tanh form
//   0.5 z (1 + tanh q) rewritten so that its negative tail keeps its relative accuracy
//                                           gelu' = s + z s (1 - s) 2 sqrt(2/pi) (1 + 3 a z^2)
//   era(z) = gelu_tanh(z) + gamma softplus(z)     (softplus is z above 20, as torch's)
//   era' = gelu' + gamma s(z)
// kFast uses the hardware's approximate exponential, logarithm and division (relative error
// about 2^-21): its results are rounded to bf16.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "dense.h"

namespace vmoe {

template <bool kFast>
__device__ __forceinline__ float act_sigmoid(float t) {
  if constexpr (kFast) return __fdividef(1.f, 1.f + __expf(-t));
  return 1.f / (1.f + expf(-t));
}

// log(1 + e^z) for z <= 20.  The fast form takes log(1 + e) from the series below e = 2^-6
// (relative error under 2^-24), where the approximate logarithm near 1 would lose it.
template <bool kFast>
__device__ __forceinline__ float act_softplus(float z) {
  if constexpr (!kFast) {
    return z > 20.f ? z : log1pf(expf(z));
  } else {
    const float e = __expf(fminf(z, 20.f));
    const float series = e * (1.f - e * (0.5f - e * (1.f / 3.f - e * 0.25f)));
    const float l = e < 0.015625f ? series : __logf(1.f + e);
    return z > 20.f ? z : l;
  }
}

constexpr float kGeluC2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

template <bool kFast, int ACT>
__device__ __forceinline__ float act_value(float z, float gamma) {
  if constexpr (ACT == kActRelu) {
    return z < 0.f ? 0.f : z;  // NaN stays NaN
  } else if constexpr (ACT == kActSilu) {
    return z * act_sigmoid<kFast>(z);
  } else if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    const float g = z * act_sigmoid<kFast>(kGeluC2 * (z + kGeluA * z * z * z));
    if constexpr (ACT == kActEra) return g + gamma * act_softplus<kFast>(z);
    return g;
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
    d = s * (1.f + z * (1.f - s));
  } else if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    const float s = act_sigmoid<kFast>(kGeluC2 * (z + kGeluA * z * z * z));
    a = z * s;
    // s (1 - s) is 0 in fp32 beyond |z| = 20; the clamp keeps 0 * z^2 from overflowing to NaN
    const float c = fminf(fmaxf(z, -20.f), 20.f);
    d = s + c * s * (1.f - s) * kGeluC2 * (1.f + 3.f * kGeluA * c * c);
    if constexpr (ACT == kActEra) {
      a += gamma * act_softplus<kFast>(z);
      d += gamma * (z > 20.f ? 1.f : act_sigmoid<kFast>(z));
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
