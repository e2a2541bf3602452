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

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kGeluC2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// ---- fp32 results: one value at a time, accurate exponential and logarithm ----------------
__device__ __forceinline__ float sigmoid1(float t) { return 1.f / (1.f + expf(-t)); }

template <int ACT>
__device__ __forceinline__ float act_value1(float z, float gamma) {
  if constexpr (ACT == kActRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if constexpr (ACT == kActSilu) return z * sigmoid1(z);
  if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    const float g = z * sigmoid1(z * (kGeluC2 + kGeluC2 * kGeluA * (z * z)));
    if constexpr (ACT == kActGeluTanh) return g;
    return g + gamma * (z > 20.f ? z : log1pf(expf(z)));
  }
  return z;
}

template <int ACT>
__device__ __forceinline__ void act_grad1(float z, float gamma, float& a, float& d) {
  if constexpr (ACT == kActRelu) {
    a = z < 0.f ? 0.f : z;
    d = z <= 0.f ? 0.f : 1.f;  // NaN hands the gradient on, as the value stays NaN
  } else if constexpr (ACT == kActSilu) {
    const float s = sigmoid1(z);
    a = z * s;
    d = s + a * (1.f - s);
  } else if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    // far out s (1 - s) is 0: the bound keeps 0 * z^2 from becoming 0 * infinity
    const float z2 = fminf(z * z, 1e30f);
    const float s = sigmoid1(z * (kGeluC2 + kGeluC2 * kGeluA * z2));
    a = z * s;
    d = s + a * (1.f - s) * (kGeluC2 + 3.f * kGeluA * kGeluC2 * z2);
    if constexpr (ACT == kActEra) {
      a += gamma * (z > 20.f ? z : log1pf(expf(z)));
      d += gamma * (z > 20.f ? 1.f : sigmoid1(z));
    }
  } else {
    a = z;
    d = 1.f;
  }
}

// ---- bf16 results: two values at a time (sm_100's packed fp32 multiply-adds) --------------
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

__device__ __forceinline__ uint64_t bits2(float2 v) {
  return static_cast<uint64_t>(__float_as_uint(v.x)) |
         static_cast<uint64_t>(__float_as_uint(v.y)) << 32;
}
__device__ __forceinline__ float2 pair_of(uint64_t b) {
  return make_float2(__uint_as_float(static_cast<uint32_t>(b)),
                     __uint_as_float(static_cast<uint32_t>(b >> 32)));
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair_of(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair_of(d);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 ex2_2(float2 v) { return make_float2(ex2_fast(v.x), ex2_fast(v.y)); }
__device__ __forceinline__ float2 rcp_2(float2 v) { return make_float2(rcp_fast(v.x), rcp_fast(v.y)); }
__device__ __forceinline__ float2 min_2(float2 v, float m) {
  return make_float2(fminf(v.x, m), fminf(v.y, m));
}

// s(2q) from z and z^2
__device__ __forceinline__ float2 gelu_gate2(float2 z, float2 z2) {
  const float2 p = fma2(both(-kLog2e * kGeluC2 * kGeluA), z2, both(-kLog2e * kGeluC2));
  return rcp_2(add2(ex2_2(mul2(z, p)), both(1.f)));
}

// softplus from e = e^min(z, 60): log(1 + e), and z where that is larger (beyond 60)
__device__ __forceinline__ float2 softplus2(float2 z, float2 e1) {
  const float2 l = mul2(make_float2(lg2_fast(e1.x), lg2_fast(e1.y)), both(kLn2));
  return make_float2(fmaxf(l.x, z.x), fmaxf(l.y, z.y));
}
__device__ __forceinline__ float2 exp_bounded2(float2 z) {
  return ex2_2(min_2(mul2(z, both(kLog2e)), 60.f * kLog2e));
}

template <int ACT>
__device__ __forceinline__ float2 act_value2(float2 z, float gamma) {
  if constexpr (ACT == kActRelu) {
    return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y);
  } else if constexpr (ACT == kActSilu) {
    return mul2(z, rcp_2(add2(ex2_2(mul2(z, both(-kLog2e))), both(1.f))));
  } else if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    const float2 g = mul2(z, gelu_gate2(z, mul2(z, z)));
    if constexpr (ACT == kActGeluTanh) return g;
    return fma2(both(gamma), softplus2(z, add2(exp_bounded2(z), both(1.f))), g);
  } else {
    return z;
  }
}

// act(z) and act'(z)
template <int ACT>
__device__ __forceinline__ void act_grad2(float2 z, float gamma, float2& a, float2& d) {
  if constexpr (ACT == kActRelu) {
    a = act_value2<kActRelu>(z, gamma);
    d = make_float2(z.x <= 0.f ? 0.f : 1.f, z.y <= 0.f ? 0.f : 1.f);
  } else if constexpr (ACT == kActSilu) {
    const float2 s = rcp_2(add2(ex2_2(mul2(z, both(-kLog2e))), both(1.f)));
    a = mul2(z, s);
    d = fma2(a, fma2(s, both(-1.f), both(1.f)), s);
  } else if constexpr (ACT == kActGeluTanh || ACT == kActEra) {
    const float2 z2 = min_2(mul2(z, z), 1e30f);  // as in act_grad1
    const float2 s = gelu_gate2(z, z2);
    a = mul2(z, s);
    const float2 m = mul2(a, fma2(s, both(-1.f), both(1.f)));
    d = fma2(m, fma2(both(3.f * kGeluA * kGeluC2), z2, both(kGeluC2)), s);
    if constexpr (ACT == kActEra) {
      const float2 e = exp_bounded2(z);
      const float2 e1 = add2(e, both(1.f));
      a = fma2(both(gamma), softplus2(z, e1), a);
      d = fma2(both(gamma), mul2(e, rcp_2(e1)), d);
    }
  } else {
    a = z;
    d = both(1.f);
  }
}

// v act'(z), where d is act'(z): what relu cuts off is 0 though v be infinite or NaN
template <int ACT>
__device__ __forceinline__ float times_slope(float v, float d) {
  if constexpr (ACT == kActRelu) return d == 0.f ? 0.f : v;
  return v * d;
}
template <int ACT>
__device__ __forceinline__ float2 times_slope2(float2 v, float2 d) {
  if constexpr (ACT == kActRelu)
    return make_float2(times_slope<ACT>(v.x, d.x), times_slope<ACT>(v.y, d.y));
  return mul2(v, d);
}

// v[i] = act(v[i]); N even
template <bool kFast, int ACT, int N>
__device__ __forceinline__ void act_values(float (&v)[N], float gamma) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    if constexpr (kFast) {
      const float2 a = act_value2<ACT>(make_float2(v[j], v[j + 1]), gamma);
      v[j] = a.x;
      v[j + 1] = a.y;
    } else {
      v[j] = act_value1<ACT>(v[j], gamma);
      v[j + 1] = act_value1<ACT>(v[j + 1], gamma);
    }
  }
}

// z becomes act(z), d act'(z)
template <bool kFast, int ACT, int N>
__device__ __forceinline__ void act_grads(float (&z)[N], float (&d)[N], float gamma) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    if constexpr (kFast) {
      float2 a, e;
      act_grad2<ACT>(make_float2(z[j], z[j + 1]), gamma, a, e);
      z[j] = a.x;
      z[j + 1] = a.y;
      d[j] = e.x;
      d[j + 1] = e.y;
    } else {
      float a0, a1;
      act_grad1<ACT>(z[j], gamma, a0, d[j]);
      act_grad1<ACT>(z[j + 1], gamma, a1, d[j + 1]);
      z[j] = a0;
      z[j + 1] = a1;
    }
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
