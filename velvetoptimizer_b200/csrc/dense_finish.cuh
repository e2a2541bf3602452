// A split product's chunk of 8 columns of a row: its sum over the splits, in split order, and its
// epilogue.
#pragma once

#include "common.cuh"
#include "dense.h"
#include "dense_act.cuh"

namespace vmoe {

constexpr int kChunk = 8;

// a product's partials: from one split to the next, and column col of a row (gated: the gate's)
__device__ __forceinline__ int64_t split_stride(const DenseGemm& g) {
  return static_cast<int64_t>(g.groups) * g.M * g.ldp;
}
template <int EPI>
__device__ __forceinline__ float* partial_at(const DenseGemm& g, int grp, int64_t row, int64_t col) {
  const int64_t pcol = EPI == kEpiGated ? (col / 128) * 256 + (col & 127) : col;
  return g.partial + (static_cast<int64_t>(grp) * g.M + row) * g.ldp + pcol;
}

// 8 partials; from L2 where another block of this kernel may have written them
template <bool L2>
__device__ __forceinline__ void load_chunk(const float* p, float (&t)[kChunk]) {
#pragma unroll
  for (int i = 0; i < kChunk; i += 4) {
    const float4 q = L2 ? __ldcg(reinterpret_cast<const float4*>(p + i))
                        : *reinterpret_cast<const float4*>(p + i);
    t[i] = q.x;
    t[i + 1] = q.y;
    t[i + 2] = q.z;
    t[i + 3] = q.w;
  }
}

// v, and for a gated product u (the up columns)
template <int EPI, bool L2 = false>
__device__ __forceinline__ void chunk_sums(const DenseGemm& g, int grp, int64_t row, int64_t col,
                                           float (&v)[kChunk], float (&u)[kChunk]) {
  const float* p = partial_at<EPI>(g, grp, row, col);
#pragma unroll
  for (int j = 0; j < kChunk; ++j) v[j] = u[j] = 0.f;
  for (int s = 0; s < g.splits; ++s, p += split_stride(g)) {
    float t[kChunk];
    load_chunk<L2>(p, t);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] += t[j];
    if constexpr (EPI == kEpiGated) {
      load_chunk<L2>(p + 128, t);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) u[j] += t[j];
    }
  }
}

// whether the sums of the chunk's `valid` columns are all finite
template <int EPI>
__device__ __forceinline__ bool chunk_finite(const float (&v)[kChunk], const float (&u)[kChunk],
                                             int64_t valid) {
  bool ok = true;
#pragma unroll
  for (int j = 0; j < kChunk; ++j) {
    ok &= j >= valid || isfinite(v[j]);
    if constexpr (EPI == kEpiGated) ok &= j >= valid || isfinite(u[j]);
  }
  return ok;
}

template <typename T, int EPI>
__device__ __forceinline__ void finish_chunk(const DenseGemm& g, int grp, int64_t row, int64_t col,
                                             float (&v)[kChunk], float (&u)[kChunk]) {
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int V = kChunk;
  const DenseEpi& ep = g.epi;
  const int64_t valid = g.N - col;
  if constexpr (EPI == kEpiGluBwd) {
    float gg[V];
    load_row<V>(static_cast<const float*>(ep.z) + row * ep.ldz + col, gg, valid, ep.vec & kVecZ);
    load_row<V>(static_cast<const float*>(ep.z2) + row * ep.ldz + col, u, valid, ep.vec & kVecZ);
    act_switch(ep.act, [&](auto A) {
      float d[V];
      act_grads<kFast, decltype(A)::value>(gg, d, ep.gamma);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float a = gg[j];
        gg[j] = times_slope<decltype(A)::value>(v[j] * u[j], d[j]);
        u[j] = v[j] * a;
      }
    });
    store_row<V>(static_cast<T*>(ep.out) + row * ep.ldo + col, gg, valid, ep.vec & kVecOut);
    store_row<V>(static_cast<T*>(ep.out2) + row * ep.ldo + col, u, valid, ep.vec & kVecOut);
    return;
  }
  if (ep.bias) {
    float b[V];
    load_row<V>(static_cast<const T*>(ep.bias) + col, b, valid, false);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += b[j];
  }
  if constexpr (EPI == kEpiGated) {
    if (ep.bias2) {
      float b[V];
      load_row<V>(static_cast<const T*>(ep.bias2) + col, b, valid, false);
#pragma unroll
      for (int j = 0; j < V; ++j) u[j] += b[j];
    }
    if (ep.z) {
      store_row<V>(static_cast<float*>(ep.z) + row * ep.ldz + col, v, valid, ep.vec & kVecZ);
      store_row<V>(static_cast<float*>(ep.z2) + row * ep.ldz + col, u, valid, ep.vec & kVecZ);
    }
    act_switch(ep.act, [&](auto A) {
      act_values<kFast, decltype(A)::value>(v, ep.gamma);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= u[j];
    });
  } else {
    if (ep.z) store_row<V>(static_cast<T*>(ep.z) + row * ep.ldz + col, v, valid, ep.vec & kVecZ);
    act_switch(ep.act, [&](auto A) { act_values<kFast, decltype(A)::value>(v, ep.gamma); });
    if (ep.res) {
      float r[V];
      load_row<V>(static_cast<const T*>(ep.res) + row * ep.ldr + col, r, valid, ep.vec & kVecRes);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += r[j];
    }
  }
  void* out = grp ? ep.out2 : ep.out;
  if (ep.out_f32)
    store_row<V>(static_cast<float*>(out) + row * ep.ldo + col, v, valid, ep.vec & kVecOut);
  else
    store_row<V>(static_cast<T*>(out) + row * ep.ldo + col, v, valid, ep.vec & kVecOut);
}

}  // namespace vmoe
