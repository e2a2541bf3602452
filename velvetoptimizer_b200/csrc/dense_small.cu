// Fused linear and gated projection for few rows (T <= 16): the weights are the work.
//
//   out[t, n] = epilogue(sum_k w[n, k] x[t, k])
//
// Bound: each weight is read once and used T times, so the kernel is as fast as the weights
// stream in.  mma.sync m16n8k16 takes 16 weight rows as its M operand and 8 tokens as N; the
// products cost nothing next to the loads, and both operands come straight from global memory
// in fragment order with 16-byte loads: k is only summed over, so within 32 consecutive k
// lane t of a row takes k = 8t..8t+7 and hands them to two MMAs as their (2t, 2t+1, 2t+8,
// 2t+9) pairs, the same permutation for weights and tokens.  No shared memory or barrier
// stands between a load and its use; four 32-wide chunks of two weight rows per lane are in
// flight.  A block owns 16 weight rows, its 8 to 32 warps take its chunks in turn and add
// their sums through shared memory in warp order.  The gated form takes 8 gate rows and 8 up rows
// of the same features as the 16, so one thread ends up with both.
#include "common.cuh"
#include "dense.h"
#include "dense_act.cuh"

namespace vmoe {
namespace {

constexpr int UNROLL = 4;

// 8 elements of a row from k on, 0 past K or without a row
template <bool VEC>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int64_t k, int64_t K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (!row) return v;
  if constexpr (VEC) {  // K % 8 == 0 and 16-byte aligned rows
    if (k < K) v = __ldg(reinterpret_cast<const uint4*>(row + k));
  } else {
    const auto* p = reinterpret_cast<const unsigned short*>(row);
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = k + j < K ? __ldg(p + k + j) : 0u;
    v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  }
  return v;
}

template <int EPI, bool VEC, int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
dense_small_kernel(const SmallGemm g) {
  constexpr bool kGate = EPI == kEpiGated;
  constexpr int ROWS = kGate ? 8 : 16;  // output features per block
  __shared__ float4 red[WARPS][NT][32];
  __shared__ float sum[NT][16][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * ROWS;
  pdl_wait_and_trigger();

  const auto* w = static_cast<const __nv_bfloat16*>(g.w);
  const auto* w2 = static_cast<const __nv_bfloat16*>(g.w2);
  const auto* x = static_cast<const __nv_bfloat16*>(g.x);
  const __nv_bfloat16* r0 = n0 + gid < g.N ? w + (n0 + gid) * g.ldw : nullptr;
  const __nv_bfloat16* r1;
  if constexpr (kGate) {
    r1 = n0 + gid < g.N ? w2 + (n0 + gid) * g.ldw2 : nullptr;
  } else {
    r1 = n0 + gid + 8 < g.N ? w + (n0 + gid + 8) * g.ldw : nullptr;
  }
  const __nv_bfloat16* xr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) xr[n] = n * 8 + gid < g.T ? x + (n * 8 + gid) * g.ldx : nullptr;

  // this thread's output, and what its epilogue reads, asked for with the weights
  const DenseEpi& ep = g.epi;
  const int f = threadIdx.x % ROWS, t = threadIdx.x / ROWS;
  const int64_t col = n0 + f;
  const bool mine = t < g.T && t < NT * 8 && col < g.N;
  auto read = [&](const void* p, int64_t i) {
    return p && mine ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : 0.f;
  };
  const float b0 = read(ep.bias, col), b1 = kGate ? read(ep.bias2, col) : 0.f;
  const float res = kGate ? 0.f : read(ep.res, t * ep.ldr + col);

  float acc[NT][4] = {};
  const int64_t chunks = (g.K + 31) / 32;
  for (int64_t c = warp; c < chunks; c += WARPS * UNROLL) {
    uint4 a[UNROLL], b[UNROLL], v[UNROLL][NT];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t k = (c + u * WARPS) * 32 + tig * 8;  // past K: zeros
      a[u] = load8<VEC>(r0, k, g.K);
      b[u] = load8<VEC>(r1, k, g.K);
#pragma unroll
      for (int n = 0; n < NT; ++n) v[u][n] = load8<VEC>(xr[n], k, g.K);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_bf16(acc[n], a[u].x, b[u].x, a[u].y, b[u].y, v[u][n].x, v[u][n].y);
        mma_bf16(acc[n], a[u].z, b[u].z, a[u].w, b[u].w, v[u][n].z, v[u][n].w);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
    red[warp][n][lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
  __syncthreads();
  if (threadIdx.x < NT * 128) {
    const int n = threadIdx.x >> 7, l = (threadIdx.x >> 2) & 31, i = threadIdx.x & 3;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) s += reinterpret_cast<const float*>(&red[k][n][l])[i];
    sum[n][(l >> 2) + 8 * (i >> 1)][(l & 3) * 2 + (i & 1)] = s;
  }
  __syncthreads();
  if (!mine) return;
  float z = sum[t >> 3][f][t & 7] + b0;
  auto* out = static_cast<__nv_bfloat16*>(ep.out);
  if constexpr (kGate) {
    const float up = sum[t >> 3][f + 8][t & 7] + b1;
    if (ep.z) {
      static_cast<float*>(ep.z)[t * ep.ldz + col] = z;
      static_cast<float*>(ep.z2)[t * ep.ldz + col] = up;
    }
    act_switch(ep.act, [&](auto A) { z = act_value2<decltype(A)::value>(both(z), ep.gamma).x * up; });
  } else {
    if (ep.z) static_cast<__nv_bfloat16*>(ep.z)[t * ep.ldz + col] = __float2bfloat16_rn(z);
    act_switch(ep.act, [&](auto A) { z = act_value2<decltype(A)::value>(both(z), ep.gamma).x; });
    z += res;
  }
  out[t * ep.ldo + col] = __float2bfloat16_rn(z);
}

// Warps per block: about four 32-wide chunks each (one batch of loads), so that all of a
// block's weights are in flight at once; 32 only where the blocks are too few to fill the SMs
// twice.  One row, cold weights, K x N: 2048 x 2048 7.4 / 4.1 / 4.2 us with 8 / 16 / 32 warps,
// 8192 x 2048 24.4 / 14.5 / 10.8 us, 2048 x 8192 9.4 / 8.9 / 13.4 us.
template <int EPI, bool VEC, int NT>
cudaError_t launch_warps(const SmallGemm& g, unsigned blocks, cudaStream_t s) {
  const int64_t chunks = (g.K + 31) / 32;
  if (chunks > 64 && blocks < 2u * static_cast<unsigned>(g.num_sms))
    return launch_kernel(dense_small_kernel<EPI, VEC, NT, 32>, dim3(blocks), dim3(1024), 0, s, g);
  if (chunks > 32)
    return launch_kernel(dense_small_kernel<EPI, VEC, NT, 16>, dim3(blocks), dim3(512), 0, s, g);
  return launch_kernel(dense_small_kernel<EPI, VEC, NT, 8>, dim3(blocks), dim3(256), 0, s, g);
}

template <int EPI, bool VEC>
cudaError_t launch_nt(const SmallGemm& g, unsigned blocks, cudaStream_t s) {
  return g.T <= 8 ? launch_warps<EPI, VEC, 1>(g, blocks, s) : launch_warps<EPI, VEC, 2>(g, blocks, s);
}

// The fp32 form on the CUDA cores: a block owns 4 output features (gated: 2 gate and 2 up rows),
// its 8 warps take the k range in turn, a lane 4 consecutive k.  A weight is loaded once and
// used for all TT tokens, a token's x (from L1) for the 4 rows.
template <int EPI, bool VEC, int TT>
__global__ void __launch_bounds__(256)
dense_small_f32_kernel(const SmallGemm g) {
  constexpr bool kGate = EPI == kEpiGated;
  constexpr int FEATURES = kGate ? 2 : 4;
  __shared__ float red[8][4][TT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * FEATURES;
  pdl_wait_and_trigger();
  const auto* w = static_cast<const float*>(g.w);
  const auto* w2 = static_cast<const float*>(g.w2);
  const auto* x = static_cast<const float*>(g.x);
  const float* row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + (kGate ? (i & 1) : i);
    row[i] = n < g.N ? (kGate && i >= 2 ? w2 + n * g.ldw2 : w + n * g.ldw) : nullptr;
  }
  auto load4 = [&](const float* p, int64_t k) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!p) return v;
    if constexpr (VEC) {  // K % 4 == 0 and 16-byte aligned rows
      if (k < g.K) v = __ldg(reinterpret_cast<const float4*>(p + k));
    } else {
      if (k < g.K) v.x = __ldg(p + k);
      if (k + 1 < g.K) v.y = __ldg(p + k + 1);
      if (k + 2 < g.K) v.z = __ldg(p + k + 2);
      if (k + 3 < g.K) v.w = __ldg(p + k + 3);
    }
    return v;
  };
  float acc[4][TT] = {};
  for (int64_t k = (warp * 32 + lane) * 4; k < g.K; k += 8 * 128) {
    float4 a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = load4(row[i], k);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const float4 b = load4(t < g.T ? x + t * g.ldx : nullptr, k);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i][t] += a[i].x * b.x + a[i].y * b.y + a[i].z * b.z + a[i].w * b.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float s = acc[i][t];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) red[warp][i][t] = s;
    }
  __syncthreads();
  const int f = threadIdx.x % FEATURES, t = threadIdx.x / FEATURES;
  const int64_t col = n0 + f;
  if (t >= g.T || t >= TT || col >= g.N) return;
  const DenseEpi& ep = g.epi;
  auto total = [&](int i, const void* bias) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += red[k][i][t];
    return s + (bias ? static_cast<const float*>(bias)[col] : 0.f);
  };
  float z = total(f, ep.bias);
  if (ep.z) static_cast<float*>(ep.z)[t * ep.ldz + col] = z;
  if constexpr (kGate) {
    const float up = total(f + 2, ep.bias2);
    if (ep.z) static_cast<float*>(ep.z2)[t * ep.ldz + col] = up;
    act_switch(ep.act, [&](auto A) { z = act_value1<decltype(A)::value>(z, ep.gamma) * up; });
  } else {
    act_switch(ep.act, [&](auto A) { z = act_value1<decltype(A)::value>(z, ep.gamma); });
    if (ep.res) z += static_cast<const float*>(ep.res)[t * ep.ldr + col];
  }
  static_cast<float*>(ep.out)[t * ep.ldo + col] = z;
}

template <int EPI, bool VEC>
cudaError_t launch_f32(const SmallGemm& g, cudaStream_t s) {
  const int features = EPI == kEpiGated ? 2 : 4;
  const dim3 grid(static_cast<unsigned>((g.N + features - 1) / features));
  if (g.T <= 2) return launch_kernel(dense_small_f32_kernel<EPI, VEC, 2>, grid, dim3(256), 0, s, g);
  if (g.T <= 8) return launch_kernel(dense_small_f32_kernel<EPI, VEC, 8>, grid, dim3(256), 0, s, g);
  return launch_kernel(dense_small_f32_kernel<EPI, VEC, 16>, grid, dim3(256), 0, s, g);
}

}  // namespace

cudaError_t launch_dense_small(int dtype, int epi, const SmallGemm& g, cudaStream_t s) {
  if (g.T < 1 || g.T > kSmallTokens) return cudaErrorInvalidValue;
  if (dtype == kF32) {
    if (epi == kEpiGated)
      return g.vec_in ? launch_f32<kEpiGated, true>(g, s) : launch_f32<kEpiGated, false>(g, s);
    return g.vec_in ? launch_f32<kEpiLinear, true>(g, s) : launch_f32<kEpiLinear, false>(g, s);
  }
  if (g.epi.out_f32) return cudaErrorInvalidValue;
  const int rows = epi == kEpiGated ? 8 : 16;
  // Persistent blocks that copy ahead (dense_stream.cu) pay where a block has several tiles or
  // several slices of k to hide the waits between, and where two token groups make the
  // register form's loads too few.  One row, cold weights, register / stream form: 8192 x 2048
  // 10.9 / 9.9 us, gate|up of 2048 x 8192 14.8 / 13.3 us, but 2048 x 8192 8.9 / 9.6 us and
  // 2048 x 2048 4.1 / 4.8 us; 16 rows: 2048 x 8192 13.0 / 11.3 us, 2048 x 2048 6.4 / 5.4 us.
  // Between 2048 and 4096 k the last slice is short and the rule is wide of the mark for a single
  // product: 2560 x 2048 5.5 / 5.9 us with one row, 2560 x 8192 15.9 / 19.7 us with 16; a block of
  // 2304 x 8192, whose second launch asks for its weights early, 33.3 / 27.9 and 39.2 / 41.5 us.
  if (g.vec_in && (g.K > 2048 || (g.N + rows - 1) / rows >= 6 * g.num_sms || (g.T > 8 && g.K > 1024)))
    return launch_dense_stream(epi, g, s);
  const unsigned blocks = static_cast<unsigned>((g.N + rows - 1) / rows);
  cudaError_t e;
  if (epi == kEpiGated)
    e = g.vec_in ? launch_nt<kEpiGated, true>(g, blocks, s) : launch_nt<kEpiGated, false>(g, blocks, s);
  else
    e = g.vec_in ? launch_nt<kEpiLinear, true>(g, blocks, s) : launch_nt<kEpiLinear, false>(g, blocks, s);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace vmoe
