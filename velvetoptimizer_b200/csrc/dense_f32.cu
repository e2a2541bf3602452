// fp32 products of the dense operators.
//
// On the tensor cores: x = hi + mid + lo with each part a bf16 (hi = bf16(x), mid = bf16(x - hi),
// lo = bf16(x - hi - mid); both differences are exact, what is left is below 2^-26 |x|), so
//   x y = lo hi + hi lo + mid mid + mid hi + hi mid + hi hi + O(2^-25) |x y|,
// six bf16 products, exact in fp32, accumulated from the smallest up by the pair kernel as six
// operand pairs of one product (512 x 768 x 1024: 12 to 16 us a product, its finish 5 more).  Six times the work of a bf16 product at sixteen times and more
// the rate of the fp32 pipes; the split kernel below writes the planes (10 bytes per element).
//
// An operand that is infinite, NaN, or rounds to infinity as bf16 has no such sum (infinity
// times a zero part would be NaN).  The split kernel flags its block, and the CUDA-core product
// below, which otherwise ends at once, then overwrites the partial sums with fp32 arithmetic.
//
// The CUDA-core product: C[m, n] = sum_k A(m, k) B(n, k) for operands of any strides, 128 x 128
// tiles of 16 k, 256 threads with 8 x 8 outputs each; the next tile's elements are loaded into
// registers while the current one is multiplied.
#include "common.cuh"
#include "dense.h"

namespace vmoe {
namespace {

constexpr int TM = 128, TK = 16, PITCH = TM + 4;

// this thread's 8 of the tile's 128 x 16 elements: along k when k is contiguous, else along m
__device__ __forceinline__ void tile_at(bool k_fast, int i, int& m, int& k) {
  const int e = threadIdx.x + 256 * i;
  if (k_fast) {
    k = e & 15;
    m = e >> 4;
  } else {
    m = e & 127;
    k = e >> 7;
  }
}

__device__ __forceinline__ void load_tile(const float* p, int64_t sm, int64_t sk, int64_t m0,
                                          int64_t M, int64_t k0, int64_t k1, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int m, k;
    tile_at(sk == 1, i, m, k);
    v[i] = (m0 + m < M && k0 + k < k1) ? p[(m0 + m) * sm + (k0 + k) * sk] : 0.f;
  }
}

__device__ __forceinline__ void store_tile(float (*s)[PITCH], int64_t sk, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int m, k;
    tile_at(sk == 1, i, m, k);
    s[k][m] = v[i];
  }
}

__global__ void __launch_bounds__(256)
dense_simt_kernel(const SimtGemm g) {
  pdl_wait_and_trigger();
  int set = 0;
  for (int i = threadIdx.x; i < g.n_flags; i += 256) set |= g.flags[i];
  if (!__syncthreads_or(set)) return;
  __shared__ __align__(16) float As[2][TK][PITCH];
  __shared__ __align__(16) float Bs[2][TK][PITCH];
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * TM, n0 = static_cast<int64_t>(blockIdx.y) * TM;
  const int64_t kb = blockIdx.z * g.k_per_split;
  const int64_t ke = min(g.K, kb + g.k_per_split);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[8][8] = {};
  float av[8], bv[8];
  load_tile(g.a, g.am, g.ak, m0, g.M, kb, ke, av);
  load_tile(g.b, g.bn, g.bk, n0, g.N, kb, ke, bv);
  int buf = 0;
  for (int64_t k = kb; k < ke; k += TK, buf ^= 1) {
    store_tile(As[buf], g.ak, av);
    store_tile(Bs[buf], g.bk, bv);
    __syncthreads();
    if (k + TK < ke) {
      load_tile(g.a, g.am, g.ak, m0, g.M, k + TK, ke, av);
      load_tile(g.b, g.bn, g.bk, n0, g.N, k + TK, ke, bv);
    }
#pragma unroll
    for (int kk = 0; kk < TK; ++kk) {
      float a[8], b[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<float4*>(a + 4 * h) =
            *reinterpret_cast<const float4*>(&As[buf][kk][64 * h + 4 * ty]);
        *reinterpret_cast<float4*>(b + 4 * h) =
            *reinterpret_cast<const float4*>(&Bs[buf][kk][64 * h + 4 * tx]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
  }
  float* out = g.partial + blockIdx.z * g.split_stride;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + 64 * (i >> 2) + 4 * ty + (i & 3);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t n = n0 + 64 * (j >> 2) + 4 * tx + (j & 3);
      if (n >= g.N) continue;
      const int64_t col = g.gated_cols ? (n / 128) * 256 + (n & 127) + (g.gated_cols == 2 ? 128 : 0) : n;
      out[m * g.ldp + col] = g.accumulate ? out[m * g.ldp + col] + acc[i][j] : acc[i][j];
    }
  }
}

struct SplitArgs {
  Split3 m[3];
  int* flags;
};

__global__ void __launch_bounds__(256)
split3_kernel(const __grid_constant__ SplitArgs args) {
  pdl_wait_and_trigger();
  const Split3& m = args.m[blockIdx.y];
  const int64_t units = m.ldo / 8, total = m.rows * units;
  const bool vec = ((reinterpret_cast<uintptr_t>(m.x) | static_cast<uintptr_t>(m.ldx * 4)) & 15u) == 0;
  auto* out = static_cast<__nv_bfloat16*>(m.out);
  int bad = 0;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t r = i / units, c = (i - r * units) * 8;
    float v[8];
    const float* p = m.x + r * m.ldx + c;
    if (vec && c + 8 <= m.cols) {
      load16_to_f(p, v);
      load16_to_f(p + 4, v + 4);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < m.cols ? p[j] : 0.f;
    }
    float mid[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float hi = __bfloat162float(__float2bfloat16_rn(v[j]));
      const bool ok = fabsf(hi) < __int_as_float(0x7f800000);
      bad |= !ok;
      const float rest = v[j] - hi;
      const float md = __bfloat162float(__float2bfloat16_rn(rest));
      v[j] = hi;
      mid[j] = ok ? md : 0.f;
      lo[j] = ok ? rest - md : 0.f;
    }
    __nv_bfloat16* q = out + r * m.ldo + c;
    store16_from_f(q, v);
    store16_from_f(q + m.plane, mid);
    store16_from_f(q + 2 * m.plane, lo);
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) args.flags[blockIdx.y * kSplitBlocks + blockIdx.x] = bad;
}

}  // namespace

cudaError_t launch_split3(const Split3* m, int n, int* flags, cudaStream_t s) {
  if (n < 1 || n > 3) return cudaErrorInvalidValue;
  SplitArgs a{};
  for (int i = 0; i < n; ++i) a.m[i] = m[i];
  a.flags = flags;
  return launch_kernel(split3_kernel, dim3(kSplitBlocks, static_cast<unsigned>(n)), dim3(256), 0, s, a);
}

cudaError_t launch_dense_simt(const SimtGemm& g, cudaStream_t s) {
  const int64_t mt = (g.M + TM - 1) / TM, nt = (g.N + TM - 1) / TM;
  if (nt > 65535 || g.splits < 1 || g.splits > 65535) return cudaErrorInvalidValue;
  return launch_kernel(dense_simt_kernel,
                       dim3(static_cast<unsigned>(mt), static_cast<unsigned>(nt),
                            static_cast<unsigned>(g.splits)),
                       dim3(256), 0, s, g);
}

}  // namespace vmoe
