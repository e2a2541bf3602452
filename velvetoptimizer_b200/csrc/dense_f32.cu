// fp32 products of the dense operators.
//
// On the tensor cores: x = hi + mid + lo with each part a bf16 (hi = bf16(x), mid = bf16(x - hi),
// lo = bf16(x - hi - mid); both differences are exact, what is left is below 2^-26 |x|), so
//   x y = lo hi + hi lo + mid mid + mid hi + hi mid + hi hi + O(2^-25) |x y|,
// six bf16 products, exact in fp32, accumulated from the smallest up by the pair kernel as six
// operand pairs of one product (512 x 768 x 1024: 12 to 16 us a product, its finish 5 more).  Six times the work of a bf16 product at sixteen times and more
// the rate of the fp32 pipes; the split kernel below writes the planes (10 bytes per element).
//
// Where such a sum leaves fp32's range the parts give NaN (infinity times a zero part, or plus and
// minus infinity from parts of either sign) though fp32 arithmetic may give infinity: operands
// that are infinite or round to infinity as bf16, and finite ones whose products overflow.  Every
// one of these shows as a sum that is not finite, which the finish kernel sees: it leaves the
// chunk of 8 columns alone and sets the product's flag, and the redo kernel below, which otherwise
// ends at once, multiplies the tiles with such chunks again on the CUDA cores and finishes them.
// Near the bottom of the range the parts end at bf16's smallest number: x is then off by up to
// 2^-134, which is more than fp32's rounding only where |x| is below 2^-109.
//
// The redo product: C[m, n] = sum_k A(m, k) B(n, k) for operands of any strides, 128 x 128 tiles of
// 16 k, 256 threads with 8 x 8 outputs each; the next tile's elements are loaded into registers
// while the current one is multiplied.  A gated tile is 64 features, gate and up.
#include "common.cuh"
#include "dense.h"
#include "dense_finish.cuh"

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

template <typename F>
__device__ __forceinline__ void load_tile(bool k_fast, int64_t k0, int64_t K, F&& value, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int m, k;
    tile_at(k_fast, i, m, k);
    v[i] = k0 + k < K ? value(m, k0 + k) : 0.f;
  }
}

__device__ __forceinline__ void store_tile(float (*s)[PITCH], bool k_fast, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int m, k;
    tile_at(k_fast, i, m, k);
    s[k][m] = v[i];
  }
}

template <int EPI>
__global__ void __launch_bounds__(256)
dense_redo_kernel(const __grid_constant__ RedoGemm r) {
  constexpr bool kGate = EPI == kEpiGated;
  constexpr int TN = kGate ? 64 : TM;    // output columns of a tile
  constexpr int CHUNKS = TN / kChunk;
  pdl_wait_and_trigger();
  const DenseGemm& g = r.g;
  if (*g.redo == 0) return;
  __shared__ __align__(16) float As[2][TK][PITCH];
  __shared__ __align__(16) float Bs[2][TK][PITCH];
  __shared__ bool again[TM * CHUNKS];
  const int64_t mt = (g.M + TM - 1) / TM, nt = (g.N + TN - 1) / TN;
  const int64_t split_stride = static_cast<int64_t>(g.groups) * g.M * g.ldp;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t tile = blockIdx.x; tile < mt * nt * g.groups; tile += gridDim.x) {
    const int grp = static_cast<int>(tile / (mt * nt));
    const int64_t in = tile - grp * (mt * nt);
    const int64_t m0 = in / nt * TM, n0 = in % nt * TN;
    int any = 0;
    for (int i = threadIdx.x; i < TM * CHUNKS; i += 256) {
      const int64_t row = m0 + i / CHUNKS, col = n0 + i % CHUNKS * kChunk;
      bool bad = false;
      if (row < g.M && col < g.N) {
        float v[kChunk], u[kChunk];
        chunk_sums<EPI>(g, grp, row, col, v, u);
        bad = !chunk_finite<EPI>(v, u, g.N - col);
      }
      again[i] = bad;
      any |= bad;
    }
    if (!__syncthreads_or(any)) continue;
    float acc[8][8] = {};
    int buf = 0;
    for (int pair = 0; pair < r.pairs; ++pair) {
      const float* a = r.a[r.pairs == 2 ? pair : grp];
      const float* b = r.b[r.pairs == 2 ? pair : 0];
      auto a_at = [&](int m, int64_t k) {
        return m0 + m < g.M ? a[(m0 + m) * r.am + k * r.ak] : 0.f;
      };
      auto b_at = [&](int n, int64_t k) {
        const float* p = b;
        int64_t f = n0 + n;
        if (kGate && n >= TN) {  // the up rows of the same features
          p = r.b[1];
          f -= TN;
        }
        return f < g.N ? p[f * r.bn + k * r.bk] : 0.f;
      };
      float av[8], bv[8];
      load_tile(r.ak == 1, 0, r.K, a_at, av);
      load_tile(r.bk == 1, 0, r.K, b_at, bv);
      for (int64_t k = 0; k < r.K; k += TK, buf ^= 1) {
        store_tile(As[buf], r.ak == 1, av);
        store_tile(Bs[buf], r.bk == 1, bv);
        __syncthreads();
        if (k + TK < r.K) {
          load_tile(r.ak == 1, k + TK, r.K, a_at, av);
          load_tile(r.bk == 1, k + TK, r.K, b_at, bv);
        }
#pragma unroll
        for (int kk = 0; kk < TK; ++kk) {
          float x[8], y[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<float4*>(x + 4 * h) =
                *reinterpret_cast<const float4*>(&As[buf][kk][64 * h + 4 * ty]);
            *reinterpret_cast<float4*>(y + 4 * h) =
                *reinterpret_cast<const float4*>(&Bs[buf][kk][64 * h + 4 * tx]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
        }
      }
    }
    // the chunks' sums are replaced (the first split's; zeros for the others), then finished
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = 64 * (i >> 2) + 4 * ty + (i & 3);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = (kGate ? 0 : 64 * (j >> 2)) + 4 * tx + (j & 3);
        const int64_t col = n0 + n;
        if (col >= g.N || !again[m * CHUNKS + n / kChunk]) continue;
        const int64_t pcol = kGate ? (col / 128) * 256 + (col & 127) + (j >= 4 ? 128 : 0) : col;
        float* p = g.partial + (static_cast<int64_t>(grp) * g.M + m0 + m) * g.ldp + pcol;
        *p = acc[i][j];
        for (int s = 1; s < g.splits; ++s) p[s * split_stride] = 0.f;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TM * CHUNKS; i += 256) {
      if (!again[i]) continue;
      const int64_t row = m0 + i / CHUNKS, col = n0 + i % CHUNKS * kChunk;
      float v[kChunk], u[kChunk];
      chunk_sums<EPI>(g, grp, row, col, v, u);
      finish_chunk<float, EPI>(g, grp, row, col, v, u);
    }
  }
}

struct SplitArgs {
  Split3 m[3];
  int* clear;
};

__global__ void __launch_bounds__(256)
split3_kernel(const __grid_constant__ SplitArgs args) {
  pdl_wait_and_trigger();
  const Split3& m = args.m[blockIdx.y];
  const int64_t units = m.ldo / 8, total = m.rows * units;
  const bool vec = ((reinterpret_cast<uintptr_t>(m.x) | static_cast<uintptr_t>(m.ldx * 4)) & 15u) == 0;
  auto* out = static_cast<__nv_bfloat16*>(m.out);
  if (args.clear && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < kRedoWords)
    args.clear[threadIdx.x] = 0;
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
}

}  // namespace

cudaError_t launch_split3(const Split3* m, int n, int* clear, cudaStream_t s) {
  if (n < 1 || n > 3) return cudaErrorInvalidValue;
  SplitArgs a{};
  for (int i = 0; i < n; ++i) a.m[i] = m[i];
  a.clear = clear;
  return launch_kernel(split3_kernel, dim3(kSplitBlocks, static_cast<unsigned>(n)), dim3(256), 0, s, a);
}

cudaError_t launch_dense_redo(int epi, const RedoGemm& r, int num_sms, cudaStream_t s) {
  if (!r.g.redo || !r.g.partial || r.pairs < 1 || r.pairs > 2 || (r.pairs == 2 && r.g.groups != 1))
    return cudaErrorInvalidValue;
  // no wider than the SMs: it hardly ever has work
  const int tn = epi == kEpiGated ? 64 : TM;
  const int64_t tiles = (r.g.M + TM - 1) / TM * ((r.g.N + tn - 1) / tn) * r.g.groups;
  const dim3 grid(static_cast<unsigned>(tiles < num_sms ? tiles : num_sms));
  if (epi == kEpiGated) return launch_kernel(dense_redo_kernel<kEpiGated>, grid, dim3(256), 0, s, r);
  if (epi == kEpiGluBwd) return launch_kernel(dense_redo_kernel<kEpiGluBwd>, grid, dim3(256), 0, s, r);
  return launch_kernel(dense_redo_kernel<kEpiLinear>, grid, dim3(256), 0, s, r);
}

}  // namespace vmoe
