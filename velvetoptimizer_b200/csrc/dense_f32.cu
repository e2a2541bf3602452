// fp32 products of the dense operators.
//
// On the tensor cores: x = hi + mid + lo with each part a bf16 (hi = bf16(x), mid = bf16(x - hi),
// lo = bf16(x - hi - mid); both differences are exact, what is left is below 2^-26 |x|), so
//   x y = lo hi + hi lo + mid mid + mid hi + hi mid + hi hi + O(2^-25) |x y|,
// six bf16 products, exact in fp32, accumulated from the smallest up by the pair kernel as six
// operand pairs of one product (512 x 768 x 1024: 12 to 13 us a product; its finish and the redo
// launch, which come up while it runs, add 5).  Six times the work of a bf16 product at sixteen
// times and more the rate of the fp32 pipes; the split kernel below writes the planes (10 bytes per
// element).
//
// Where such a sum leaves fp32's range the parts give NaN (infinity times a zero part, or plus and
// minus infinity from parts of either sign) though fp32 arithmetic may give infinity: operands
// that are infinite or round to infinity as bf16, and finite ones whose products overflow.  Every
// one of these shows as a sum that is not finite, which the finish kernel sees: it marks the
// chunk of 8 columns in its partials and sets the product's flag, and the redo kernel below, which
// otherwise ends at once, multiplies the tiles with such chunks again on the CUDA cores, k divided
// as the product's was; the last of a tile's blocks adds the parts, in order, and finishes them.
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

// A thread's 8 of a tile's 128 rows x 16 k, read tile after tile along k: consecutive k of 8 rows
// 16 apart where k is contiguous, else 8 k two apart of one row.  The tile's upper 64 rows may
// belong to another matrix.
struct Reader {
  const float *lo, *hi;  // elements 0 to 3, and 4 to 7
  int64_t step, next;    // between elements, and to the next tile
  int k, dk;             // the first element's k in the tile, and between elements
  uint32_t inside;       // elements whose row exists

  // rows [0, n) of `p` are the tile's first, rows [0, n2) of `p2` its upper 64
  __device__ __forceinline__ Reader(const float* p, int64_t n, const float* p2, int64_t n2, int64_t sr,
                                    int64_t sk, int64_t k0) {
    const bool k_fast = sk == 1;
    const int t = threadIdx.x, row = k_fast ? t >> 4 : t & 127;
    k = k_fast ? t & 15 : t >> 7;
    dk = k_fast ? 0 : 2;
    step = k_fast ? 16 * sr : 2 * sk;
    next = TK * sk;
    inside = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = row + (k_fast ? 16 * i : 0);
      if (m < 64 ? m < n : m - 64 < n2) inside |= 1u << i;
    }
    lo = (row < 64 ? p + row * sr : p2 + (row - 64) * sr) + (k0 + k) * sk;
    hi = k_fast ? p2 + row * sr + (k0 + k) * sk : lo + 4 * step;
  }

  __device__ __forceinline__ void load(int64_t left, float (&v)[8]) {  // k left, from this tile on
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* q = i < 4 ? lo : hi;
      v[i] = (inside >> i & 1) && k + i * dk < left ? q[(i & 3) * step] : 0.f;
    }
    lo += next;
    hi += next;
  }

  __device__ __forceinline__ void store(float (*s)[PITCH], const float (&v)[8]) const {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (dk) s[k + 2 * i][t & 127] = v[i];
      else s[k][(t >> 4) + 16 * i] = v[i];
    }
  }
};

template <int EPI>
__global__ void __launch_bounds__(256, 2)
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
  __shared__ int last;
  const int64_t mt = (g.M + TM - 1) / TM, nt = (g.N + TN - 1) / TN;
  const int64_t per = (r.K + g.splits - 1) / g.splits;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t item = blockIdx.x; item < g.redo_tiles * g.splits; item += gridDim.x) {
    const int64_t tile = item / g.splits;
    const int split = static_cast<int>(item - tile * g.splits);
    const int grp = static_cast<int>(tile / (mt * nt));
    const int64_t in = tile - grp * (mt * nt);
    const int64_t m0 = in / nt * TM, n0 = in % nt * TN;
    const int64_t k0 = split * per, k1 = min(r.K, k0 + per);
    int any = 0;
    for (int i = threadIdx.x; i < TM * CHUNKS; i += 256) {
      const int64_t row = m0 + i / CHUNKS, col = n0 + i % CHUNKS * kChunk;
      // a chunk whose sums are finite has no partial that is not
      const bool bad = row < g.M && col < g.N &&
                       !isfinite(partial_at<EPI>(g, grp, row, col)[split * split_stride(g)]);
      again[i] = bad;
      any |= bad;
    }
    if (!__syncthreads_or(any)) continue;
    float acc[8][8] = {};
    int buf = 0;
    for (int pair = 0; pair < r.pairs; ++pair) {
      const float* a = r.a[r.pairs == 2 ? pair : grp] + m0 * r.am;
      const float* b = r.b[r.pairs == 2 ? pair : 0] + n0 * r.bn;
      const int64_t rows = g.M - m0, cols = g.N - n0;
      Reader ra(a, rows, a + 64 * r.am, rows - 64, r.am, r.ak, k0);
      Reader rb(b, cols, kGate ? r.b[1] + n0 * r.bn : b + 64 * r.bn, kGate ? cols : cols - 64, r.bn,
                r.bk, k0);
      float av[8], bv[8];
      ra.load(k1 - k0, av);
      rb.load(k1 - k0, bv);
      for (int64_t k = k0; k < k1; k += TK, buf ^= 1) {
        ra.store(As[buf], av);
        rb.store(Bs[buf], bv);
        __syncthreads();
        if (k + TK < k1) {
          ra.load(k1 - k - TK, av);
          rb.load(k1 - k - TK, bv);
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = 64 * (i >> 2) + 4 * ty + (i & 3);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = (kGate ? 0 : 64 * (j >> 2)) + 4 * tx + (j & 3);
        if (n0 + n >= g.N || !again[m * CHUNKS + n / kChunk]) continue;
        partial_at<EPI>(g, grp, m0 + m, n0 + n)[split * split_stride(g) + (kGate && j >= 4 ? 128 : 0)] =
            acc[i][j];
      }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(g.arrived + tile, 1) == g.splits - 1;
    __syncthreads();
    if (last) {
      __threadfence();
      for (int i = threadIdx.x; i < TM * CHUNKS; i += 256) {
        if (!again[i]) continue;
        const int64_t row = m0 + i / CHUNKS, col = n0 + i % CHUNKS * kChunk;
        float v[kChunk], u[kChunk];
        chunk_sums<EPI, true>(g, grp, row, col, v, u);
        finish_chunk<float, EPI>(g, grp, row, col, v, u);
      }
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

int64_t redo_tiles(int epi, int64_t M, int64_t N, int groups) {
  const int tn = epi == kEpiGated ? 64 : TM;
  return (M + TM - 1) / TM * ((N + tn - 1) / tn) * groups;
}

cudaError_t launch_dense_redo(int epi, const RedoGemm& r, int num_sms, cudaStream_t s) {
  if (!r.g.redo || !r.g.arrived || !r.g.partial || r.pairs < 1 || r.pairs > 2 ||
      (r.pairs == 2 && r.g.groups != 1) ||
      r.g.redo_tiles != redo_tiles(epi, r.g.M, r.g.N, r.g.groups))
    return cudaErrorInvalidValue;
  // no more blocks than run at once: it hardly ever has work
  const int64_t items = r.g.redo_tiles * r.g.splits;
  const dim3 grid(static_cast<unsigned>(items < 2 * num_sms ? items : 2 * num_sms));
  if (epi == kEpiGated) return launch_kernel(dense_redo_kernel<kEpiGated>, grid, dim3(256), 0, s, r);
  if (epi == kEpiGluBwd) return launch_kernel(dense_redo_kernel<kEpiGluBwd>, grid, dim3(256), 0, s, r);
  return launch_kernel(dense_redo_kernel<kEpiLinear>, grid, dim3(256), 0, s, r);
}

}  // namespace vmoe
