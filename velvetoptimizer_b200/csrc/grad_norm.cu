// Global norm of many tensors and clipping in place (vmoe_grad_norm).
//
//   norm = (sum over all elements |g|^p)^(1/p),  p = 1, 2 or infinity
//   c = min(1, max_norm / (norm + 1e-6));  g *= c
//
// Two launches for up to 1024 tensors (two more for every further 1024): their addresses and
// sizes travel in the kernel's parameters, so nothing is copied to the device first and a captured call replays as it is.
// Tensors are cut into pieces of 1 to 16 KB (as many as give every warp one), and every warp
// takes pieces at a fixed stride, so many small tensors and a few large ones load the SMs alike
// and the order of every sum is fixed.
// 402 M fp32 values in 898 tensors: 235 us (6.9 TB/s).
// Bound by HBM: N bytes are read for the norm; where c < 1 they are read again and written, in
// reverse order, so that what the norm read last is still in L2.  Where c is 1 nothing is
// written (x * 1 has the same bits).  Sums are held in fp64: fp32 squares leave its range
// beyond 1e19, and a long fp32 sum of equal terms stops growing.
#include <type_traits>

#include "common.cuh"
#include "ops_host.h"

namespace vmoe {
namespace {

constexpr int kWarps = 8;
constexpr int kBlocksPerSm = 4;
constexpr int kMinPiece = 1024, kMaxPiece = 16384;  // bytes
constexpr int kBatch = 1024;     // tensors per launch: 20 KB of kernel parameters
constexpr int kSmallBatch = 64;

template <int N>
struct GradTable {
  void* ptr[N];
  int64_t count[N];      // elements; negative: bf16
  int32_t end_piece[N];  // pieces of tensors 0..i
  int n = 0;
  int first_partial = 0;
  int piece = kMaxPiece;
};

// Elements [first, last) of a tensor that its piece k covers.  Pieces are counted from the
// first 16-byte boundary, so all but the ends are whole aligned vectors.
template <typename T>
__device__ __forceinline__ void piece_range(const T* p, int64_t count, int64_t k, int piece,
                                            int64_t& first, int64_t& last) {
  const int64_t E = piece / static_cast<int>(sizeof(T));
  const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T);
  first = k == 0 ? 0 : head + k * E;
  last = min(count, head + (k + 1) * E);
}

// f(value) over the n elements at p (one piece): scalars up to the first 16-byte boundary,
// vectors, scalars
template <typename T, typename S, typename V>
__device__ __forceinline__ void walk(T* p, int n, int lane, S&& scalar, V&& vector) {
  constexpr int W = 16 / sizeof(T);
  constexpr int U = 8;  // loads in flight per lane
  const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) /
                                           sizeof(T)));
  if (lane < head) scalar(p + lane);
  uint4* q = reinterpret_cast<uint4*>(p + head) + lane;
  int left = (n - head) / W - lane;  // vectors from this lane's on
  const int tail = (n - head) % W;
  if (lane < tail) scalar(p + n - tail + lane);
  for (; left > 32 * (U - 1); left -= 32 * U, q += 32 * U) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = q[32 * u];
#pragma unroll
    for (int u = 0; u < U; ++u) vector(reinterpret_cast<T*>(q + 32 * u), v[u]);
  }
  for (; left > 0; left -= 32 * 4, q += 32 * 4) {  // what does not fill a round
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (left > 32 * u) v[u] = q[32 * u];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (left > 32 * u) vector(reinterpret_cast<T*>(q + 32 * u), v[u]);
  }
}

template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

// NaN wins over every number
__device__ __forceinline__ double max_nan(double a, double b) {
  return (a != a || a > b) ? a : b;
}

template <int P>
__device__ __forceinline__ void add_value(double& acc, float g) {
  if constexpr (P == 2) {
    const double d = static_cast<double>(g);
    acc = fma(d, d, acc);
  } else if constexpr (P == 1) {
    acc += static_cast<double>(fabsf(g));
  } else {
    acc = max_nan(static_cast<double>(fabsf(g)), acc);
  }
}

template <int P>
__device__ __forceinline__ double join(double a, double b) {
  return P == 0 ? max_nan(a, b) : a + b;
}

// index of the tensor that piece k belongs to
template <int N>
__device__ __forceinline__ int tensor_of(const GradTable<N>& t, int k) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (k < t.end_piece[mid]) hi = mid; else lo = mid + 1;
  }
  return lo;
}

template <int N, int P>
__global__ void __launch_bounds__(32 * kWarps, kBlocksPerSm)
grad_norm_kernel(const __grid_constant__ GradTable<N> t, double* partial) {
  __shared__ double red[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total = t.end_piece[t.n - 1];
  pdl_wait_and_trigger();
  double acc = 0.0;
  for (int k = blockIdx.x * kWarps + warp; k < total; k += gridDim.x * kWarps) {
    const int i = tensor_of(t, k);
    const int64_t at = k - (i ? t.end_piece[i - 1] : 0);
    auto run = [&](auto* p, int64_t count) {
      using T = std::remove_reference_t<decltype(*p)>;
      int64_t first, last;
      piece_range(p, count, at, t.piece, first, last);
      walk(p + first, static_cast<int>(last - first), lane, [&](T* q) { add_value<P>(acc, Elt<T>::to_f(*q)); },
           [&](T*, uint4 v) {
             float f[16 / sizeof(T)];
             unpack<T>(v, f);
#pragma unroll
             for (int j = 0; j < 16 / static_cast<int>(sizeof(T)); ++j) add_value<P>(acc, f[j]);
           });
    };
    if (t.count[i] < 0) run(static_cast<__nv_bfloat16*>(t.ptr[i]), -t.count[i]);
    else run(static_cast<float*>(t.ptr[i]), t.count[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc = join<P>(acc, __shfl_xor_sync(0xffffffffu, acc, o));
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s = join<P>(s, red[w]);
    partial[t.first_partial + blockIdx.x] = s;
  }
}

// Every block forms the same norm from the partials, then scales its pieces (N = 0: none).
template <int N, int P>
__global__ void __launch_bounds__(32 * kWarps, kBlocksPerSm)
grad_scale_kernel(const __grid_constant__ GradTable<N> t, const double* partial, int partials,
                  float max_norm, int clip, float* norm_out) {
  __shared__ double red[kWarps];
  __shared__ float coef_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait_and_trigger();
  double acc = 0.0;
  for (int i = threadIdx.x; i < partials; i += 32 * kWarps) acc = join<P>(acc, partial[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc = join<P>(acc, __shfl_xor_sync(0xffffffffu, acc, o));
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s = join<P>(s, red[w]);
    const double norm = P == 2 ? sqrt(s) : s;
    if (blockIdx.x == 0 && norm_out) *norm_out = static_cast<float>(norm);
    // NaN stays NaN (and so do the gradients), an infinite norm gives 0
    const double c = static_cast<double>(max_norm) / (norm + 1e-6);
    coef_s = c > 1.0 ? 1.f : static_cast<float>(c);
  }
  __syncthreads();
  const float coef = coef_s;
  if (!clip || coef == 1.f) return;
  const int total = t.end_piece[t.n - 1];
  for (int k = total - 1 - (blockIdx.x * kWarps + warp); k >= 0; k -= gridDim.x * kWarps) {
    const int i = tensor_of(t, k);
    const int64_t at = k - (i ? t.end_piece[i - 1] : 0);
    auto run = [&](auto* p, int64_t count) {
      using T = std::remove_reference_t<decltype(*p)>;
      int64_t first, last;
      piece_range(p, count, at, t.piece, first, last);
      walk(p + first, static_cast<int>(last - first), lane, [&](T* q) { *q = Elt<T>::from_f(Elt<T>::to_f(*q) * coef); },
           [&](T* q, uint4 v) {
             float f[16 / sizeof(T)];
             unpack<T>(v, f);
#pragma unroll
             for (int j = 0; j < 16 / static_cast<int>(sizeof(T)); ++j) f[j] *= coef;
             store16_from_f(q, f);
           });
    };
    if (t.count[i] < 0) run(static_cast<__nv_bfloat16*>(t.ptr[i]), -t.count[i]);
    else run(static_cast<float*>(t.ptr[i]), t.count[i]);
  }
}

int64_t pieces_of(const void* p, int64_t count, int dtype, int piece) {
  const int64_t elt = dtype == kF32 ? 4 : 2;
  const int64_t head = ((16 - static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) & 15u)) & 15) / elt;
  const int64_t per = piece / elt;
  const int64_t rest = count - head;
  return rest <= 0 ? 1 : (rest + per - 1) / per;
}

struct GradList {
  void* const* ptrs;
  const int64_t* counts;
  const int32_t* dtypes;
  int n;
};

template <int N, int P>
cudaError_t run_list(const GradList& l, float max_norm, bool clip, float* norm, double* partial,
                     int num_sms, cudaStream_t s) {
  const int max_blocks = num_sms * kBlocksPerSm;
  int64_t bytes = 0;
  for (int i = 0; i < l.n; ++i) bytes += l.counts[i] * static_cast<int64_t>(dtype_bytes(l.dtypes[i]));
  int piece = kMaxPiece;
  while (piece > kMinPiece && bytes / piece < static_cast<int64_t>(max_blocks) * kWarps) piece /= 2;
  int partials = 0;
  bool first = true;
  for (int pass = 0; pass < (clip ? 2 : 1); ++pass) {
    const int all = partials;
    for (int at = 0; at < l.n;) {
      GradTable<N> t;
      int64_t total = 0;
      t.n = 0;
      t.piece = piece;
      for (; at < l.n && t.n < N; ++at) {
        if (l.counts[at] == 0) continue;
        const int64_t more = pieces_of(l.ptrs[at], l.counts[at], l.dtypes[at], piece);
        if (total + more > 0x3fffffff) {
          if (t.n == 0) return cudaErrorInvalidValue;
          break;
        }
        total += more;
        t.ptr[t.n] = l.ptrs[at];
        t.count[t.n] = l.dtypes[at] == kBF16 ? -l.counts[at] : l.counts[at];
        t.end_piece[t.n++] = static_cast<int32_t>(total);
      }
      if (t.n == 0) break;
      const int64_t want = (total + kWarps - 1) / kWarps;
      const unsigned blocks = static_cast<unsigned>(want < max_blocks ? want : max_blocks);
      // the first kernel of the call follows the caller's work in full; the later ones may
      // launch while the one before ends
      PdlScope pdl(!first);
      first = false;
      cudaError_t e;
      if (pass == 0) {
        t.first_partial = partials;
        partials += static_cast<int>(blocks);
        e = launch_kernel(grad_norm_kernel<N, P>, dim3(blocks), dim3(32 * kWarps), 0, s, t, partial);
      } else {
        e = launch_kernel(grad_scale_kernel<N, P>, dim3(blocks), dim3(32 * kWarps), 0, s, t,
                          static_cast<const double*>(partial), all, max_norm, 1, norm);
      }
      if (e != cudaSuccess) return e;
    }
  }
  if (!clip || partials == 0) {  // the norm alone (of nothing: 0)
    GradTable<1> none;
    PdlScope pdl(!first);
    return launch_kernel(grad_scale_kernel<1, P>, dim3(1), dim3(32 * kWarps), 0, s, none,
                         static_cast<const double*>(partial), partials, max_norm, 0, norm);
  }
  return cudaSuccess;
}

template <int N>
cudaError_t run_norm(int p, const GradList& l, float max_norm, bool clip, float* norm,
                     double* partial, int num_sms, cudaStream_t s) {
  if (p == 2) return run_list<N, 2>(l, max_norm, clip, norm, partial, num_sms, s);
  if (p == 1) return run_list<N, 1>(l, max_norm, clip, norm, partial, num_sms, s);
  return run_list<N, 0>(l, max_norm, clip, norm, partial, num_sms, s);
}

}  // namespace
}  // namespace vmoe

namespace {
size_t norm_workspace(const vmoe_ops* o, int n) {
  // launches take kBatch tensors each (fewer only past 2^30 pieces, 16 TB)
  const size_t launches = static_cast<size_t>(n) / kBatch + 2;
  return launches * static_cast<size_t>(o->num_sms) * kBlocksPerSm * sizeof(double);
}
}  // namespace

extern "C" {

int vmoe_grad_norm_workspace_size(vmoe_ops* o, int n, size_t* bytes) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (!bytes || n < 0) return ops_fail(o, VMOE_ERR_INVALID_ARG, "bytes and n >= 0 are required");
  *bytes = norm_workspace(o, n);
  return VMOE_OK;
}

int vmoe_grad_norm(vmoe_ops* o, void* const* tensors, const int64_t* counts, const int32_t* dtypes,
                   int n, int norm_type, float max_norm, float* total_norm, void* workspace,
                   size_t workspace_bytes, void* stream) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (n < 0 || (n > 0 && (!tensors || !counts || !dtypes)))
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "tensors, counts and dtypes are required");
  if (norm_type != VMOE_NORM_1 && norm_type != VMOE_NORM_2 && norm_type != VMOE_NORM_INF)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "unknown norm type %d", norm_type);
  if (max_norm != max_norm)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "max_norm is not a number");
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0 || counts[i] >= (static_cast<int64_t>(1) << 42))
      return ops_fail(o, VMOE_ERR_INVALID_ARG, "tensor %d has %lld elements", i,
                      static_cast<long long>(counts[i]));
    if (counts[i] == 0) continue;
    if (dtypes[i] != VMOE_F32 && dtypes[i] != VMOE_BF16)
      return ops_fail(o, VMOE_ERR_INVALID_ARG, "tensor %d: dtype must be VMOE_F32 or VMOE_BF16", i);
    if (!tensors[i] || reinterpret_cast<uintptr_t>(tensors[i]) % dtype_bytes(dtypes[i]))
      return ops_fail(o, VMOE_ERR_INVALID_ARG, "tensor %d is null or not aligned to its elements", i);
  }
  if (reinterpret_cast<uintptr_t>(total_norm) % sizeof(float))
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "total_norm is not aligned to its element");
  const size_t need = norm_workspace(o, n);
  if (!workspace || workspace_bytes < need)
    return ops_fail(o, VMOE_ERR_WORKSPACE, "workspace needs %zu bytes (got %zu)", need,
                    workspace ? workspace_bytes : static_cast<size_t>(0));
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return ops_fail(o, VMOE_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  DeviceGuard g(o->device);
  const GradList l{tensors, counts, dtypes, n};
  const bool clip = max_norm >= 0.f;
  auto* partial = static_cast<double*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      n <= kSmallBatch ? run_norm<kSmallBatch>(norm_type, l, max_norm, clip, total_norm, partial,
                                               o->num_sms, s)
                       : run_norm<kBatch>(norm_type, l, max_norm, clip, total_norm, partial,
                                          o->num_sms, s);
  return e == cudaSuccess ? VMOE_OK : ops_cuda_fail(o, e, "gradient norm");
}

}  // extern "C"
