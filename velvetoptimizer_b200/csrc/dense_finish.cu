// The elementwise and column kernels around the dense products.
//
//   finish   sums a split product's fp32 partials in split order and runs the epilogue
//   dz       dz = dy act'(z) with the column sums of dz (the bias gradient) in the same pass;
//            also the plain column sums, and the copy of dy to a pitch the TMA can read
//   colsum   adds the row blocks' column sums in block order
// All are bound by the bytes they move: 16-byte accesses where the buffers allow them.
// dz of 16,384 x 2048, bf16: 43 us for 201 MB (4.7 TB/s).
#include "common.cuh"
#include "dense.h"
#include "dense_act.cuh"
#include "dense_finish.cuh"

namespace vmoe {
namespace {

template <typename T, int EPI>
__global__ void __launch_bounds__(256)
dense_finish_kernel(const DenseGemm g) {
  pdl_wait_and_trigger();
  const int64_t per_row = (g.N + kChunk - 1) / kChunk;
  const int64_t total = g.M * per_row;
  const int grp = blockIdx.y;
  bool redo = false;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t row = i / per_row, col = (i - row * per_row) * kChunk;
    float v[kChunk], u[kChunk];
    chunk_sums<EPI>(g, grp, row, col, v, u);
    if constexpr (sizeof(T) == 4) {
      if (g.redo && !chunk_finite<EPI>(v, u, g.N - col)) {
        // left to dense_redo_kernel, and marked in every split's partials
        redo = true;
        float* p = partial_at<EPI>(g, grp, row, col);
        for (int s = 0; s < g.splits; ++s) p[s * split_stride(g)] = __int_as_float(0x7fffffff);
        continue;
      }
    }
    finish_chunk<T, EPI>(g, grp, row, col, v, u);
  }
  if constexpr (sizeof(T) == 4) {
    if (redo) *g.redo = 1;
    if (g.arrived && grp == 0)
      for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < g.redo_tiles; i += gridDim.x * 256ll)
        g.arrived[i] = 0;
  }
}

// Four rows per thread in flight: with one, 201 MB (16,384 x 2048, silu) took 61 us.
template <typename T>
__global__ void __launch_bounds__(256, 3)
dense_dz_kernel(const DzArgs a, bool vec_dy, bool vec_z, bool vec_dz) {
  constexpr int W = Vec16<T>::N;
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int ROWS = 4;
  __shared__ float red[8][32 * W];
  pdl_wait_and_trigger();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * 32 + tx) * W;
  const int64_t valid = a.N - col;
  const int64_t r0 = blockIdx.y * a.rows_per_block;
  const int64_t r1 = min(a.T, r0 + a.rows_per_block);
  float sum[W] = {};
  if (valid > 0) {
    const T* dy = static_cast<const T*>(a.dy) + col;
    const T* z = static_cast<const T*>(a.z) + col;
    T* dz = static_cast<T*>(a.dz) + col;
    auto scale = [&](float (&v)[W], float (&g)[W]) {
      act_switch(a.act, [&](auto A) {
        float d[W];
        act_grads<kFast, decltype(A)::value>(g, d, a.gamma);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = times_slope<decltype(A)::value>(v[j], d[j]);
      });
    };
    auto finish = [&](float (&v)[W], int64_t r) {
      if (a.dz) store_row<W>(dz + r * a.lddz, v, valid, vec_dz);
#pragma unroll
      for (int j = 0; j < W; ++j) sum[j] += v[j];
    };
    int64_t r = r0 + ty;
    if (vec_dy && (vec_z || a.act == kActNone) && valid >= W) {
      for (; r + 8 * (ROWS - 1) < r1; r += 8 * ROWS) {
        uint4 pv[ROWS], pz[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
          pv[i] = __ldg(reinterpret_cast<const uint4*>(dy + (r + 8 * i) * a.lddy));
        if (a.act != kActNone) {
#pragma unroll
          for (int i = 0; i < ROWS; ++i)
            pz[i] = __ldg(reinterpret_cast<const uint4*>(z + (r + 8 * i) * a.ldz));
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          float v[W], g[W];
          load16_to_f(reinterpret_cast<const T*>(&pv[i]), v);
          if (a.act != kActNone) {
            load16_to_f(reinterpret_cast<const T*>(&pz[i]), g);
            scale(v, g);
          }
          finish(v, r + 8 * i);
        }
      }
    }
    for (; r < r1; r += 8) {
      float v[W], g[W];
      load_row<W>(dy + r * a.lddy, v, valid, vec_dy);
      if (a.act != kActNone) {
        load_row<W>(z + r * a.ldz, g, valid, vec_z);
        scale(v, g);
      }
      finish(v, r);
    }
  }
  if (!a.colsum && !a.db) return;
#pragma unroll
  for (int j = 0; j < W; ++j) red[ty][tx * W + j] = sum[j];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * W; c += 256) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 32 * W + c;
    if (n >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += red[k][c];
    if (!a.db) a.colsum[blockIdx.y * a.N + n] = s;
    else if (a.db_f32) static_cast<float*>(a.db)[n] = s;
    else static_cast<T*>(a.db)[n] = Elt<T>::from_f(s);
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
colsum_finish_kernel(const float* partial, int64_t row_blocks, int64_t N, T* out, T* out2) {
  __shared__ float red[8][32];
  if (blockIdx.y == 1) {
    partial += row_blocks * N;
    out = out2;
  }
  pdl_wait_and_trigger();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t n = blockIdx.x * 32ll + tx;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int64_t b = ty; b < row_blocks; b += 8) s += partial[b * N + n];
  }
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && n < N) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][tx];
    out[n] = Elt<T>::from_f(s);
  }
}

// 8 elements per thread: scalar reads from anywhere, one 16-byte store
__global__ void __launch_bounds__(256)
pad_copy_kernel(const unsigned short* src, int64_t lds, int64_t rows, int64_t cols,
                unsigned short* dst, int64_t ldd) {
  pdl_wait_and_trigger();
  const int units = static_cast<int>(ldd / 8);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const unsigned short* p = src + r * lds;
    for (int64_t u = threadIdx.x; u < units; u += 256) {
      uint32_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = u * 8 + j < cols ? __ldg(p + u * 8 + j) : 0u;
      *reinterpret_cast<uint4*>(dst + r * ldd + u * 8) =
          make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
  }
}

unsigned blocks_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256;
  return static_cast<unsigned>(b < 148 * 16 ? (b > 0 ? b : 1) : 148 * 16);
}

template <typename T>
bool vec_ok(const void* p, int64_t ld) {
  return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * sizeof(T))) & 15u) == 0;
}

}  // namespace

cudaError_t launch_dense_finish(int dtype, int epi, const DenseGemm& g, cudaStream_t s) {
  const dim3 grid(blocks_for(g.M * ((g.N + kChunk - 1) / kChunk)), static_cast<unsigned>(g.groups));
  cudaError_t e;
  if (dtype == kF32) {
    if (epi == kEpiGated) e = launch_kernel(dense_finish_kernel<float, kEpiGated>, grid, dim3(256), 0, s, g);
    else if (epi == kEpiGluBwd) e = launch_kernel(dense_finish_kernel<float, kEpiGluBwd>, grid, dim3(256), 0, s, g);
    else e = launch_kernel(dense_finish_kernel<float, kEpiLinear>, grid, dim3(256), 0, s, g);
  } else {
    using B = __nv_bfloat16;
    if (epi == kEpiGated) e = launch_kernel(dense_finish_kernel<B, kEpiGated>, grid, dim3(256), 0, s, g);
    else if (epi == kEpiGluBwd) e = launch_kernel(dense_finish_kernel<B, kEpiGluBwd>, grid, dim3(256), 0, s, g);
    else e = launch_kernel(dense_finish_kernel<B, kEpiLinear>, grid, dim3(256), 0, s, g);
  }
  return e;
}

cudaError_t launch_dense_dz(int dtype, const DzArgs& a, cudaStream_t s) {
  const int width = 32 * (dtype == kF32 ? 4 : 8);
  const dim3 grid(static_cast<unsigned>((a.N + width - 1) / width),
                  static_cast<unsigned>(a.row_blocks));
  using B = __nv_bfloat16;
  if (dtype == kF32)
    return launch_kernel(dense_dz_kernel<float>, grid, dim3(256), 0, s, a,
                         vec_ok<float>(a.dy, a.lddy), vec_ok<float>(a.z, a.ldz),
                         vec_ok<float>(a.dz, a.lddz));
  return launch_kernel(dense_dz_kernel<B>, grid, dim3(256), 0, s, a, vec_ok<B>(a.dy, a.lddy),
                       vec_ok<B>(a.z, a.ldz), vec_ok<B>(a.dz, a.lddz));
}

cudaError_t launch_colsum_finish(const float* partial, int64_t row_blocks, int64_t N, void* out,
                                 void* out2, bool out_f32, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((N + 31) / 32), out2 ? 2 : 1);
  if (out_f32)
    return launch_kernel(colsum_finish_kernel<float>, grid, dim3(256), 0, s, partial, row_blocks, N,
                         static_cast<float*>(out), static_cast<float*>(out2));
  return launch_kernel(colsum_finish_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, partial, row_blocks,
                       N, static_cast<__nv_bfloat16*>(out), static_cast<__nv_bfloat16*>(out2));
}

cudaError_t launch_pad_copy(const void* src, int64_t lds, int64_t rows, int64_t cols, void* dst,
                            int64_t ldd, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>(rows < 148 * 16 ? rows : 148 * 16);
  return launch_kernel(pad_copy_kernel, dim3(blocks), dim3(256), 0, s,
                       static_cast<const unsigned short*>(src), lds, rows, cols,
                       static_cast<unsigned short*>(dst), ldd);
}

}  // namespace vmoe
