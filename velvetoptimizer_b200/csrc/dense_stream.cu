// Fused linear and gated projection for few rows (T <= 16) and many output features: weights
// streamed through shared memory by bulk copies.
//
//   out[t, n] = epilogue(sum_k w[n, k] x[t, k])
//
// The same arithmetic as dense_small.cu (mma.sync m16n8k16, 16 weight rows as M, tokens as N,
// the k permutation that lets a lane read 16 consecutive bytes), but a block is persistent: a
// producer warp copies the 16 rows of the next tiles, up to 2048 k at a time, row by row
// (cp.async.bulk) into a ring of about 200 KB, while 8 warps multiply the current one.  What a
// block waits for between two tiles in the register form (its loads, the sum over its warps,
// the next block's start) is spent with the ring filling, so HBM sees requests all the time.
// Rows lie 16 bytes apart from a multiple of 128 in shared memory, which keeps the 8 rows a
// fragment load touches in different banks.
// Bound by HBM.  Block 2048 x 8192, one row: 22.3 us for its 100.7 MB (4.5 TB/s).
#include <atomic>

#include "common.cuh"
#include "dense.h"
#include "dense_act.cuh"

namespace vmoe {
namespace {

constexpr int WARPS = 8;              // multiplying warps; one more copies
constexpr int SLICE = 2048;           // k per stage
constexpr int CHUNKS = SLICE / 32 / WARPS;  // 32-wide chunks of a slice per warp
constexpr int MAX_STAGES = 8;
constexpr size_t RING_LIMIT = 200 * 1024;

template <int NT>
struct Shared {
  uint64_t full[MAX_STAGES];
  uint64_t empty[MAX_STAGES];
  int abort;
  alignas(16) float4 red[2][WARPS][NT][32];
  float sum[2][NT][16][8];
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void sync_multipliers() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
}

template <int EPI, int NT>
__global__ void __launch_bounds__(32 * (WARPS + 1), 1)
dense_stream_kernel(const __grid_constant__ SmallGemm g, const int stages, const uint32_t pitch) {
  constexpr bool kGate = EPI == kEpiGated;
  constexpr int ROWS = kGate ? 8 : 16;  // output features per tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 127u) & ~127u;
  const uint32_t stage_bytes = 16 * pitch;
  auto* sh = reinterpret_cast<Shared<NT>*>(smem_raw + (ring - smem_u32(smem_raw)) +
                                           ((stages * stage_bytes + 127) & ~127u));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = static_cast<int>((g.N + ROWS - 1) / ROWS);
  const int slices = static_cast<int>((g.K + SLICE - 1) / SLICE);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), WARPS);
    }
    sh->abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  // in a call's second kernel the weights were there before its first began
  if (!(g.early_weights && warp == WARPS)) pdl_wait_and_trigger();
  auto aborted = [&] { return *reinterpret_cast<volatile int*>(&sh->abort) != 0; };
  auto give_up = [&](int code) {
    *reinterpret_cast<volatile int*>(&sh->abort) = 1;
    report(g.status, code);
  };

  if (warp == WARPS) {
    int it = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
      const int64_t n0 = static_cast<int64_t>(tile) * ROWS;
      const int64_t row = n0 + (kGate ? lane & 7 : lane);
      const auto* base = static_cast<const __nv_bfloat16*>(kGate && lane >= 8 ? g.w2 : g.w) +
                         row * (kGate && lane >= 8 ? g.ldw2 : g.ldw);
      const bool mine = lane < 16 && row < g.N;
      const uint32_t rows = __popc(__ballot_sync(0xffffffffu, mine));
      for (int sl = 0; sl < slices; ++sl, ++it) {
        const int s = it % stages;
        if (!mbar_wait(smem_u32(&sh->empty[s]), ((it / stages) & 1) ^ 1)) {
          give_up(kStatusTimeoutProducer);
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok) && !aborted();
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int64_t k0 = static_cast<int64_t>(sl) * SLICE;
        const uint32_t bytes = static_cast<uint32_t>((g.K - k0 < SLICE ? g.K - k0 : SLICE) * 2);
        const uint32_t fb = smem_u32(&sh->full[s]);
        if (lane == 0) mbar_arrive_expect_tx(fb, rows * bytes);
        __syncwarp();
        if (mine) bulk_load(ring + s * stage_bytes + lane * pitch, base + k0, bytes, fb);
      }
    }
    // copies still in flight land before the block ends: the multipliers wait for every stage;
    // after an abort they may not, so give them a bounded time
    if (aborted()) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) {
      }
    }
  } else {
    const int gid = lane >> 2, tig = lane & 3;
    const auto* x = static_cast<const __nv_bfloat16*>(g.x);
    uint4 xv[CHUNKS][NT];
    int it = 0, buf = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, buf ^= 1) {
      float acc[NT][4] = {};
      // this thread's output, and what its epilogue reads, asked for before the weights' wait
      const DenseEpi& ep = g.epi;
      const int f = threadIdx.x % ROWS, t = threadIdx.x / ROWS;
      const int64_t col = static_cast<int64_t>(tile) * ROWS + f;
      const bool mine = t < g.T && t < NT * 8 && col < g.N;
      auto read = [&](const void* p, int64_t i) {
        return p && mine ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : 0.f;
      };
      const float b0 = read(ep.bias, col), b1 = kGate ? read(ep.bias2, col) : 0.f;
      const float res = kGate ? 0.f : read(ep.res, t * ep.ldr + col);
      for (int sl = 0; sl < slices; ++sl, ++it) {
        const int64_t k0 = static_cast<int64_t>(sl) * SLICE + tig * 8;
        if (slices > 1 || it == 0) {  // one slice: the same tokens for every tile
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int64_t k = k0 + (warp + c * WARPS) * 32, t = n * 8 + gid;
              xv[c][n] = make_uint4(0, 0, 0, 0);
              if (t < g.T && k < g.K)
                xv[c][n] = __ldg(reinterpret_cast<const uint4*>(x + t * g.ldx + k));
            }
        }
        const int s = it % stages;
        if (ok && !mbar_wait(smem_u32(&sh->full[s]), (it / stages) & 1)) {
          give_up(kStatusTimeoutMma);
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint8_t* at = smem_raw + (ring - smem_u32(smem_raw)) + s * stage_bytes + gid * pitch + tig * 16;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const int chunk = warp + c * WARPS;
          uint4 a = make_uint4(0, 0, 0, 0), b = a;
          if (k0 + chunk * 32 < g.K) {
            a = *reinterpret_cast<const uint4*>(at + chunk * 64);
            b = *reinterpret_cast<const uint4*>(at + 8 * pitch + chunk * 64);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_bf16(acc[n], a.x, b.x, a.y, b.y, xv[c][n].x, xv[c][n].y);
            mma_bf16(acc[n], a.z, b.z, a.w, b.w, xv[c][n].z, xv[c][n].w);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->empty[s]));
      }
      // the sum over the warps, in warp order (two buffers: one barrier pair per tile)
#pragma unroll
      for (int n = 0; n < NT; ++n)
        sh->red[buf][warp][n][lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
      sync_multipliers();
      if (threadIdx.x < NT * 128) {
        const int n = threadIdx.x >> 7, l = (threadIdx.x >> 2) & 31, i = threadIdx.x & 3;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k)
          s += reinterpret_cast<const float*>(&sh->red[buf][k][n][l])[i];
        sh->sum[buf][n][(l >> 2) + 8 * (i >> 1)][(l & 3) * 2 + (i & 1)] = s;
      }
      sync_multipliers();
      if (ok && mine) {
        float z = sh->sum[buf][t >> 3][f][t & 7] + b0;
        if constexpr (kGate) {
          const float up = sh->sum[buf][t >> 3][f + 8][t & 7] + b1;
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
        static_cast<__nv_bfloat16*>(ep.out)[t * ep.ldo + col] = __float2bfloat16_rn(z);
      }
    }
  }
}

template <int EPI, int NT>
cudaError_t launch(const SmallGemm& g, cudaStream_t s) {
  auto kern = dense_stream_kernel<EPI, NT>;
  const int rows = EPI == kEpiGated ? 8 : 16;
  const int64_t tiles = (g.N + rows - 1) / rows;
  const int64_t width = g.K < SLICE ? g.K : SLICE;
  const uint32_t pitch = static_cast<uint32_t>((width * 2 + 127) / 128 * 128 + 16);
  int stages = static_cast<int>(RING_LIMIT / (16 * pitch));
  if (stages > MAX_STAGES) stages = MAX_STAGES;
  const size_t smem = 128 + ((static_cast<size_t>(stages) * 16 * pitch + 127) & ~static_cast<size_t>(127)) +
                      sizeof(Shared<NT>);
  cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(RING_LIMIT + 256 + sizeof(Shared<NT>)));
  if (err != cudaSuccess) return err;
  const unsigned blocks = static_cast<unsigned>(tiles < g.num_sms ? tiles : g.num_sms);
  return launch_kernel(kern, dim3(blocks), dim3(32 * (WARPS + 1)), smem, s, g, stages, pitch);
}

}  // namespace

cudaError_t launch_dense_stream(int epi, const SmallGemm& g, cudaStream_t s) {
  if (g.T < 1 || g.T > kSmallTokens || !g.vec_in || g.epi.out_f32) return cudaErrorInvalidValue;
  if (epi == kEpiGated)
    return g.T <= 8 ? launch<kEpiGated, 1>(g, s) : launch<kEpiGated, 2>(g, s);
  return g.T <= 8 ? launch<kEpiLinear, 1>(g, s) : launch<kEpiLinear, 2>(g, s);
}

}  // namespace vmoe
