// Fused linear and gated projection for a decode batch (17 to 128 rows): the weights stream
// through the tensor cores as the MMA's M operand, the tokens are its N.
//
//   D[feature, token] = sum_k w[feature, k] x[token, k]
//
// Bound: the weights are read once from HBM.  A CTA takes 128 features (gated: 64 gate and 64
// up rows of the same features) and a share of k, M128 with N = T rounded up to 16, so no
// stage byte is spent on rows that do not exist and the ring holds the weights of many k
// blocks in flight.  Features alone leave SMs idle, so k is divided over the CTAs of a cluster
// (up to 8): each sends the fp32 sums of the others' tokens into their shared memory, and each
// adds its own tokens' parts in rank order and runs the epilogue for them.  One launch, no
// partial sums in global memory, no atomics.  TMEM lanes are features, so a warp's stores of
// one token are 32 consecutive features without a transpose.
// 64 rows, cold weights, K x N: 2048 x 8192 12.8 us, 4096 x 8192 19.3 (5.2 TB/s between the two),
// 64 x 8192 5.3, which is what launch, ring fill and exchange cost; 8192 x 2048 14.9.
// Every mbarrier wait is bounded; a CTA that gives up still takes both cluster barriers.
#include <atomic>

#include "common.cuh"
#include "dense.h"
#include "dense_act.cuh"

namespace vmoe {
namespace {

constexpr int BK = 64;
constexpr uint32_t W_BYTES = 128 * BK * 2;  // 16 KB of weights a stage
constexpr int MAX_STAGES = 12;
constexpr int EPI_WARPS = 8;  // two per TMEM lane quarter, each half of the tokens
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int kMaxDevices = 64;
constexpr size_t SMEM_LIMIT = 224 * 1024;  // ring and exchange

struct Shared {
  uint64_t full[MAX_STAGES];
  uint64_t empty[MAX_STAGES];
  uint64_t done;
  uint32_t tmem_base;
  int abort;
};

__device__ __forceinline__ bool aborted(const Shared* sh) {
  return *reinterpret_cast<const volatile int*>(&sh->abort) != 0;
}
__device__ __forceinline__ void set_abort(Shared* sh, int* status, int code) {
  *reinterpret_cast<volatile int*>(&sh->abort) = 1;
  report(status, code);
}

__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// the first n of a thread's values, GROUPS rows apart
template <int GROUPS, typename T, int PER>
__device__ __forceinline__ void store_rows(T* p, int64_t ld, const float (&v)[PER], int n) {
#pragma unroll
  for (int i = 0; i < PER; ++i, p += GROUPS * ld)
    if (i < n) *p = Elt<T>::from_f(v[i]);
}

template <int EPI>
__global__ void __launch_bounds__(THREADS, 1)
dense_skinny_kernel(const __grid_constant__ CUtensorMap w_map,
                    const __grid_constant__ CUtensorMap w2_map,
                    const __grid_constant__ CUtensorMap x_map,
                    const __grid_constant__ SkinnyGemm g) {
  constexpr bool kGate = EPI == kEpiGated;
  constexpr int FEATURES = kGate ? 64 : 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t x_bytes = static_cast<uint32_t>(g.t_pad) * BK * 2;
  const uint32_t stage_bytes = W_BYTES + x_bytes;
  auto* sh = reinterpret_cast<Shared*>(gbase + g.ring_bytes + g.exchange_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = g.parts;  // CTAs of the cluster
  const int rank = parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / parts;
  const int kb0 = rank * g.kb_per_part;
  const int kb1 = min(g.kbs, kb0 + g.kb_per_part);

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), 1);
    }
    mbar_init(smem_u32(&sh->done), 1);
    sh->abort = 0;
    fence_mbar_init();
    prefetch_tmap(&w_map);
    prefetch_tmap(&x_map);
  }
  if (warp == 1) tmem_alloc(smem_u32(&sh->tmem_base), g.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  // in a call's second kernel the weights were there before its first began: the producer asks
  // for them, as far as the ring goes, before it waits for the tokens
  const bool early = g.early_weights && warp == 0;
  if (!early) pdl_wait_and_trigger();
  // the others' stores into this CTA's exchange wait for this (at the end of the main loop)
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  if (warp == 0) {
    if (lane == 0) {
      auto weights = [&](int kb, uint32_t fb, uint32_t dst) {
        mbar_arrive_expect_tx(fb, stage_bytes);
        if constexpr (kGate) {
          tma_load_2d(dst, &w_map, fb, kb * BK, tile * 64);
          tma_load_2d(dst + W_BYTES / 2, &w2_map, fb, kb * BK, tile * 64);
        } else {
          tma_load_2d(dst, &w_map, fb, kb * BK, tile * 128);
        }
      };
      const int ahead = early ? min(g.stages, kb1 - kb0) : 0;
      for (int i = 0; i < ahead; ++i)
        weights(kb0 + i, smem_u32(&sh->full[i]), base + i * stage_bytes);
      if (early) pdl_wait_and_trigger();
      int it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % g.stages;
        const uint32_t fb = smem_u32(&sh->full[s]), dst = base + s * stage_bytes;
        if (it >= ahead) {
          const uint32_t ph = (it / g.stages) & 1;
          if (!mbar_wait(smem_u32(&sh->empty[s]), ph ^ 1)) {
            set_abort(sh, g.status, kStatusTimeoutProducer);
            break;
          }
          if (aborted(sh)) break;
          weights(kb, fb, dst);
        }
        tma_load_2d(dst + W_BYTES, &x_map, fb, kb * BK, 0);
      }
      // an abort leaves copies in flight: give them a bounded time before the memory is reused
      if (aborted(sh)) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_bf16(128, g.t_pad);
      int it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % g.stages;
        const uint32_t ph = (it / g.stages) & 1;
        if (!mbar_wait(smem_u32(&sh->full[s]), ph)) {
          set_abort(sh, g.status, kStatusTimeoutMma);
          break;
        }
        tc_fence_after();
        const uint32_t a = base + s * stage_bytes, b = a + W_BYTES;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          umma_bf16(tmem, umma_desc_sw128(a + k * 32), umma_desc_sw128(b + k * 32), idesc,
                    (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit(smem_u32(&sh->empty[s]));
      }
      umma_commit(smem_u32(&sh->done));
    }
    __syncwarp();
  }
  // an epilogue thread's feature, and its biases before the product is done
  const int f = static_cast<int>(threadIdx.x - 64) % FEATURES;
  const int group = static_cast<int>(threadIdx.x - 64) / FEATURES;
  const int64_t col = static_cast<int64_t>(tile) * FEATURES + f;
  const DenseEpi& ep = g.epi;
  auto bias = [&](const void* p) {
    return warp >= 2 && p && col < g.N
               ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[col])
               : 0.f;
  };
  const float b0 = bias(ep.bias), b1 = kGate ? bias(ep.bias2) : 0.f;
  // every thread: the product is complete (all copies landed, all stages read)
  if (!mbar_wait(smem_u32(&sh->done), 0)) set_abort(sh, g.status, kStatusTimeoutDrain);
  __syncwarp();
  tc_fence_after();
  // The exchange, beside the ring (others may still read theirs).  Tokens go in chunks of 16;
  // CTA c % parts finishes chunk c, in its slot c / parts: [part][16 tokens][128 rows] of fp32.
  if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  constexpr uint32_t CHUNK = 16 * 128 * 4;
  const int chunks = g.t_pad / 16;
  const uint32_t exchange = base + g.ring_bytes;
  if (warp >= 2) {
    const int q = warp & 3;
#pragma unroll 1
    for (int c = (warp - 2) >> 2; c < chunks; c += EPI_WARPS / 4) {
      float v[16];
      __syncwarp();
      tmem_ld16(tmem + (static_cast<uint32_t>(q * 32) << 16) + c * 16, v);
      const int slot = c / parts;
      uint32_t at = exchange + (slot * parts + rank) * CHUNK + (q * 32 + lane) * 4;
      if (parts > 1) {
        at = mapa_shared(at, static_cast<uint32_t>(c - slot * parts));
#pragma unroll
        for (int j = 0; j < 16; ++j) st_cluster(at + j * 512, v[j]);
      } else {
        float* own = reinterpret_cast<float*>(smem_raw + (at - raw));
#pragma unroll
        for (int j = 0; j < 16; ++j) own[j * 128] = v[j];
      }
    }
    tc_fence_before();
  }
  if (parts > 1) cluster_sync_all(); else __syncthreads();
  if (warp >= 2) {
    // a thread per feature: PER of a chunk's 16 tokens, GROUPS apart
    constexpr int GROUPS = 32 * EPI_WARPS / FEATURES, PER = 16 / GROUPS;
    act_switch(ep.act, [&](auto A) {
#pragma unroll 1
      for (int c = rank, slot = 0; c < chunks; c += parts, ++slot) {
        const int64_t t0 = c * 16 + group;
        // this thread's tokens of the chunk that exist
        const int64_t left = g.T - t0;
        const int n = col >= g.N || left <= 0
                          ? 0
                          : static_cast<int>(min((left + GROUPS - 1) / GROUPS, static_cast<int64_t>(PER)));
        float z[PER], up[PER], r[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          z[i] = b0;
          up[i] = b1;
          r[i] = 0.f;
        }
        if (!kGate && ep.res) {
          const auto* p = static_cast<const __nv_bfloat16*>(ep.res) + t0 * ep.ldr + col;
#pragma unroll
          for (int i = 0; i < PER; ++i, p += GROUPS * ep.ldr)
            if (i < n) r[i] = __bfloat162float(*p);
        }
        const float* sums = reinterpret_cast<const float*>(
            gbase + g.ring_bytes + static_cast<uint32_t>(slot * parts) * CHUNK) + group * 128 + f;
        for (int p = 0; p < parts; ++p, sums += CHUNK / 4) {
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            z[i] += sums[i * GROUPS * 128];
            if constexpr (kGate) up[i] += sums[i * GROUPS * 128 + 64];
          }
        }
        if (ep.z) {
          if constexpr (kGate) {
            store_rows<GROUPS>(static_cast<float*>(ep.z) + t0 * ep.ldz + col, ep.ldz, z, n);
            store_rows<GROUPS>(static_cast<float*>(ep.z2) + t0 * ep.ldz + col, ep.ldz, up, n);
          } else {
            store_rows<GROUPS>(static_cast<__nv_bfloat16*>(ep.z) + t0 * ep.ldz + col, ep.ldz, z, n);
          }
        }
        act_values<true, decltype(A)::value>(z, ep.gamma);
#pragma unroll
        for (int i = 0; i < PER; ++i) z[i] = kGate ? z[i] * up[i] : z[i] + r[i];
        store_rows<GROUPS>(static_cast<__nv_bfloat16*>(ep.out) + t0 * ep.ldo + col, ep.ldo, z, n);
      }
    });
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, g.tmem_cols);
  }
}

template <int EPI>
cudaLaunchConfig_t config(cudaLaunchAttribute* attr, int parts, int64_t tiles, size_t smem,
                          cudaStream_t s) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = g_launch_pdl ? 2 : 1;
  return cfg;
}

// Clusters of `parts` CTAs that can run at once (a cluster lives in one GPC, so 8 x 16 CTAs
// may not fit where 7 x 18 do); every launch has one CTA per SM.
template <int EPI>
cudaError_t resident(int parts, int* clusters) {
  static std::atomic<int> known[kMaxDevices][9];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < kMaxDevices && (*clusters = known[dev][parts].load(std::memory_order_relaxed)) > 0)
    return cudaSuccess;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = config<EPI>(attr, parts, 148, SMEM_LIMIT, nullptr);
  cfg.numAttrs = 1;
  err = cudaOccupancyMaxActiveClusters(
      clusters, reinterpret_cast<const void*>(dense_skinny_kernel<EPI>), &cfg);
  if (err != cudaSuccess) return err;
  if (dev < kMaxDevices) known[dev][parts].store(*clusters, std::memory_order_relaxed);
  return cudaSuccess;
}

template <int EPI>
cudaError_t launch(const CUtensorMap& w, const CUtensorMap& w2, const CUtensorMap& x,
                   SkinnyGemm g, cudaStream_t s) {
  auto kern = dense_skinny_kernel<EPI>;
  cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(SMEM_LIMIT + 2048));
  if (err != cudaSuccess) return err;
  const int features = EPI == kEpiGated ? 64 : 128;
  const int64_t tiles = (g.N + features - 1) / features;
  if (tiles > 0xffffff) return cudaErrorInvalidValue;
  g.t_pad = static_cast<int>((g.T + 15) / 16 * 16);
  g.tmem_cols = 32;
  while (g.tmem_cols < static_cast<uint32_t>(g.t_pad)) g.tmem_cols *= 2;
  // as many parts as all run at once, each with two k blocks or more
  int parts = 1;
  for (int p = 2; p <= 8 && p <= g.kbs / 2; ++p) {
    int clusters = 0;
    if ((err = resident<EPI>(p, &clusters)) != cudaSuccess) return err;
    if (tiles <= clusters) parts = p;
  }
  g.kb_per_part = (g.kbs + parts - 1) / parts;
  g.parts = (g.kbs + g.kb_per_part - 1) / g.kb_per_part;
  const size_t stage = W_BYTES + static_cast<size_t>(g.t_pad) * BK * 2;
  // the exchange: 8 KB for each part of each of this CTA's 16-token chunks
  const size_t chunks = static_cast<size_t>(g.t_pad) / 16;
  const size_t exchange = (chunks + g.parts - 1) / g.parts * g.parts * 8192;
  size_t stages = (SMEM_LIMIT - exchange) / stage;
  if (stages > MAX_STAGES) stages = MAX_STAGES;
  if (stages > static_cast<size_t>(g.kb_per_part)) stages = static_cast<size_t>(g.kb_per_part);
  g.stages = static_cast<int>(stages);
  g.ring_bytes = static_cast<uint32_t>(stages * stage);
  g.exchange_bytes = static_cast<uint32_t>(exchange);
  // more than half of an SM's shared memory, so that no second CTA with TMEM shares the SM: one
  // that waited for TMEM while its cluster's others hold theirs might wait for good
  size_t smem = 1024 + g.ring_bytes + g.exchange_bytes + sizeof(Shared) + 16;
  if (smem < 116 * 1024) smem = 116 * 1024;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config<EPI>(attr, g.parts, tiles, smem, s);
  return cudaLaunchKernelEx(&cfg, kern, w, w2, x, g);
}

}  // namespace

cudaError_t launch_dense_skinny(int epi, const CUtensorMap& w, const CUtensorMap& w2,
                                const CUtensorMap& x, const SkinnyGemm& g, cudaStream_t s) {
  if (g.T < 1 || g.T > kSkinnyTokens || g.kbs < 1) return cudaErrorInvalidValue;
  return epi == kEpiGated ? launch<kEpiGated>(w, w2, x, g, s) : launch<kEpiLinear>(w, w2, x, g, s);
}

}  // namespace vmoe
