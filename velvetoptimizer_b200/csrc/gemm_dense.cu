// Dense bf16 products on CTA pairs (tcgen05.mma.cta_group::2) for the fused linear and the
// gated feed-forward block, reading every operand in the layout the user holds it in.
//
//   forward           C[T, N] = x[T, K] w[N, K]^T       both operands K-major
//   input gradient    C[T, K] = dz[T, N] w[N, K]        B stored [k, n]: read MN-major
//   weight gradient   C[N, K] = dz[T, N]^T x[T, K]      both stored [k, mn]: read MN-major
//
// so no transposed or repacked copy of a weight or an activation is written.  A pair of CTAs
// computes a 256 x 256 tile: each loads its own 128 rows of A and its own half of B per
// 64-wide k block (32 KB a stage, 6 stages), the leader issues M256 N256 K16, each CTA's TMEM
// holds its 128 rows, two accumulators deep, and eight epilogue warps per CTA drain one while
// the other fills.  A K-major stage is one box of 64 k x 128 rows, an MN-major one two boxes
// of 64 columns x 64 k rows (128-byte swizzle; descriptor leading offset 8 KB between the
// 64-column chunks, stride offset 1 KB between 8-row groups).
//
// Extra forms of the k loop and of B:
//   * several operand pairs (segs): dx = dg Wg + du Wu runs as one product whose k blocks come
//     from (dg, Wg) and then from (du, Wu), in one accumulator; an fp32 product as six pairs of
//     its operands' bf16 planes (dense_f32.cu);
//   * kEpiGated: the leader's half of B is 128 gate rows and the follower's 128 up rows of the
//     same features, so a row's gate and up values meet in the epilogue;
//   * groups: two A operands against one B (the gate's and the up's weight gradients);
//   * splits: when the tiles are too few for the SMs the k blocks are divided, every split
//     writes fp32 partials, and launch_dense_finish sums them in split order and runs the
//     epilogue: no atomics, the same bits every run.
// Rows, columns and k past the operands' extents are zero-filled by the TMA and never stored.
// Every wait is bounded and reports a status code; no TMA multicast.
//
// Bound by the tensor cores, the activation's gradient also by its epilogue's bytes.  Block of
// 32,768 x 2048 x 8192, bf16, fraction of a measured 1627.5 TFLOP/s (boxes differ by 5 %): down
// 776 us (87 %), dx 1611 (84 %), gate's and up's weight gradients 1658 (81 %), gate|up keeping fp32
// g and u 1764 (77 %), down's weight gradient, split, 873 + 35 (74 % with its finish), dh with the
// gradient 1352 (50 %).
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "dense.h"
#include "dense_act.cuh"

namespace vmoe {
namespace {

constexpr int BK = 64;
constexpr int PAIR_M = 256;
constexpr int BN = 256;
constexpr uint32_t CHUNK_BYTES = 64 * BK * 2;  // one MN-major box
constexpr uint32_t HALF_BYTES = 128 * BK * 2;  // one operand's part of a stage in one CTA
constexpr uint32_t STAGE_BYTES = 2 * HALF_BYTES;
constexpr int STAGES = 6;
constexpr uint32_t TMEM_COLS = 2 * BN;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int kMaxDevices = 64;

struct Shared {
  uint64_t full[STAGES];
  uint64_t empty[STAGES];
  uint64_t tfull[2];
  uint64_t tempty[2];  // the leader's are used: 16 arrivals (8 epilogue warps x 2 CTAs)
  uint64_t done;
  uint32_t tmem_base;
  int abort;
  alignas(16) __nv_bfloat16 bias[EPI_WARPS][2][32];
};

// Each epilogue warp turns 32 x 32 blocks between a thread per row (the accumulator's layout)
// and coalesced rows through 4 KB of its own: two bf16 blocks or one fp32 block.
constexpr uint32_t BLOCK_BYTES = 32 * 64;
constexpr uint32_t TURN_BYTES = EPI_WARPS * 2 * BLOCK_BYTES;

constexpr size_t SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + TURN_BYTES + sizeof(Shared) + 16;
static_assert(SMEM_BYTES <= 232448, "shared memory budget");

__device__ __forceinline__ bool aborted(const Shared* sh) {
  return *reinterpret_cast<const volatile int*>(&sh->abort) != 0;
}
__device__ __forceinline__ void set_abort(Shared* sh, int* status, int code) {
  *reinterpret_cast<volatile int*>(&sh->abort) = 1;
  report(status, code);
}

__device__ __forceinline__ uint64_t desc_mn(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(CHUNK_BYTES >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// descriptor of the 16-wide k step `k` of a stage part at `addr`
template <bool MN>
__device__ __forceinline__ uint64_t op_desc(uint32_t addr, int k) {
  if constexpr (MN) return desc_mn(addr + k * 2048);  // two 8-row groups further on
  return umma_desc_sw128(addr + k * 32);
}

// Arrive on another CTA's barrier to say that TMEM has been read.  Only the TMEM reads are
// ordered (tcgen05 fences on both sides); a release at cluster scope would also wait for every
// global store of the epilogue so far.
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// 8 accumulator columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

// First accumulator column of the i-th 32-wide block of an epilogue warp's share (two shares;
// gated: two blocks of gate columns, then the up columns of the same features).
template <int EPI>
__device__ __forceinline__ int column_of(int part, int i) {
  return EPI == kEpiGated ? (i >> 1) * 128 + part * 64 + (i & 1) * 32 : part * 128 + i * 32;
}

struct Item {
  int g, m, n, kb, ke;
};

// Work item -> (group, tile, k-block range).  Tiles go in bands of `band` n tiles, all m tiles
// of a band before the next, so the pairs running at one time share few A and B tiles.
__device__ __forceinline__ Item item_of(const DenseGemm& a, int item) {
  Item w;
  const int split = item % a.splits;
  int t = item / a.splits;
  const int per_group = a.m_tiles * a.n_tiles;
  w.g = t / per_group;
  t -= w.g * per_group;
  const int full = a.n_tiles / a.band;
  const int band = t / (a.m_tiles * a.band);
  if (band < full) {
    const int r = t - band * a.m_tiles * a.band;
    w.m = r / a.band;
    w.n = band * a.band + r % a.band;
  } else {
    const int width = a.n_tiles - full * a.band;
    const int r = t - full * a.m_tiles * a.band;
    w.m = r / width;
    w.n = full * a.band + r % width;
  }
  w.kb = split * a.kb_per_split;
  w.ke = min(w.kb + a.kb_per_split, a.segs * a.kbs);
  return w;
}

// 32 bias values of the columns [col, col + 32) into this warp's shared row (0 past N)
__device__ __forceinline__ void stage_bias(__nv_bfloat16* dst, const void* bias, int64_t col,
                                           int64_t N, int lane) {
  const auto* b = static_cast<const __nv_bfloat16*>(bias);
  dst[lane] = (b && col + lane < N) ? b[col + lane] : __float2bfloat16_rn(0.f);
}

__device__ __forceinline__ void add_bias(float (&v)[32], const __nv_bfloat16* b) {
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    float f[8];
    load16_to_f(b + j, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j + i] += f[i];
  }
}

// A 32 x 32 block of a bf16 matrix: where it starts, its pitch, and how much of it is inside.
// With `vec` its rows are whole aligned 16-byte units (cols a multiple of 8).
struct Block {
  __nv_bfloat16* p;
  int64_t ld;
  int rows, cols;  // valid, at most 32; rows may be <= 0
  bool vec;
  __device__ __forceinline__ bool whole() const { return vec && rows == 32 && cols == 32; }
};

// shared address of 16-byte unit c of row r (bf16: 4 units a row, fp32: 8); the XOR keeps both
// a unit of every row and whole rows free of bank conflicts
__device__ __forceinline__ uint4* unit16(uint8_t* buf, int r, int c) {
  return reinterpret_cast<uint4*>(buf + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}
__device__ __forceinline__ uint4* unit32(uint8_t* buf, int r, int c) {
  return reinterpret_cast<uint4*>(buf + r * 128 + ((c ^ (r & 7)) << 4));
}

// Block -> registers: units with four lanes per row, or single elements with a lane per column
// and two rows per register
__device__ __forceinline__ void fetch(const Block& b, uint4 (&v)[4], int lane) {
  if (b.vec) {
    const __nv_bfloat16* p = b.p + (lane >> 2) * b.ld + (lane & 3) * 8;
    if (b.whole()) {
#pragma unroll
      for (int i = 0; i < 4; ++i, p += 8 * b.ld) v[i] = __ldg(reinterpret_cast<const uint4*>(p));
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i, p += 8 * b.ld) {
      v[i] = make_uint4(0, 0, 0, 0);
      if (i * 8 + (lane >> 2) < b.rows && (lane & 3) * 8 < b.cols)
        v[i] = __ldg(reinterpret_cast<const uint4*>(p));
    }
    return;
  }
  const auto* p = reinterpret_cast<const unsigned short*>(b.p) + lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j, p += 2 * b.ld) {
      const int r = 8 * i + 2 * j;
      const uint32_t lo = lane < b.cols && r < b.rows ? __ldg(p) : 0u;
      const uint32_t hi = lane < b.cols && r + 1 < b.rows ? __ldg(p + b.ld) : 0u;
      w[j] = lo | hi << 16;
    }
    v[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// registers -> shared
__device__ __forceinline__ void land(const Block& b, const uint4 (&v)[4], uint8_t* buf, int lane) {
  if (b.vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *unit16(buf, i * 8 + (lane >> 2), lane & 3) = v[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      reinterpret_cast<unsigned short*>(unit16(buf, 8 * i + j, lane >> 3))[lane & 7] =
          static_cast<unsigned short>(w[j >> 1] >> (16 * (j & 1)));
  }
}

// 32 rows x 16 columns of an fp32 matrix whose rows are whole aligned 16-byte units
struct Kept {
  const float* p;
  int64_t ld;
  int rows, cols;  // cols a multiple of 4
};

__device__ __forceinline__ void fetch16(const Kept& b, uint4 (&v)[4], int lane) {
  const float* p = b.p + (lane >> 2) * b.ld + (lane & 3) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i, p += 8 * b.ld) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (i * 8 + (lane >> 2) < b.rows && (lane & 3) * 4 < b.cols)
      v[i] = __ldg(reinterpret_cast<const uint4*>(p));
  }
}

__device__ __forceinline__ void land16(const uint4 (&v)[4], uint8_t* buf, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) *unit16(buf, i * 8 + (lane >> 2), lane & 3) = v[i];
}

__device__ __forceinline__ void get_row(uint8_t* buf, float (&v)[32], int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    load16_to_f(reinterpret_cast<const __nv_bfloat16*>(unit16(buf, lane, c)), v + 8 * c);
}

__device__ __forceinline__ void put_row(uint8_t* buf, const float (&v)[32], int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    store16_from_f(reinterpret_cast<__nv_bfloat16*>(unit16(buf, lane, c)), v + 8 * c);
}

// shared -> Block, coalesced
__device__ __forceinline__ void flush(const Block& b, uint8_t* buf, int lane) {
  if (b.vec) {
    __nv_bfloat16* p = b.p + (lane >> 2) * b.ld + (lane & 3) * 8;
    if (b.whole()) {
#pragma unroll
      for (int i = 0; i < 4; ++i, p += 8 * b.ld)
        *reinterpret_cast<uint4*>(p) = *unit16(buf, i * 8 + (lane >> 2), lane & 3);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i, p += 8 * b.ld)
      if (i * 8 + (lane >> 2) < b.rows && (lane & 3) * 8 < b.cols)
        *reinterpret_cast<uint4*>(p) = *unit16(buf, i * 8 + (lane >> 2), lane & 3);
    return;
  }
  __nv_bfloat16* p = b.p + lane;
#pragma unroll 8
  for (int r = 0; r < 32; ++r, p += b.ld)
    if (lane < b.cols && r < b.rows)
      *p = reinterpret_cast<__nv_bfloat16*>(unit16(buf, r, lane >> 3))[lane & 7];
}

// a thread's row of fp32 values -> an fp32 matrix, coalesced (the whole 4 KB buffer)
__device__ __forceinline__ void flush_f32(float* p, int64_t ld, int rows, int cols, bool vec,
                                          const float (&v)[32], uint8_t* buf, int lane) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4*>(unit32(buf, lane, c)) =
        make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  __syncwarp();
  if (vec && cols % 4 == 0) {
    float* q = p + (lane >> 3) * ld + (lane & 7) * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i, q += 4 * ld) {
      const int r = i * 4 + (lane >> 3), c = lane & 7;
      if (r < rows && c * 4 < cols) *reinterpret_cast<uint4*>(q) = *unit32(buf, r, c);
    }
  } else {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (lane < cols && r < rows)
        p[r * ld + lane] = reinterpret_cast<const float*>(unit32(buf, r, lane >> 2))[lane & 3];
  }
}

// Column sums of the 32 x 32 block in `buf` (rows outside hold zeros) to dst[0..cols): a lane
// adds 4 rows of its 8 columns, then the 8 lanes of the same columns halve their columns with
// a partner's three times.
__device__ __forceinline__ void column_sums(uint8_t* buf, int cols, float* dst, int lane) {
  float s[8] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[8];
    load16_to_f(reinterpret_cast<const __nv_bfloat16*>(unit16(buf, i * 8 + (lane >> 2), lane & 3)), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += f[j];
  }
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1) {
    const bool upper = (lane & (4 * o)) != 0;
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const float other = __shfl_xor_sync(0xffffffffu, upper ? s[j] : s[j + o], 4 * o);
      s[j] = (upper ? s[j + o] : s[j]) + other;
    }
  }
  const int col = (lane & 3) * 8 + ((lane >> 4) & 1) * 4 + ((lane >> 3) & 1) * 2 + ((lane >> 2) & 1);
  if (col < cols) dst[col] = s[0];
}

template <bool A_MN, bool B_MN, int EPI, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
gemm_dense_kernel(const __grid_constant__ DenseMaps maps, const __grid_constant__ DenseGemm args) {
  constexpr uint32_t IDESC = umma_idesc_bf16(PAIR_M, BN) | (A_MN ? 1u << 15 : 0u) |
                             (B_MN ? 1u << 16 : 0u);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t a_s = base;
  const uint32_t b_s = base + STAGES * HALF_BYTES;
  Shared* sh = reinterpret_cast<Shared*>(gbase + STAGES * STAGE_BYTES + TURN_BYTES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&sh->full[s]), 1);
      mbar_init(smem_u32(&sh->empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&sh->tfull[a]), 1);
      mbar_init(smem_u32(&sh->tempty[a]), 2 * EPI_WARPS);
    }
    mbar_init(smem_u32(&sh->done), 1);
    sh->abort = 0;
    fence_mbar_init();
    prefetch_tmap(&maps.a[0]);
    prefetch_tmap(&maps.b[0]);
  }
  cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA arrive or copy
  if (warp == 1) tmem_alloc_pair(smem_u32(&sh->tmem_base), TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // nothing above touches global memory
  const int total = args.groups * args.m_tiles * args.n_tiles * args.splits;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    if (lane == 0) {
      int it = 0;
      for (int item = pair; item < total; item += num_pairs) {
        const Item w = item_of(args, item);
        const int a_at = w.m * PAIR_M + static_cast<int>(rank) * 128;
        // gated: this CTA's 128 rows are gate (leader) or up (follower) rows of one weight each
        const int b_at = EPI == kEpiGated ? w.n * 128 : w.n * BN + static_cast<int>(rank) * 128;
        // one row of tiles: every pair reads other weights, and pairs that went through k in
        // step would ask for the same columns of far rows at the same time
        int at = w.kb;
        if (args.m_tiles == 1) at += (w.n * 5) % (w.ke - w.kb);
        int seg = at / args.kbs, kk = at - seg * args.kbs;
        bool ok = true;
        for (int kb = w.kb; kb < w.ke; ++kb, ++it) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(smem_u32(&sh->empty[s]), ph ^ 1)) {
            set_abort(sh, args.status, kStatusTimeoutProducer);
            ok = false;
            break;
          }
          if (aborted(sh)) { ok = false; break; }
          const int k0 = kk * BK;
          const CUtensorMap* am = &maps.a[args.seg_a[seg] + w.g * args.group_a];
          const CUtensorMap* bm = &maps.b[args.seg_b[seg] + (leader ? 0 : args.follower_b)];
          if (++at == w.ke) {
            at = w.kb;
            seg = at / args.kbs;
            kk = at - seg * args.kbs;
          } else if (++kk == args.kbs) {
            kk = 0;
            ++seg;
          }
          const uint32_t fb = smem_u32(&sh->full[s]);
          if (leader) mbar_arrive_expect_tx(fb, 2 * STAGE_BYTES);
          const uint32_t fb_leader = mapa_shared(fb, 0);
          const uint32_t a_dst = a_s + s * HALF_BYTES, b_dst = b_s + s * HALF_BYTES;
          if constexpr (A_MN) {
            tma_load_2d_pair(a_dst, am, fb_leader, a_at, k0);
            tma_load_2d_pair(a_dst + CHUNK_BYTES, am, fb_leader, a_at + 64, k0);
          } else {
            tma_load_2d_pair(a_dst, am, fb_leader, k0, a_at);
          }
          if constexpr (B_MN) {
            tma_load_2d_pair(b_dst, bm, fb_leader, b_at, k0);
            tma_load_2d_pair(b_dst + CHUNK_BYTES, bm, fb_leader, b_at + 64, k0);
          } else {
            tma_load_2d_pair(b_dst, bm, fb_leader, k0, b_at);
          }
        }
        if (!ok) break;
      }
      // the kernel after this one may come up while the last tiles are multiplied and stored
      asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader only) ----------------
    if (leader && lane == 0) {
      int it = 0, local = 0;
      for (int item = pair; item < total; item += num_pairs) {
        const Item w = item_of(args, item);
        bool ok = true;
        // a split product may read its accumulator out in between (see the epilogue)
        const int run = SPLIT ? args.run_kb : w.ke - w.kb;
        for (int k0 = w.kb; ok && k0 < w.ke; k0 += run, ++local) {
          const int acc = local & 1;
          const uint32_t aph = (local >> 1) & 1;
          if (!mbar_wait_cluster(smem_u32(&sh->tempty[acc]), aph ^ 1)) {
            set_abort(sh, args.status, kStatusTimeoutMma);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem + acc * BN;
          const int k1 = min(w.ke, k0 + run);
          for (int kb = k0; kb < k1; ++kb, ++it) {
            const int s = it % STAGES;
            const uint32_t ph = (it / STAGES) & 1;
            if (!mbar_wait(smem_u32(&sh->full[s]), ph)) {
              set_abort(sh, args.status, kStatusTimeoutMma);
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a_addr = a_s + s * HALF_BYTES, b_addr = b_s + s * HALF_BYTES;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              umma_bf16_pair(d_tmem, op_desc<A_MN>(a_addr, k), op_desc<B_MN>(b_addr, k), IDESC,
                             (kb > k0 || k > 0) ? 1u : 0u);
            umma_commit_pair(smem_u32(&sh->empty[s]), 0x3);  // frees the stage in both CTAs
          }
          if (ok) umma_commit_pair(smem_u32(&sh->tfull[acc]), 0x3);
        }
        if (!ok || aborted(sh)) break;
      }
      umma_commit_pair(smem_u32(&sh->done), 0x1);
      if (!mbar_wait(smem_u32(&sh->done), 0)) report(args.status, kStatusTimeoutDrain);
    }
  } else {
    // ---------------- epilogue (warps 2..9, both CTAs) ----------------
    const int q = warp & 3;            // TMEM lane quarter this warp may access
    const int part = (warp - 2) >> 2;  // which half of the columns
    __nv_bfloat16(*bias_s)[32] = sh->bias[warp - 2];
    uint8_t* turn_a = gbase + STAGES * STAGE_BYTES + (warp - 2) * 2 * BLOCK_BYTES;
    uint8_t* turn_b = turn_a + BLOCK_BYTES;
    const DenseEpi& ep = args.epi;
    constexpr int COLS = EPI == kEpiGated ? 64 : 128;  // columns (features) of a warp's share
    if constexpr (SPLIT) {
      // fp32 partials in the accumulator's own column order (gated: gate | up per tile).  The
      // tensor cores truncate when they add to the accumulator, an error that grows with the
      // number of additions: an fp32 product is read out every run_kb k blocks and summed here,
      // rounded to nearest (relative error of a sum over 8192: 9.1e-6 without, 4.8e-7 with; no measurable time).
      int local = 0;
      for (int item = pair; item < total; item += num_pairs) {
        const Item w = item_of(args, item);
        float v[4][32] = {};
        bool ok = true;
        for (int k0 = w.kb; k0 < w.ke; k0 += args.run_kb, ++local) {
          const int acc = local & 1;
          const bool got = mbar_wait(smem_u32(&sh->tfull[acc]), (local >> 1) & 1);
          __syncwarp();
          ok = __all_sync(0xffffffffu, got);
          if (!ok) {
            if (lane == 0) set_abort(sh, args.status, kStatusTimeoutEpilogue);
            break;
          }
          tc_fence_after();
          const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * BN;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int h = 0; h < 32; h += 8) {
              float t[8];
              tmem_ld8(t_row + column_of<EPI>(part, i) + h, t);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[i][h + j] += t[j];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_remote(mapa_shared(smem_u32(&sh->tempty[acc]), 0));
        }
        if (!ok) break;
        const int64_t row0 = static_cast<int64_t>(w.m) * PAIR_M + rank * 128 + q * 32;
        const int rows = static_cast<int>(args.M - row0 < 32 ? args.M - row0 : 32);
        float* dst = args.partial +
                     ((static_cast<int64_t>(item % args.splits) * args.groups + w.g) * args.M + row0) *
                         args.ldp +
                     static_cast<int64_t>(w.n) * BN;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          __syncwarp();
          flush_f32(dst + column_of<EPI>(part, i), args.ldp, rows, 32, true, v[i], turn_a, lane);
        }
      }
    } else {
    int local = 0;
    for (int item = pair; item < total; item += num_pairs, ++local) {
      const Item w = item_of(args, item);
      const int acc = local & 1;
      const uint32_t aph = (local >> 1) & 1;
      const int64_t row0 = static_cast<int64_t>(w.m) * PAIR_M + rank * 128 + q * 32;
      const int rows = static_cast<int>(args.M - row0 < 32 ? args.M - row0 : 32);
      const int64_t col0 =
          static_cast<int64_t>(w.n) * (EPI == kEpiGated ? 128 : BN) + part * COLS;
      // block of the matrix p at column offset c of this warp's share
      auto block = [&](const void* p, int64_t ld, int c, int flag) {
        const int64_t left = args.N - col0 - c;
        const bool vec = (ep.vec & flag) != 0;
        const int cols = static_cast<int>(left < 32 ? (left > 0 ? left : 0) : 32);
        return Block{static_cast<__nv_bfloat16*>(const_cast<void*>(p)) + row0 * ld + col0 + c, ld,
                     rows, vec ? (cols + 7) & ~7 : cols, vec};
      };
      // 16 columns at offset c of g or u, which the forward kept in fp32 rows of whole units
      auto kept = [&](const void* p, int c) {
        const int64_t left = args.N - col0 - c;
        return Kept{static_cast<const float*>(p) + row0 * ep.ldz + col0 + c, ep.ldz, rows,
                    static_cast<int>(left < 16 ? (left > 0 ? (left + 3) & ~3 : 0) : 16)};
      };
      // what the epilogue reads besides the accumulator is asked for before the product is done
      uint4 pre0[4], pre1[4];
      const bool has_res = EPI == kEpiLinear && ep.res;
      if constexpr (EPI == kEpiGluBwd) {
        fetch16(kept(ep.z, 0), pre0, lane);
        fetch16(kept(ep.z2, 0), pre1, lane);
      } else if (has_res) {
        fetch(block(ep.res, ep.ldr, 0, kVecRes), pre0, lane);
      }
      const bool got = mbar_wait(smem_u32(&sh->tfull[acc]), aph);
      __syncwarp();
      if (!__all_sync(0xffffffffu, got)) {
        if (lane == 0) set_abort(sh, args.status, kStatusTimeoutEpilogue);
        break;
      }
      tc_fence_after();
      const uint32_t t_row =
          tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * BN + part * COLS;
      // the accumulator is free for the next item once this warp's last columns are read
      auto release = [&](int c) {
        if (c != COLS - 32) return;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_remote(mapa_shared(smem_u32(&sh->tempty[acc]), 0));
      };
#pragma unroll 1
      for (int c = 0; c < COLS; c += 32) {
        __syncwarp();
        if constexpr (EPI == kEpiGated) {
          float g[32], u[32];
          tmem_ld32(t_row + c, g);
          tmem_ld32(t_row + 128 + c, u);
          release(c);
          const Block h = block(ep.out, ep.ldo, c, kVecOut);
          if (h.cols == 0) continue;  // the same for the whole warp
          if (ep.bias || ep.bias2) {
            stage_bias(bias_s[0], ep.bias, col0 + c, args.N, lane);
            stage_bias(bias_s[1], ep.bias2, col0 + c, args.N, lane);
            __syncwarp();
            add_bias(g, bias_s[0]);
            add_bias(u, bias_s[1]);
          }
          if (ep.z) {
            const int64_t at = row0 * ep.ldz + col0 + c;
            flush_f32(static_cast<float*>(ep.z) + at, ep.ldz, rows, h.cols, true, g, turn_a, lane);
            __syncwarp();
            flush_f32(static_cast<float*>(ep.z2) + at, ep.ldz, rows, h.cols, true, u, turn_a, lane);
            __syncwarp();
          }
          act_switch(ep.act, [&](auto A) {
            act_values<true, decltype(A)::value>(g, ep.gamma);
#pragma unroll
            for (int j = 0; j < 32; ++j) g[j] *= u[j];
          });
          put_row(turn_a, g, lane);
          __syncwarp();
          flush(h, turn_a, lane);
        } else if constexpr (EPI == kEpiGluBwd) {
          const Block bg = block(ep.out, ep.ldo, c, kVecOut), bu = block(ep.out2, ep.ldo, c, kVecOut);
          if (bg.cols == 0) {
            release(c);
            continue;
          }
          // 16 columns of g and u at a time through the two halves of the buffer, 32 of dg and
          // du out
          uint4 dg[4], du[4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            land16(pre0, turn_a, lane);
            land16(pre1, turn_b, lane);
            __syncwarp();
            if (c + 16 * half + 16 < COLS) {
              fetch16(kept(ep.z, c + 16 * half + 16), pre0, lane);
              fetch16(kept(ep.z2, c + 16 * half + 16), pre1, lane);
            }
            float dh[16];
            tmem_ld16(t_row + c + 16 * half, dh);
            if (half == 1) release(c);
            act_switch(ep.act, [&](auto A) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {  // a unit of 4 columns
                const float4 gv = *reinterpret_cast<const float4*>(unit16(turn_a, lane, k));
                const float4 uv = *reinterpret_cast<const float4*>(unit16(turn_b, lane, k));
                const float2 p0 = make_float2(dh[4 * k], dh[4 * k + 1]),
                             p1 = make_float2(dh[4 * k + 2], dh[4 * k + 3]);
                float2 a0, d0, a1, d1;
                act_grad2<decltype(A)::value>(make_float2(gv.x, gv.y), ep.gamma, a0, d0);
                act_grad2<decltype(A)::value>(make_float2(gv.z, gv.w), ep.gamma, a1, d1);
                const float2 g0 = times_slope2<decltype(A)::value>(mul2(p0, make_float2(uv.x, uv.y)), d0);
                const float2 g1 = times_slope2<decltype(A)::value>(mul2(p1, make_float2(uv.z, uv.w)), d1);
                const float2 u0 = mul2(p0, a0), u1 = mul2(p1, a1);
                uint32_t* tg = reinterpret_cast<uint32_t*>(dg) + 8 * half + 2 * k;
                uint32_t* tu = reinterpret_cast<uint32_t*>(du) + 8 * half + 2 * k;
                tg[0] = pack_bf16x2(g0.x, g0.y);
                tg[1] = pack_bf16x2(g1.x, g1.y);
                tu[0] = pack_bf16x2(u0.x, u0.y);
                tu[1] = pack_bf16x2(u1.x, u1.y);
              }
            });
            __syncwarp();
          }
          // a row outside has zeros for dy but not for its product: 0 x infinity in the weights
          const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            *unit16(turn_a, lane, k) = lane < rows ? dg[k] : zero;
            *unit16(turn_b, lane, k) = lane < rows ? du[k] : zero;
          }
          __syncwarp();
          flush(bg, turn_a, lane);
          flush(bu, turn_b, lane);
          if (ep.colsum) {
            float* dst = ep.colsum + row0 / 32 * args.N + col0 + c;
            const int cols = static_cast<int>(min(args.N - col0 - c, static_cast<int64_t>(32)));
            if (rows > 0) {
              column_sums(turn_a, cols, dst, lane);
              column_sums(turn_b, cols, dst + ep.colsum_stride, lane);
            }
          }
        } else {
          float v[32];
          tmem_ld32(t_row + c, v);
          release(c);
          const Block out = block(w.g ? ep.out2 : ep.out, ep.ldo, c, kVecOut);
          if (out.cols == 0) continue;
          if (has_res) land(block(ep.res, ep.ldr, c, kVecRes), pre0, turn_a, lane);
          if (ep.bias) stage_bias(bias_s[0], ep.bias, col0 + c, args.N, lane);
          __syncwarp();
          if (has_res && c + 32 < COLS) fetch(block(ep.res, ep.ldr, c + 32, kVecRes), pre0, lane);
          if (ep.bias) add_bias(v, bias_s[0]);
          if (ep.z) {
            put_row(turn_b, v, lane);
            __syncwarp();
            flush(block(ep.z, ep.ldz, c, kVecZ), turn_b, lane);
          }
          if (ep.act != kActNone) {
            act_switch(ep.act,
                       [&](auto A) { act_values<true, decltype(A)::value>(v, ep.gamma); });
          }
          if (has_res) {
            float r[32];
            get_row(turn_a, r, lane);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += r[j];
          }
          if (ep.out_f32) {
            __syncwarp();
            // the columns that exist: an fp32 row is whole 16-byte units from a multiple of 4
            // columns on, so `out`, rounded up to 8 for bf16's, may reach into the next row
            const int cols = static_cast<int>(min(args.N - col0 - c, static_cast<int64_t>(32)));
            flush_f32(static_cast<float*>(w.g ? ep.out2 : ep.out) + row0 * ep.ldo + col0 + c, ep.ldo,
                      rows, cols, out.vec, v, turn_a, lane);
          } else {
            put_row(turn_a, v, lane);
            __syncwarp();
            flush(out, turn_a, lane);
          }
        }
      }
    }
    }
  }

  __syncthreads();
  if (threadIdx.x == 0 && aborted(sh)) {
    // copies issued by this CTA land on the leader's barriers; give any still in flight a
    // bounded time to finish before the shared memory is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
  }
  cluster_sync_all();  // the leader's MMAs (which read both CTAs' smem) are complete
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
}

template <bool A_MN, bool B_MN, int EPI, bool SPLIT>
cudaError_t launch(const DenseMaps& maps, const DenseGemm& g, int num_sms, cudaStream_t s) {
  auto kern = gemm_dense_kernel<A_MN, B_MN, EPI, SPLIT>;
  cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(SMEM_BYTES));
  if (err != cudaSuccess) return err;
  const int64_t work = static_cast<int64_t>(g.groups) * g.m_tiles * g.n_tiles * g.splits;
  if (work < 1 || work > 0x7fffffff || g.band < 1 || g.kb_per_split < 1 || g.kbs < 1 ||
      g.segs < 1 || g.segs > 12)
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // persistent, as many pairs as can be resident at once (a pair needs two free SMs of one
  // GPC), so that no pair's share of the items starts after another's has ended
  static std::atomic<int> resident[kMaxDevices];
  int dev = 0;
  if ((err = cudaGetDevice(&dev)) != cudaSuccess) return err;
  int max_pairs = dev < kMaxDevices ? resident[dev].load(std::memory_order_relaxed) : 0;
  if (max_pairs == 0) {
    cfg.gridDim = dim3(static_cast<unsigned>(num_sms & ~1), 1, 1);
    err = cudaOccupancyMaxActiveClusters(&max_pairs, reinterpret_cast<const void*>(kern), &cfg);
    if (err != cudaSuccess) return err;
    if (max_pairs < 1) return cudaErrorInvalidConfiguration;
    if (dev < kMaxDevices) resident[dev].store(max_pairs, std::memory_order_relaxed);
  }
  int64_t pairs = num_sms / 2;
  if (pairs > max_pairs) pairs = max_pairs;
  if (pairs > work) pairs = work;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs), 1, 1);
  cfg.numAttrs = g_launch_pdl ? 2 : 1;
  err = cudaLaunchKernelEx(&cfg, kern, maps, g);
  return err != cudaSuccess ? err : cudaGetLastError();
}

}  // namespace

cudaError_t launch_gemm_dense(bool a_mn, bool b_mn, int epi, const DenseMaps& maps,
                              const DenseGemm& g, int num_sms, cudaStream_t s) {
  if (g.splits > 1 && !g.partial) return cudaErrorInvalidValue;
  if (g.partial) {
    if (g.ldp % 4) return cudaErrorInvalidValue;
    if (!a_mn && !b_mn)
      return epi == kEpiGated ? launch<false, false, kEpiGated, true>(maps, g, num_sms, s)
                              : launch<false, false, kEpiLinear, true>(maps, g, num_sms, s);
    if (!a_mn) return launch<false, true, kEpiLinear, true>(maps, g, num_sms, s);
    return launch<true, true, kEpiLinear, true>(maps, g, num_sms, s);
  }
  if (!a_mn && !b_mn)
    return epi == kEpiGated ? launch<false, false, kEpiGated, false>(maps, g, num_sms, s)
                            : launch<false, false, kEpiLinear, false>(maps, g, num_sms, s);
  if (!a_mn && b_mn)
    return epi == kEpiGluBwd ? launch<false, true, kEpiGluBwd, false>(maps, g, num_sms, s)
                             : launch<false, true, kEpiLinear, false>(maps, g, num_sms, s);
  if (a_mn && b_mn && epi == kEpiLinear)
    return launch<true, true, kEpiLinear, false>(maps, g, num_sms, s);
  return cudaErrorInvalidValue;
}

}  // namespace vmoe
