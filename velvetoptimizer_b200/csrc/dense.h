// Kernel launchers of the dense training operators (fused linear, gated feed-forward,
// gradient norm): the interface between their kernels and the C-ABI host side in dense.cu
// and grad_norm.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace vmoe {

// activations, the values of VMOE_ACT_*
enum Act : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGeluTanh = 3, kActEra = 4 };

// What happens to an accumulated product on its way to memory.
//   kEpiLinear  z = acc + bias; [z kept]; out = res + act(z)
//   kEpiGated   g = acc_g + bias, u = acc_u + bias2; [g, u kept]; out = act(g) * u
//   kEpiGluBwd  acc = dh, g and u read: out = dh * u * act'(g), out2 = dh * act(g)
enum EpiKind : int { kEpiLinear = 0, kEpiGated = 1, kEpiGluBwd = 2 };

// `vec` bits: every row of the buffer is whole aligned 16-byte units: base and pitch are
// multiples of 16 bytes, and so are the columns, or what follows them up to the pitch is the
// buffer's own padding (it may be read and overwritten)
enum : int { kVecOut = 1, kVecRes = 2, kVecZ = 4 };

struct DenseEpi {
  int act = kActNone;
  float gamma = 0.f;
  const void* bias = nullptr;   // [N], the operands' type
  const void* bias2 = nullptr;  // kEpiGated: the up projection's
  const void* res = nullptr;
  int64_t ldr = 0;
  void* out = nullptr;
  void* out2 = nullptr;  // kEpiGluBwd: du; second group of a grouped launch: its output
  int64_t ldo = 0;
  // kept pre-activations.  The linear's z has the operands' type: its rounding reaches the
  // gradient only through act'.  The gated block's g and u are fp32: both scale the gradient
  // directly, and rounded to bf16 they would add as much error again as rounding dg and du for
  // the products does (relative error of dx 0.0030 against 0.0024; 3 % more time).
  void* z = nullptr;   // linear: z; gated, and its gradient: g
  void* z2 = nullptr;  // u
  int64_t ldz = 0;
  int out_f32 = 0;  // out is fp32 (gradients of fp32 parameters)
  int vec = 0;
  // kEpiGluBwd, optional: column sums of every 32 rows of dg, [ceil(M / 32)][N], and of du
  // colsum_stride floats further
  float* colsum = nullptr;
  int64_t colsum_stride = 0;
};

// One product C[M, N] = sum over k of A(m, k) B(n, k) on CTA pairs (gemm_dense.cu).
struct DenseGemm {
  int64_t M = 0, N = 0;  // valid rows and columns (kEpiGated: N = features)
  int m_tiles = 0, n_tiles = 0;
  // the k loop: `segs` operand pairs of `kbs` 64-wide k blocks each, in one accumulator
  int segs = 1, kbs = 0;
  unsigned char seg_a[12] = {}, seg_b[12] = {};  // a pair's maps
  int groups = 1;   // independent products sharing B: A maps group_a further, out / out2
  int group_a = 0;
  int follower_b = 0;  // kEpiGated: the follower's B maps (the up weight)
  int splits = 1, kb_per_split = 0;
  int run_kb = 1 << 30;  // partials: k blocks the tensor cores accumulate before a read-out
  int band = 0;          // n tiles per band of the tile order
  float* partial = nullptr;  // given: [splits][groups][M][ldp], and no epilogue
  int64_t ldp = 0;
  // fp32 (dense_f32.cu): set where a sum is not finite, and a counter for each of its tiles
  int* redo = nullptr;
  int* arrived = nullptr;
  int64_t redo_tiles = 0;
  DenseEpi epi;
  int* status = nullptr;
};

struct DenseMaps {
  CUtensorMap a[6], b[6];
};

// a_mn / b_mn: the operand is stored [k rows, M (or N) columns] and read MN-major;
// otherwise [M (or N) rows, k columns].  Built combinations: K-K (forward), K-MN (input
// gradients), MN-MN (weight gradients).
cudaError_t launch_gemm_dense(bool a_mn, bool b_mn, int epi, const DenseMaps& maps,
                              const DenseGemm& g, int num_sms, cudaStream_t s);

// Sum of a split product's partials in split order, then its epilogue (dense_finish.cu).
cudaError_t launch_dense_finish(int dtype, int epi, const DenseGemm& g, cudaStream_t s);

// fp32 as three bf16 planes (dense_f32.cu): x = hi + mid + lo to 2^-26.  Matrices of one
// launch; plane k of a matrix is at out + k * plane elements, rows ldo apart.
struct Split3 {
  const float* x;
  int64_t ldx, rows, cols;
  void* out;
  int64_t ldo, plane;
};
constexpr int kSplitBlocks = 592;  // blocks per matrix
constexpr int kRedoWords = 8;      // a call's products at most; `clear`: theirs to be zeroed, or null
cudaError_t launch_split3(const Split3* m, int n, int* clear, cudaStream_t s);

// The fp32 product `g` once more on the CUDA cores (dense_f32.cu), where its finish has found sums
// that are not finite: element (m, k) of A at a[m * am + k * ak], (n, k) of B at b[n * bn + k * bk].
struct RedoGemm {
  DenseGemm g;
  const float *a[2], *b[2];  // two pairs, one A for each group, or (gated) gate and up
  int pairs;
  int64_t am, ak, bn, bk, K;
};
int64_t redo_tiles(int epi, int64_t M, int64_t N, int groups);
cudaError_t launch_dense_redo(int epi, const RedoGemm& r, int num_sms, cudaStream_t s);

// Few rows (at most kSmallTokens): weights streamed once through registers (dense_small.cu).
constexpr int kSmallTokens = 16;
struct SmallGemm {
  const void* x;
  const void* w;   // [N, K]; kEpiGated: gate weight
  const void* w2;  // kEpiGated: up weight
  int64_t ldx, ldw, ldw2;
  int64_t T, N, K;
  DenseEpi epi;
  int vec_in;  // x and the weights allow 16-byte loads
  int num_sms;
  int* status;
  int early_weights;  // the weights may be read before the kernel ahead has ended
};
cudaError_t launch_dense_stream(int epi, const SmallGemm& g, cudaStream_t s);  // dense_stream.cu
cudaError_t launch_dense_small(int dtype, int epi, const SmallGemm& g, cudaStream_t s);

// A decode batch (at most kSkinnyTokens rows): weights as the MMA's M operand, k divided over a
// cluster (dense_skinny.cu).  Maps: weights in boxes of 64 k x 128 rows (gated: 64 rows of gate
// and of up), x in boxes of 64 k x t_pad rows.
constexpr int kSkinnyTokens = 128;
struct SkinnyGemm {
  int64_t T, N;
  int kbs;  // 64-wide k blocks
  DenseEpi epi;
  int* status;
  int early_weights;  // as SmallGemm's
  // set by the launcher
  int t_pad, parts, kb_per_part, stages;
  uint32_t tmem_cols, ring_bytes, exchange_bytes;
};
cudaError_t launch_dense_skinny(int epi, const CUtensorMap& w, const CUtensorMap& w2,
                                const CUtensorMap& x, const SkinnyGemm& g, cudaStream_t s);

// Elementwise and column work (dense_finish.cu).
// dz = dy * act'(z) into dz [T, ld_dz] (null: not written), and the column sums of dz.
struct DzArgs {
  const void* dy;
  int64_t lddy;
  const void* z;
  int64_t ldz;
  void* dz;
  int64_t lddz;
  int64_t T, N;
  int act;
  float gamma;
  float* colsum;  // [row_blocks][N] partials, or null
  void* db;       // one row block: the sums' own place instead
  bool db_f32;
  int row_blocks;
  int64_t rows_per_block;
};
cudaError_t launch_dense_dz(int dtype, const DzArgs& a, cudaStream_t s);
cudaError_t launch_colsum_finish(const float* partial, int64_t row_blocks, int64_t N, void* out,
                                 void* out2, bool out_f32, cudaStream_t s);
// (out2: the sums of a second set of partials after the first)
// rows of bf16 to a buffer whose pitch is a multiple of 8
cudaError_t launch_pad_copy(const void* src, int64_t lds, int64_t rows, int64_t cols, void* dst,
                            int64_t ldd, cudaStream_t s);

}  // namespace vmoe
