// C-ABI of the dense training operators: the vmoe_ops context, the fused linear and the gated
// feed-forward block (include/vesper_moe.h), forward and backward.
//
// Every call first lays its workspace out (Arena), then launches; the size functions run the
// same layout without a base.  Nothing is allocated and the host never waits.
#include <initializer_list>

#include "dense.h"
#include "ops_host.h"

namespace {

// The status word of a device, zero from the module's load on.  One for all its contexts: a
// gradient's kernels are launched from autograd's thread, through a context that the thread
// which asks for the status never sees.
__device__ int g_ops_status;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool pitch16(const void* p, int64_t ld, size_t elt) {
  return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * static_cast<int64_t>(elt))) &
          15u) == 0;
}

// rows of n elements in whole 16-byte units (DenseEpi::vec)
bool vec_ok(const void* p, int64_t ld, int64_t n, size_t elt) {
  return pitch16(p, ld, elt) && n * static_cast<int64_t>(elt) % 16 == 0;
}

// A bf16 matrix [rows, cols] as the TMA reads it.
struct Mat {
  const void* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
};

// One call: the context, its stream, its workspace, and whether anything is launched (the
// size functions only count).
struct Call {
  vmoe_ops* o;
  Arena ws;
  cudaStream_t s;
  bool dry;
  int dtype;

  bool overlap = true;
  bool first = true;

  // Runs a launch.  Every kernel here waits for the one before it (griddepcontrol.wait) before
  // it touches memory, so all but a call's first, which follows the caller's work, may be
  // launched while their predecessor still runs (`overlap`).  That shortens the backward's
  // chains (777 x 520 x 1304 block, both ways: 99 -> 92 us) and the short kernels' (one-token
  // block 27.3 -> 26.6 us), but not a product followed by its finish (64-row block 39.2 ->
  // 42.0 us), so bf16 forwards beyond the small batches leave it off.
  template <typename F>
  int run(F&& launch, const char* what) {
    PdlScope pdl(!first && overlap);
    first = false;
    const cudaError_t e = launch();
    return e == cudaSuccess ? VMOE_OK : ops_cuda_fail(o, e, what);
  }

  // `m` with a pitch the TMA can read: itself, or a copy with its rows padded to 8 elements
  int tma_ready(Mat& m, const char* what) {
    if (m.ld % 8 == 0) return VMOE_OK;
    const int64_t ld = round_up(m.cols, 8);
    void* dst = ws.take(static_cast<size_t>(m.rows) * ld * 2);
    const Mat src = m;
    m.p = dst;
    m.ld = ld;
    if (dry || m.rows == 0) return VMOE_OK;
    return run([&] { return launch_pad_copy(src.p, src.ld, src.rows, src.cols, dst, ld, s); }, what);
  }
};

#define TRY(x)                     \
  do {                             \
    const int rc_ = (x);           \
    if (rc_ != VMOE_OK) return rc_; \
  } while (0)

// How many parts the k blocks of a product are divided into.  In units of one k block of a
// pair's tile (0.27 us at the full rate): a wave of items costs its k blocks and about four
// for filling the pipe and draining the last accumulator; splitting adds a launch (about ten)
// and the partials' way through L2 (written and read once).
int choose_splits(int64_t tiles, int kb, int pairs, int64_t partial_bytes) {
  int best = 1;
  double best_cost = 1e30;
  for (int s = 1; s <= 16 && s <= kb; ++s) {
    const int per = (kb + s - 1) / s;
    if ((kb + per - 1) / per != s) continue;  // would leave an empty part
    const double waves = static_cast<double>((tiles * s + pairs - 1) / pairs);
    double cost = waves * (per + 4);
    if (s > 1) cost += 10 + 2.0 * static_cast<double>(partial_bytes) * s / 8e6 / 0.27;
    if (cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

// A product on the CTA pairs.  Its operand pairs (a[i], b[j]) are summed in one accumulator;
// with two groups the second reads a[.. + group_a], and a gated one's follower b[.. + follower_b].
struct Product {
  bool a_mn = false, b_mn = false;
  int epi = kEpiLinear;
  Mat a[6], b[6];
  int segs = 1;
  unsigned char seg_a[12] = {}, seg_b[12] = {};
  int64_t M = 0, N = 0, K = 0;  // K: one pair's reduction length
  int groups = 1, group_a = 0, follower_b = 0;
  DenseEpi e;
  const char* what = "";

  int kbs() const { return static_cast<int>((K + 63) / 64); }
  int64_t m_tiles() const { return (M + 255) / 256; }
  int64_t n_tiles() const { return epi == kEpiGated ? (N + 127) / 128 : (N + 255) / 256; }
  int splits(const vmoe_ops* o) const {
    return choose_splits(m_tiles() * n_tiles() * groups, segs * kbs(), o->num_sms / 2,
                         M * n_tiles() * 1024 * groups);
  }
};

// Lays a product out: its tiles, its splits and, where it has splits or `partials` asks for
// them, its partial sums.
DenseGemm plan_product(Call& c, const Product& p, bool partials) {
  DenseGemm g;
  g.M = p.M;
  g.N = p.N;
  g.m_tiles = static_cast<int>(p.m_tiles());
  g.n_tiles = static_cast<int>(p.n_tiles());
  g.segs = p.segs;
  g.kbs = p.kbs();
  memcpy(g.seg_a, p.seg_a, sizeof(g.seg_a));
  memcpy(g.seg_b, p.seg_b, sizeof(g.seg_b));
  g.groups = p.groups;
  g.group_a = p.group_a;
  g.follower_b = p.follower_b;
  g.ldp = p.n_tiles() * 256;
  g.splits = p.splits(c.o);
  g.kb_per_split = (p.segs * g.kbs + g.splits - 1) / g.splits;
  g.band = g.n_tiles < 8 ? g.n_tiles : 8;
  g.epi = p.e;
  g.status = c.o->status;
  if (g.splits > 1 || partials)
    g.partial = c.ws.take<float>(static_cast<size_t>(p.M * g.ldp * 4 * p.groups) * g.splits);
  return g;
}

int launch_product(Call& c, const Product& p, const DenseGemm& g) {
  DenseMaps maps;
  char why[256];
  for (int i = 0; i < 6; ++i) {
    const struct { CUtensorMap* map; const Mat& m; bool mn; } two[2] = {
        {&maps.a[i], p.a[i], p.a_mn}, {&maps.b[i], p.b[i], p.b_mn}};
    for (const auto& t : two) {
      if (t.m.p && !make_tmap_bf16(t.map, t.m.p, static_cast<uint64_t>(t.m.rows),
                                   static_cast<uint64_t>(t.m.cols), static_cast<uint64_t>(t.m.ld),
                                   t.mn ? 64 : 128, why, sizeof(why)))
        return ops_fail(c.o, VMOE_ERR_CUDA, "%s: %s", p.what, why);
    }
  }
  return c.run(
      [&] { return launch_gemm_dense(p.a_mn, p.b_mn, p.epi, maps, g, c.o->num_sms, c.s); }, p.what);
}

int check_tiles(Call& c, const Product& p) {
  if (p.m_tiles() * p.n_tiles() * p.groups * 16 > 0x7fffffff)
    return ops_fail(c.o, VMOE_ERR_UNSUPPORTED_SHAPE, "%s: too many output tiles", p.what);
  return VMOE_OK;
}

// One bf16 product, split over k where its tiles leave SMs idle.
int run_product(Call& c, const Product& p) {
  TRY(check_tiles(c, p));
  const DenseGemm g = plan_product(c, p, false);
  if (c.dry) return VMOE_OK;
  TRY(launch_product(c, p, g));
  if (!g.partial) return VMOE_OK;
  return c.run([&] { return launch_dense_finish(kBF16, p.epi, g, c.s); }, p.what);
}

// The same for a decode batch's forward: x [T, K] and weights [N, K] (gated: two of them).
int run_skinny(Call& c, int epi, Mat x, Mat w, Mat w2, const DenseEpi& e, const char* what,
               bool second = false) {
  // a second product's weights may be asked for early, unless they are copied just before
  const bool early = second && w.ld % 8 == 0;
  TRY(c.tma_ready(x, what));
  TRY(c.tma_ready(w, what));
  if (epi == kEpiGated) TRY(c.tma_ready(w2, what));
  if (c.dry) return VMOE_OK;
  CUtensorMap mw, mw2, mx;
  char why[256];
  auto map = [&](CUtensorMap* m, const Mat& t, int64_t box) {
    return make_tmap_bf16(m, t.p, static_cast<uint64_t>(t.rows), static_cast<uint64_t>(t.cols),
                          static_cast<uint64_t>(t.ld), static_cast<uint32_t>(box), why, sizeof(why));
  };
  const bool gated = epi == kEpiGated;
  if (!map(&mx, x, round_up(x.rows, 16)) || !map(&mw, w, gated ? 64 : 128) ||
      (gated && !map(&mw2, w2, 64)))
    return ops_fail(c.o, VMOE_ERR_CUDA, "%s: %s", what, why);
  if (!gated) mw2 = mw;
  SkinnyGemm g{};
  g.T = x.rows;
  g.N = w.rows;
  g.kbs = static_cast<int>((x.cols + 63) / 64);
  g.epi = e;
  g.status = c.o->status;
  g.early_weights = early;
  return c.run([&] { return launch_dense_skinny(epi, mw, mw2, mx, g, c.s); }, what);
}

// ---- fp32 products: six bf16 ones (dense_f32.cu) -------------------------------------------
struct F32Mat {
  const float* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
  Mat plane[3];
};

// The planes of one call's matrices, and its products' redo words, which the first launch clears.
struct F32Planes {
  int* words = nullptr;
  int used = 0;
  bool cleared = false;

  explicit F32Planes(Call& c) { words = c.ws.take<int>(kRedoWords * sizeof(int)); }

  int* word() { return words ? words + used++ : nullptr; }

  int split(Call& c, std::initializer_list<F32Mat*> mats) {
    Split3 s[3];
    int k = 0;
    for (F32Mat* m : mats) {
      const int64_t ld = round_up(m->cols, 8), plane = m->rows * ld;
      auto* out = c.ws.take<uint16_t>(static_cast<size_t>(3 * plane) * 2);
      for (int i = 0; i < 3; ++i)
        m->plane[i] = {out ? out + i * plane : nullptr, m->rows, m->cols, ld};
      s[k++] = {m->p, m->ld, m->rows, m->cols, out, ld, plane};
    }
    int* clear = cleared ? nullptr : words;
    cleared = true;
    if (c.dry) return VMOE_OK;
    return c.run([&] { return launch_split3(s, k, clear, c.s); }, "fp32 planes");
  }
};

// k blocks (64 products per output each) that an fp32 product's accumulator takes before it is
// read out and added in registers.
constexpr int kF32RunBlocks = 8;

// C = sum over the pairs of A B, or with two groups (gated: two Bs) one product for each, then
// the epilogue.  p.a / p.b and the pairs' lists are filled in here.
int run_f32(Call& c, Product p, F32Planes& planes, std::initializer_list<const F32Mat*> as,
            std::initializer_list<const F32Mat*> bs) {
  TRY(check_tiles(c, p));
  const int na = static_cast<int>(as.size()), nb = static_cast<int>(bs.size());
  const bool two_pairs = na == 2 && nb == 2;
  int i = 0;
  for (const F32Mat* m : as)
    for (int k = 0; k < 3; ++k) p.a[i++] = m->plane[k];
  i = 0;
  for (const F32Mat* m : bs)
    for (int k = 0; k < 3; ++k) p.b[i++] = m->plane[k];
  static const unsigned char ka[6] = {2, 0, 1, 1, 0, 0}, kb[6] = {0, 2, 1, 0, 1, 0};
  p.segs = two_pairs ? 12 : 6;
  for (int s = 0; s < p.segs; ++s) {  // both pairs' small terms first
    const int pair = two_pairs ? s % 2 : 0, t = two_pairs ? s / 2 : s;
    p.seg_a[s] = static_cast<unsigned char>(3 * pair + ka[t]);
    p.seg_b[s] = static_cast<unsigned char>(3 * pair + kb[t]);
  }
  p.group_a = 3;
  p.follower_b = p.epi == kEpiGated ? 3 : 0;
  DenseGemm g = plan_product(c, p, true);
  g.run_kb = kF32RunBlocks;
  g.redo_tiles = redo_tiles(p.epi, p.M, p.N, p.groups);
  g.arrived = c.ws.take<int>(static_cast<size_t>(g.redo_tiles) * sizeof(int));
  if (c.dry) return VMOE_OK;
  if (planes.used == kRedoWords)
    return ops_fail(c.o, VMOE_ERR_UNSUPPORTED_SHAPE, "%s: too many products in a call", p.what);
  g.redo = planes.word();
  TRY(launch_product(c, p, g));
  TRY(c.run([&] { return launch_dense_finish(kF32, p.epi, g, c.s); }, p.what));
  RedoGemm r{};
  r.g = g;
  const F32Mat &a = *as.begin()[0], &b = *bs.begin()[0];
  for (int q = 0; q < 2; ++q) {
    r.a[q] = as.begin()[na == 2 ? q : 0]->p;
    r.b[q] = bs.begin()[nb == 2 ? q : 0]->p;
  }
  r.pairs = two_pairs ? 2 : 1;
  r.am = p.a_mn ? 1 : a.ld;  // both of a kind have one pitch
  r.ak = p.a_mn ? a.ld : 1;
  r.bn = p.b_mn ? 1 : b.ld;
  r.bk = p.b_mn ? b.ld : 1;
  r.K = p.K;
  return c.run([&] { return launch_dense_redo(p.epi, r, c.o->num_sms, c.s); }, p.what);
}

constexpr int kDzBlocksPerSm = 6;
// so few rows are summed by one block per column strip, which spares the second launch
constexpr int64_t kDzOneBlock = 256;

// dz = dy act'(z) (written when `dz` is given) and the column sums into `db`.
int run_dz(Call& c, const void* dy, int64_t lddy, const void* z, int64_t ldz, void* dz,
           int64_t lddz, int64_t T, int64_t N, int act, float gamma, void* db, bool db_f32) {
  if (!dz && !db) return VMOE_OK;
  DzArgs a{};
  a.dy = dy;
  a.lddy = lddy;
  a.z = z;
  a.ldz = ldz;
  a.dz = dz;
  a.lddz = lddz;
  a.T = T;
  a.N = N;
  a.act = act;
  a.gamma = gamma;
  const int64_t width = 32 * (c.dtype == kF32 ? 4 : 8);
  const int64_t strips = (N + width - 1) / width;
  int64_t rb = (kDzBlocksPerSm * static_cast<int64_t>(c.o->num_sms) + strips - 1) / strips;
  if (rb > (T + 31) / 32) rb = (T + 31) / 32;
  if (rb > 128) rb = 128;
  if (rb < 1 || T <= kDzOneBlock) rb = 1;
  a.rows_per_block = (T + rb - 1) / rb;
  a.row_blocks = static_cast<int>((T + a.rows_per_block - 1) / a.rows_per_block);
  if (db && a.row_blocks == 1) {
    a.db = db;
    a.db_f32 = db_f32;
  } else if (db) {
    a.colsum = c.ws.take<float>(static_cast<size_t>(a.row_blocks) * N * 4);
  }
  if (c.dry) return VMOE_OK;
  TRY(c.run([&] { return launch_dense_dz(c.dtype, a, c.s); }, "activation gradient"));
  if (a.colsum)
    return c.run([&] { return launch_colsum_finish(a.colsum, a.row_blocks, N, db, nullptr, db_f32, c.s); }, "bias gradient");
  return VMOE_OK;
}

constexpr int64_t kMaxDim = (static_cast<int64_t>(1) << 31) - 1;

int check_common(vmoe_ops* o, int64_t T, int32_t dtype, int32_t act, int32_t grad_dtype,
                 float gamma) {
  if (T < 0 || T > kMaxDim)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "tokens must be in [0, 2^31) (got %lld)",
                    static_cast<long long>(T));
  if (dtype != VMOE_F32 && dtype != VMOE_BF16)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "dtype must be VMOE_F32 or VMOE_BF16 (got %d)", dtype);
  if (grad_dtype != VMOE_F32 && grad_dtype != dtype)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "grad_dtype must be dtype or VMOE_F32 (got %d)",
                    grad_dtype);
  if (act < VMOE_ACT_NONE || act > VMOE_ACT_ERA)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "unknown activation %d", act);
  if (act == VMOE_ACT_ERA && !(gamma - gamma == 0.f))
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "gamma must be finite");
  if (!o->sm100)  // fp32 products run on the tensor cores too
    return ops_fail(o, VMOE_ERR_UNSUPPORTED_SHAPE, "the dense operators need an sm_100 GPU");
  return VMOE_OK;
}

int check_dim(vmoe_ops* o, const char* name, int64_t v) {
  if (v < 1 || v > kMaxDim)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "%s must be in [1, 2^31) (got %lld)", name,
                    static_cast<long long>(v));
  return VMOE_OK;
}

// A matrix of the call: below 2^40 elements, so that no size or offset derived from it (its
// bytes, three planes, two groups of 16 splits) leaves 64 bits.
int check_area(vmoe_ops* o, const char* name, int64_t rows, int64_t cols) {
  if (rows * cols > static_cast<int64_t>(1) << 40)  // both are below 2^31
    return ops_fail(o, VMOE_ERR_UNSUPPORTED_SHAPE, "%s of %lld x %lld is more than 2^40 elements",
                    name, static_cast<long long>(rows), static_cast<long long>(cols));
  return VMOE_OK;
}

int check_ld(vmoe_ops* o, const char* name, int64_t ld, int64_t cols) {
  if (ld < cols || ld > (static_cast<int64_t>(1) << 36))
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "%s must be at least the row length %lld (got %lld)",
                    name, static_cast<long long>(cols), static_cast<long long>(ld));
  return VMOE_OK;
}

// bf16 matrices the TMA reads in place start on a 16-byte boundary; anything is aligned to
// its element
int check_ptr(vmoe_ops* o, const char* name, const void* p, int64_t ld, int dtype) {
  if (!p) return ops_fail(o, VMOE_ERR_INVALID_ARG, "%s is required", name);
  if (dtype == VMOE_BF16 && ld % 8 == 0 && !aligned16(p))
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "%s must be 16-byte aligned", name);
  if (reinterpret_cast<uintptr_t>(p) & (dtype_bytes(dtype) - 1))
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "%s is not aligned to its elements", name);
  return VMOE_OK;
}

// an operand that is read or written element by element, or none
int check_elt(vmoe_ops* o, const char* name, const void* p, size_t elt) {
  if (reinterpret_cast<uintptr_t>(p) & (elt - 1))
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "%s is not aligned to its elements", name);
  return VMOE_OK;
}

// dy [T, cols]: contiguous, or (bf16) a pitch the TMA reads in place, so that the workspace
// size needs no pitch
int check_dy(vmoe_ops* o, const void* dy, int64_t lddy, int64_t cols, int dtype) {
  TRY(check_ld(o, "lddy", lddy, cols));
  if (dtype == VMOE_BF16 && lddy != cols && lddy % 8)
    return ops_fail(o, VMOE_ERR_INVALID_ARG,
                    "lddy must be the row length or a multiple of 8 (got %lld)",
                    static_cast<long long>(lddy));
  return check_ptr(o, "dy", dy, lddy, dtype);
}

int check_linear(vmoe_ops* o, const vmoe_linear* d) {
  TRY(check_common(o, d->tokens, d->dtype, d->activation, d->grad_dtype, d->gamma));
  TRY(check_dim(o, "in_features", d->in_features));
  TRY(check_dim(o, "out_features", d->out_features));
  TRY(check_area(o, "x", d->tokens, d->in_features));
  TRY(check_area(o, "y", d->tokens, d->out_features));
  TRY(check_area(o, "weight", d->out_features, d->in_features));
  TRY(check_ld(o, "ldx", d->ldx, d->in_features));
  return check_ld(o, "ldw", d->ldw, d->in_features);
}

int check_ffn(vmoe_ops* o, const vmoe_gated_ffn* d) {
  TRY(check_common(o, d->tokens, d->dtype, d->activation, d->grad_dtype, d->gamma));
  if (d->activation == VMOE_ACT_NONE)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "the gated block needs an activation");
  TRY(check_dim(o, "hidden", d->hidden));
  TRY(check_dim(o, "inter", d->inter));
  TRY(check_area(o, "x", d->tokens, d->hidden));
  TRY(check_area(o, "h", d->tokens, d->inter));
  TRY(check_area(o, "weight", d->inter, d->hidden));
  return check_ld(o, "ldx", d->ldx, d->hidden);
}

int check_workspace(vmoe_ops* o, const void* ws, size_t have, size_t need) {
  if (need == 0) return VMOE_OK;
  if (!ws || have < need)
    return ops_fail(o, VMOE_ERR_WORKSPACE, "workspace needs %zu bytes (got %zu)", need,
                    ws ? have : static_cast<size_t>(0));
  if (reinterpret_cast<uintptr_t>(ws) & 255u)
    return ops_fail(o, VMOE_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  return VMOE_OK;
}

// ---- fused linear ------------------------------------------------------------------------
struct LinearPtrs {
  const void *x, *w, *b, *r, *z_in, *dy;
  int64_t lddy;
  void *y, *z, *dx, *dw, *db;
};

int linear_forward(Call& c, const vmoe_linear& d, const LinearPtrs& p) {
  const int64_t T = d.tokens, K = d.in_features, N = d.out_features;
  const size_t elt = dtype_bytes(d.dtype);
  DenseEpi e;
  e.act = d.activation;
  e.gamma = d.gamma;
  e.bias = p.b;
  e.res = p.r;
  e.ldr = d.ldr;
  e.out = p.y;
  e.ldo = N;
  e.z = p.z;
  e.ldz = N;
  e.vec = (vec_ok(p.y, N, N, elt) ? kVecOut : 0) | (vec_ok(p.r, d.ldr, N, elt) ? kVecRes : 0) |
          (vec_ok(p.z, N, N, elt) ? kVecZ : 0);
  if (T <= kSmallTokens) {
    if (c.dry) return VMOE_OK;
    SmallGemm g{};
    g.x = p.x;
    g.w = p.w;
    g.ldx = d.ldx;
    g.ldw = d.ldw;
    g.T = T;
    g.N = N;
    g.K = K;
    g.epi = e;
    g.num_sms = c.o->num_sms;
    g.status = c.o->status;
    g.vec_in = K * elt % 16 == 0 && pitch16(p.x, d.ldx, elt) && pitch16(p.w, d.ldw, elt);
    return c.run([&] { return launch_dense_small(d.dtype, kEpiLinear, g, c.s); }, "linear");
  }
  c.overlap = d.dtype == VMOE_F32;
  if (d.dtype == VMOE_BF16 && T <= kSkinnyTokens)
    return run_skinny(c, kEpiLinear, {p.x, T, K, d.ldx}, {p.w, N, K, d.ldw}, {}, e, "linear");
  Product q;
  q.M = T;
  q.N = N;
  q.K = K;
  q.e = e;
  q.what = "linear";
  if (d.dtype == VMOE_F32) {
    F32Mat x{static_cast<const float*>(p.x), T, K, d.ldx}, w{static_cast<const float*>(p.w), N, K, d.ldw};
    F32Planes planes(c);
    TRY(planes.split(c, {&x, &w}));
    return run_f32(c, q, planes, {&x}, {&w});
  }
  q.a[0] = {p.x, T, K, d.ldx};
  q.b[0] = {p.w, N, K, d.ldw};
  TRY(c.tma_ready(q.a[0], "linear"));
  TRY(c.tma_ready(q.b[0], "linear"));
  return run_product(c, q);
}

int linear_backward(Call& c, const vmoe_linear& d, const LinearPtrs& p) {
  const int64_t T = d.tokens, K = d.in_features, N = d.out_features;
  const size_t elt = dtype_bytes(d.dtype);
  const bool gf32 = d.grad_dtype == VMOE_F32;
  const size_t gelt = gf32 ? 4 : elt;
  // every size below holds for any of the outputs being absent
  const bool f32 = d.dtype == VMOE_F32;
  const bool copy = d.activation != VMOE_ACT_NONE || (!f32 && p.lddy % 8 != 0);
  const bool products = c.dry || p.dx || p.dw;
  const void* dz = p.dy;
  int64_t lddz = p.lddy;
  if (copy && products) {
    lddz = round_up(N, 8);
    dz = c.ws.take(static_cast<size_t>(T) * lddz * elt);
  }
  TRY(run_dz(c, p.dy, p.lddy, p.z_in, N, copy && products ? const_cast<void*>(dz) : nullptr, lddz,
             T, N, d.activation, d.gamma, c.dry ? static_cast<void*>(c.o) : p.db, gf32));
  DenseEpi ex, ew;
  ex.out = p.dx;
  ex.ldo = K;
  ex.vec = vec_ok(p.dx, K, K, elt) ? kVecOut : 0;
  ew.out = p.dw;
  ew.ldo = K;
  ew.out_f32 = gf32;
  ew.vec = vec_ok(p.dw, K, K, gelt) ? kVecOut : 0;
  Product qx, qw;
  qx.b_mn = true;
  qx.M = T;
  qx.N = K;
  qx.K = N;
  qx.e = ex;
  qx.what = "linear dx";
  qw.a_mn = qw.b_mn = true;
  qw.M = N;
  qw.N = K;
  qw.K = T;
  qw.e = ew;
  qw.what = "linear dW";
  const bool need_x = c.dry || p.dx, need_w = c.dry || p.dw;
  if (!need_x && !need_w) return VMOE_OK;
  if (f32) {
    F32Mat z{static_cast<const float*>(dz), T, N, lddz}, x{static_cast<const float*>(p.x), T, K, d.ldx},
        w{static_cast<const float*>(p.w), N, K, d.ldw};
    F32Planes planes(c);
    if (need_x && need_w) TRY(planes.split(c, {&z, &x, &w}));
    else if (need_x) TRY(planes.split(c, {&z, &w}));
    else TRY(planes.split(c, {&z, &x}));
    if (need_x) TRY(run_f32(c, qx, planes, {&z}, {&w}));
    if (need_w) TRY(run_f32(c, qw, planes, {&z}, {&x}));
    return VMOE_OK;
  }
  const Mat z{dz, T, N, lddz};
  if (need_x) {
    qx.a[0] = z;
    qx.b[0] = {p.w, N, K, d.ldw};
    TRY(c.tma_ready(qx.b[0], "linear dx"));
    TRY(run_product(c, qx));
  }
  if (need_w) {
    qw.a[0] = z;
    qw.b[0] = {p.x, T, K, d.ldx};
    TRY(c.tma_ready(qw.b[0], "linear dW"));
    TRY(run_product(c, qw));
  }
  return VMOE_OK;
}

// ---- gated feed-forward block --------------------------------------------------------------
struct FfnPtrs {
  const void* x;
  vmoe_ffn_weights w;
  const void *r, *dy;
  int64_t lddy;
  void *y, *dx;
  vmoe_ffn_grads grads;
  char* saved;  // training: g | u | h
};

// g and u [T, ld] in fp32, then h [T, ld]; ld keeps every row in whole 16-byte units
struct FfnSaved {
  int64_t ld;
  size_t part, total;  // bytes of g (and of u), and of all
};

FfnSaved ffn_saved(const vmoe_gated_ffn& d) {
  FfnSaved s;
  s.ld = round_up(d.inter, 8);
  auto round256 = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
  const size_t n = static_cast<size_t>(d.tokens) * s.ld;
  s.part = round256(n * 4);
  s.total = 2 * s.part + round256(n * dtype_bytes(d.dtype));
  return s;
}

int ffn_forward(Call& c, const vmoe_gated_ffn& d, const FfnPtrs& p) {
  const int64_t T = d.tokens, H = d.hidden, I = d.inter;
  const size_t elt = dtype_bytes(d.dtype);
  const FfnSaved sv = ffn_saved(d);
  void* h = p.saved && !c.dry ? static_cast<void*>(p.saved + 2 * sv.part)
                              : c.ws.take(static_cast<size_t>(T) * sv.ld * elt);
  DenseEpi e1, e2;
  e1.act = d.activation;
  e1.gamma = d.gamma;
  e1.bias = p.w.gate_b;
  e1.bias2 = p.w.up_b;
  e1.out = h;
  e1.ldo = sv.ld;
  if (p.saved) {
    e1.z = p.saved;
    e1.z2 = p.saved + sv.part;
  }
  e1.ldz = sv.ld;
  e1.vec = kVecOut | kVecZ;
  e2.bias = p.w.down_b;
  e2.res = p.r;
  e2.ldr = d.ldr;
  e2.out = p.y;
  e2.ldo = H;
  e2.vec = (vec_ok(p.y, H, H, elt) ? kVecOut : 0) | (vec_ok(p.r, d.ldr, H, elt) ? kVecRes : 0);
  if (T <= kSmallTokens) {
    if (c.dry) return VMOE_OK;
    SmallGemm g{};
    g.x = p.x;
    g.w = p.w.gate_w;
    g.w2 = p.w.up_w;
    g.ldx = d.ldx;
    g.ldw = g.ldw2 = H;
    g.T = T;
    g.N = I;
    g.K = H;
    g.epi = e1;
    g.num_sms = c.o->num_sms;
    g.status = c.o->status;
    g.vec_in = H * elt % 16 == 0 && pitch16(p.x, d.ldx, elt) && aligned16(p.w.gate_w) &&
               aligned16(p.w.up_w);
    TRY(c.run([&] { return launch_dense_small(d.dtype, kEpiGated, g, c.s); }, "gate|up"));
    SmallGemm q{};
    q.x = h;
    q.w = p.w.down_w;
    q.ldx = sv.ld;
    q.ldw = I;
    q.T = T;
    q.N = H;
    q.K = I;
    q.epi = e2;
    q.num_sms = c.o->num_sms;
    q.status = c.o->status;
    q.early_weights = 1;
    q.vec_in = I * elt % 16 == 0 && aligned16(p.w.down_w);
    return c.run([&] { return launch_dense_small(d.dtype, kEpiLinear, q, c.s); }, "down");
  }
  if (d.dtype == VMOE_BF16 && T <= kSkinnyTokens) {
    TRY(run_skinny(c, kEpiGated, {p.x, T, H, d.ldx}, {p.w.gate_w, I, H, H}, {p.w.up_w, I, H, H}, e1,
                   "gate|up"));
    return run_skinny(c, kEpiLinear, {h, T, I, sv.ld}, {p.w.down_w, H, I, I}, {}, e2, "down", true);
  }
  c.overlap = d.dtype == VMOE_F32;
  Product g, q;
  g.epi = kEpiGated;
  g.M = T;
  g.N = I;
  g.K = H;
  g.e = e1;
  g.what = "gate|up";
  q.M = T;
  q.N = H;
  q.K = I;
  q.e = e2;
  q.what = "down";
  if (d.dtype == VMOE_F32) {
    auto F = [](const void* m) { return static_cast<const float*>(m); };
    F32Mat x{F(p.x), T, H, d.ldx}, wg{F(p.w.gate_w), I, H, H}, wu{F(p.w.up_w), I, H, H},
        hm{F(h), T, I, sv.ld}, wd{F(p.w.down_w), H, I, I};
    F32Planes planes(c);
    TRY(planes.split(c, {&x, &wg, &wu}));
    TRY(run_f32(c, g, planes, {&x}, {&wg, &wu}));
    TRY(planes.split(c, {&hm, &wd}));
    return run_f32(c, q, planes, {&hm}, {&wd});
  }
  g.follower_b = 1;
  g.a[0] = {p.x, T, H, d.ldx};
  g.b[0] = {p.w.gate_w, I, H, H};
  g.b[1] = {p.w.up_w, I, H, H};
  TRY(c.tma_ready(g.a[0], "gate|up"));
  TRY(c.tma_ready(g.b[0], "gate|up"));
  TRY(c.tma_ready(g.b[1], "gate|up"));
  TRY(run_product(c, g));
  q.a[0] = {h, T, I, sv.ld};
  q.b[0] = {p.w.down_w, H, I, I};
  TRY(c.tma_ready(q.b[0], "down"));
  return run_product(c, q);
}

int ffn_backward(Call& c, const vmoe_gated_ffn& d, const FfnPtrs& p) {
  const int64_t T = d.tokens, H = d.hidden, I = d.inter;
  const size_t elt = dtype_bytes(d.dtype);
  const bool gf32 = d.grad_dtype == VMOE_F32;
  const size_t gelt = gf32 ? 4 : elt;
  const bool f32 = d.dtype == VMOE_F32;
  const FfnSaved sv = ffn_saved(d);
  const vmoe_ffn_grads& gr = p.grads;
  const void* g = p.saved;
  const void* u = p.saved ? p.saved + sv.part : nullptr;
  const void* h = p.saved ? p.saved + 2 * sv.part : nullptr;
  void* any = c.o;  // sizes count every output
  const int64_t row_blocks = (T + 31) / 32;
  float* colsum = nullptr;
  bool summed = false;
  // the activation's side: dg and du
  const bool need_dgu = c.dry || p.dx || gr.gate_w || gr.up_w || gr.gate_b || gr.up_b;
  void *dg = nullptr, *du = nullptr;
  if (need_dgu) {
    dg = c.ws.take(static_cast<size_t>(T) * sv.ld * elt);
    du = c.ws.take(static_cast<size_t>(T) * sv.ld * elt);
  }
  Mat dy{p.dy, T, H, p.lddy};
  if (!f32) TRY(c.tma_ready(dy, "dy"));
  if (c.dry || gr.down_b)
    TRY(run_dz(c, p.dy, p.lddy, nullptr, 0, nullptr, 0, T, H, kActNone, 0.f,
               c.dry ? any : gr.down_b, gf32));
  DenseEpi e;
  e.act = d.activation;
  e.gamma = d.gamma;
  e.z = const_cast<void*>(g);
  e.z2 = const_cast<void*>(u);
  e.ldz = sv.ld;
  e.out = dg;
  e.out2 = du;
  e.ldo = sv.ld;
  e.vec = kVecOut | kVecZ;
  auto plain = [&](void* out, int64_t ld, bool grad) {
    DenseEpi q;
    q.out = out;
    q.ldo = ld;
    q.out_f32 = grad && gf32;
    q.vec = vec_ok(out, ld, ld, grad ? gelt : elt) ? kVecOut : 0;
    return q;
  };
  Product qh, qx, qgu, qd;
  qh.b_mn = true;
  qh.epi = kEpiGluBwd;
  qh.M = T;
  qh.N = I;
  qh.K = H;
  qh.e = e;
  qh.what = "dh";
  qx.b_mn = true;
  qx.M = T;
  qx.N = H;
  qx.K = I;
  qx.e = plain(p.dx, H, false);
  qx.what = "dx";
  const bool need_x = c.dry || p.dx;
  // the gate's and the up's weight gradients in one launch where both are asked for
  const bool need_gu = c.dry || gr.gate_w || gr.up_w, both = c.dry || (gr.gate_w && gr.up_w);
  const bool only_up = !both && gr.up_w;
  qgu.a_mn = qgu.b_mn = true;
  qgu.M = I;
  qgu.N = H;
  qgu.K = T;
  qgu.groups = both ? 2 : 1;
  qgu.e = plain(only_up ? gr.up_w : gr.gate_w, H, true);
  if (both) {
    qgu.e.out2 = gr.up_w;
    if (!vec_ok(gr.up_w, H, H, gelt)) qgu.e.vec = 0;
  }
  qgu.what = "dW gate|up";
  const bool need_d = c.dry || gr.down_w;
  qd.a_mn = qd.b_mn = true;
  qd.M = H;
  qd.N = I;
  qd.K = T;
  qd.e = plain(gr.down_w, I, true);
  qd.what = "dW down";
  if (f32) {
    auto F = [](const void* m) { return static_cast<const float*>(m); };
    F32Mat mdy{F(p.dy), T, H, p.lddy}, wd{F(p.w.down_w), H, I, I}, mdg{F(dg), T, I, sv.ld},
        mdu{F(du), T, I, sv.ld}, x{F(p.x), T, H, d.ldx}, wg{F(p.w.gate_w), I, H, H},
        wu{F(p.w.up_w), I, H, H}, hm{F(h), T, I, sv.ld};
    F32Planes planes(c);
    if (need_dgu) {
      TRY(planes.split(c, {&mdy, &wd}));
      TRY(run_f32(c, qh, planes, {&mdy}, {&wd}));
      if (need_x || need_gu) TRY(planes.split(c, {&mdg, &mdu}));
    } else if (need_d) {
      TRY(planes.split(c, {&mdy}));
    }
    if (need_x) {
      TRY(planes.split(c, {&wg, &wu}));
      TRY(run_f32(c, qx, planes, {&mdg, &mdu}, {&wg, &wu}));
    }
    if (need_gu) {
      TRY(planes.split(c, {&x}));
      if (both) TRY(run_f32(c, qgu, planes, {&mdg, &mdu}, {&x}));
      if (c.dry) qgu.groups = 1;  // one gradient alone may be split into more parts
      if (c.dry || !both) TRY(run_f32(c, qgu, planes, {only_up ? &mdu : &mdg}, {&x}));
    }
    if (need_d) {
      TRY(planes.split(c, {&hm}));
      TRY(run_f32(c, qd, planes, {&mdy}, {&hm}));
    }
  } else {
    if (need_dgu) {
      qh.a[0] = dy;
      qh.b[0] = {p.w.down_w, H, I, I};
      TRY(c.tma_ready(qh.b[0], "dh"));
      // the gate's and the up's bias gradients: column sums in the epilogue, where it runs once
      if ((c.dry || gr.gate_b || gr.up_b) && qh.splits(c.o) == 1) {
        qh.e.colsum_stride = row_blocks * I;
        qh.e.colsum = colsum = c.ws.take<float>(static_cast<size_t>(2 * row_blocks * I) * 4);
        summed = true;
      }
      TRY(run_product(c, qh));
    }
    const Mat mdg{dg, T, I, sv.ld}, mdu{du, T, I, sv.ld};
    if (need_x) {
      qx.segs = 2;
      qx.seg_a[1] = qx.seg_b[1] = 1;
      qx.a[0] = mdg;
      qx.a[1] = mdu;
      qx.b[0] = {p.w.gate_w, I, H, H};
      qx.b[1] = {p.w.up_w, I, H, H};
      TRY(c.tma_ready(qx.b[0], "dx"));
      TRY(c.tma_ready(qx.b[1], "dx"));
      TRY(run_product(c, qx));
    }
    if (need_gu) {
      qgu.b[0] = {p.x, T, H, d.ldx};
      TRY(c.tma_ready(qgu.b[0], "dW gate|up"));
      qgu.group_a = 1;
      qgu.a[0] = only_up ? mdu : mdg;
      if (both) qgu.a[1] = mdu;
      TRY(run_product(c, qgu));
      if (c.dry) {
        qgu.groups = 1;
        TRY(run_product(c, qgu));
      }
    }
    if (need_d) {
      qd.a[0] = dy;
      qd.b[0] = {h, T, I, sv.ld};
      TRY(run_product(c, qd));
    }
  }
  if (summed) {
    if (c.dry) return VMOE_OK;
    if (!gr.gate_b) {
      if (!gr.up_b) return VMOE_OK;
      return c.run(
          [&] {
            return launch_colsum_finish(colsum + row_blocks * I, row_blocks, I, gr.up_b, nullptr,
                                        gf32, c.s);
          },
          "dbu");
    }
    return c.run(
        [&] { return launch_colsum_finish(colsum, row_blocks, I, gr.gate_b, gr.up_b, gf32, c.s); },
        "dbg");
  }
  TRY(run_dz(c, dg, sv.ld, nullptr, 0, nullptr, 0, T, I, kActNone, 0.f, c.dry ? any : gr.gate_b,
             gf32));
  return run_dz(c, du, sv.ld, nullptr, 0, nullptr, 0, T, I, kActNone, 0.f, c.dry ? any : gr.up_b,
                gf32);
}

}  // namespace

extern "C" {

int vmoe_ops_create(int device, vmoe_ops** out) {
  if (!out) return VMOE_ERR_INVALID_ARG;
  *out = nullptr;
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
    cudaGetLastError();
    fprintf(stderr, "vmoe_ops_create: CUDA device %d is not available\n", device);
    return VMOE_ERR_CUDA;
  }
  vmoe_ops* o = new (std::nothrow) vmoe_ops();
  if (!o) return VMOE_ERR_CUDA;
  o->device = device;
  DeviceGuard g(device);
  int major = 0, minor = 0;
  cudaDeviceGetAttribute(&o->num_sms, cudaDevAttrMultiProcessorCount, device);
  cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
  o->sm100 = major == 10 && minor == 0;
  // the word is the library's own: a thread whose first call falls into a stream capture (a
  // captured backward on autograd's thread) must allocate and clear nothing
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  void* word = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&word, g_ops_status);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) {
    fprintf(stderr, "vmoe_ops_create: %s\n", cudaGetErrorString(e));
    delete o;
    return VMOE_ERR_CUDA;
  }
  o->status = static_cast<int*>(word);
  *out = o;
  return VMOE_OK;
}

int vmoe_ops_destroy(vmoe_ops* o) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  delete o;
  return VMOE_OK;
}

const char* vmoe_ops_last_error(const vmoe_ops* o) { return o ? o->err : ""; }

int vmoe_ops_device_status(vmoe_ops* o, int32_t* code, void* stream) {
  if (!o || !code) return VMOE_ERR_INVALID_ARG;
  DeviceGuard g(o->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int v = 0;
  cudaError_t e = cudaMemcpyAsync(&v, o->status, sizeof(int), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess) e = cudaMemsetAsync(o->status, 0, sizeof(int), s);
  if (e != cudaSuccess) return ops_cuda_fail(o, e, "status read");
  *code = v;
  if (v == 0) return VMOE_OK;
  if (v >= 0x101 && v <= 0x1FF)
    return ops_fail(o, VMOE_ERR_TIMEOUT, "a bounded device wait gave up (status 0x%x)", v);
  return ops_fail(o, VMOE_ERR_DEVICE_STATUS, "device status 0x%x", v);
}

int vmoe_linear_workspace_size(vmoe_ops* o, const vmoe_linear* d, int backward, size_t* bytes) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (!d || !bytes) return ops_fail(o, VMOE_ERR_INVALID_ARG, "d and bytes are required");
  TRY(check_linear(o, d));
  *bytes = 0;
  if (d->tokens == 0) return VMOE_OK;
  Call c{o, {}, nullptr, true, d->dtype};
  LinearPtrs p{};
  p.lddy = d->out_features;
  TRY(backward ? linear_backward(c, *d, p) : linear_forward(c, *d, p));
  *bytes = c.ws.off;
  return VMOE_OK;
}

int vmoe_linear_forward(vmoe_ops* o, const vmoe_linear* d, const void* x, const void* weight,
                        const void* bias, const void* residual, void* y, void* z, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (!d) return ops_fail(o, VMOE_ERR_INVALID_ARG, "d is required");
  size_t need = 0;
  TRY(vmoe_linear_workspace_size(o, d, 0, &need));
  if (d->tokens == 0) return VMOE_OK;
  TRY(check_ptr(o, "x", x, d->ldx, d->dtype));
  TRY(check_ptr(o, "weight", weight, d->ldw, d->dtype));
  if (residual) TRY(check_ld(o, "ldr", d->ldr, d->out_features));
  if (!y) return ops_fail(o, VMOE_ERR_INVALID_ARG, "y is required");
  const size_t elt = dtype_bytes(d->dtype);
  TRY(check_elt(o, "bias", bias, elt));
  TRY(check_elt(o, "residual", residual, elt));
  TRY(check_elt(o, "y", y, elt));
  TRY(check_elt(o, "z", z, elt));
  TRY(check_workspace(o, workspace, workspace_bytes, need));
  DeviceGuard g(o->device);
  Call c{o, {static_cast<char*>(workspace), 0}, static_cast<cudaStream_t>(stream), false, d->dtype};
  LinearPtrs p{};
  p.x = x;
  p.w = weight;
  p.b = bias;
  p.r = residual;
  p.y = y;
  p.z = z;
  return linear_forward(c, *d, p);
}

int vmoe_linear_backward(vmoe_ops* o, const vmoe_linear* d, const void* x, const void* weight,
                         const void* z, const void* dy, int64_t lddy, void* dx, void* dweight,
                         void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (!d) return ops_fail(o, VMOE_ERR_INVALID_ARG, "d is required");
  size_t need = 0;
  TRY(vmoe_linear_workspace_size(o, d, 1, &need));
  const size_t gelt = dtype_bytes(d->grad_dtype);
  TRY(check_elt(o, "dx", dx, dtype_bytes(d->dtype)));
  TRY(check_elt(o, "dweight", dweight, gelt));
  TRY(check_elt(o, "dbias", dbias, gelt));
  DeviceGuard g(o->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->tokens == 0) {  // sums over no rows
    cudaError_t e = cudaSuccess;
    if (dweight) e = cudaMemsetAsync(dweight, 0, d->in_features * d->out_features * gelt, s);
    if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, d->out_features * gelt, s);
    return e == cudaSuccess ? VMOE_OK : ops_cuda_fail(o, e, "zero gradients");
  }
  TRY(check_ptr(o, "x", x, d->ldx, d->dtype));
  TRY(check_ptr(o, "weight", weight, d->ldw, d->dtype));
  TRY(check_dy(o, dy, lddy, d->out_features, d->dtype));
  if (d->activation != VMOE_ACT_NONE && !z)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "the activation's gradient needs z");
  TRY(check_elt(o, "z", z, dtype_bytes(d->dtype)));
  TRY(check_workspace(o, workspace, workspace_bytes, need));
  Call c{o, {static_cast<char*>(workspace), 0}, s, false, d->dtype};
  LinearPtrs p{};
  p.x = x;
  p.w = weight;
  p.z_in = z;
  p.dy = dy;
  p.lddy = lddy;
  p.dx = dx;
  p.dw = dweight;
  p.db = dbias;
  return linear_backward(c, *d, p);
}

int vmoe_gated_ffn_workspace_size(vmoe_ops* o, const vmoe_gated_ffn* d, int backward,
                                  size_t* bytes, size_t* saved_bytes) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (!d || !bytes) return ops_fail(o, VMOE_ERR_INVALID_ARG, "d and bytes are required");
  TRY(check_ffn(o, d));
  *bytes = 0;
  if (saved_bytes) *saved_bytes = d->tokens ? ffn_saved(*d).total : 0;
  if (d->tokens == 0) return VMOE_OK;
  Call c{o, {}, nullptr, true, d->dtype};
  FfnPtrs p{};
  p.lddy = d->hidden;
  TRY(backward ? ffn_backward(c, *d, p) : ffn_forward(c, *d, p));
  *bytes = c.ws.off;
  return VMOE_OK;
}

namespace {
int check_ffn_call(vmoe_ops* o, const vmoe_gated_ffn* d, const void* x, const vmoe_ffn_weights* w) {
  if (!w) return ops_fail(o, VMOE_ERR_INVALID_ARG, "the weights are required");
  TRY(check_ptr(o, "x", x, d->ldx, d->dtype));
  TRY(check_ptr(o, "gate_w", w->gate_w, d->hidden, d->dtype));
  TRY(check_ptr(o, "up_w", w->up_w, d->hidden, d->dtype));
  return check_ptr(o, "down_w", w->down_w, d->inter, d->dtype);
}

int check_saved(vmoe_ops* o, const vmoe_gated_ffn* d, const void* saved, size_t bytes) {
  const size_t need = ffn_saved(*d).total;
  if (!saved || bytes < need)
    return ops_fail(o, VMOE_ERR_WORKSPACE, "saved needs %zu bytes (got %zu)", need,
                    saved ? bytes : static_cast<size_t>(0));
  if (reinterpret_cast<uintptr_t>(saved) & 255u)
    return ops_fail(o, VMOE_ERR_WORKSPACE, "saved must be 256-byte aligned");
  return VMOE_OK;
}
}  // namespace

int vmoe_gated_ffn_forward(vmoe_ops* o, const vmoe_gated_ffn* d, const void* x,
                           const vmoe_ffn_weights* w, const void* residual, void* y, void* saved,
                           size_t saved_bytes, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (!d) return ops_fail(o, VMOE_ERR_INVALID_ARG, "d is required");
  size_t need = 0;
  TRY(vmoe_gated_ffn_workspace_size(o, d, 0, &need, nullptr));
  if (d->tokens == 0) return VMOE_OK;
  TRY(check_ffn_call(o, d, x, w));
  if (residual) TRY(check_ld(o, "ldr", d->ldr, d->hidden));
  if (!y) return ops_fail(o, VMOE_ERR_INVALID_ARG, "y is required");
  const size_t elt = dtype_bytes(d->dtype);
  TRY(check_elt(o, "gate_b", w->gate_b, elt));
  TRY(check_elt(o, "up_b", w->up_b, elt));
  TRY(check_elt(o, "down_b", w->down_b, elt));
  TRY(check_elt(o, "residual", residual, elt));
  TRY(check_elt(o, "y", y, elt));
  if (saved) TRY(check_saved(o, d, saved, saved_bytes));
  TRY(check_workspace(o, workspace, workspace_bytes, need));
  DeviceGuard g(o->device);
  Call c{o, {static_cast<char*>(workspace), 0}, static_cast<cudaStream_t>(stream), false, d->dtype};
  FfnPtrs p{};
  p.x = x;
  p.w = *w;
  p.r = residual;
  p.y = y;
  p.saved = static_cast<char*>(saved);
  return ffn_forward(c, *d, p);
}

int vmoe_gated_ffn_backward(vmoe_ops* o, const vmoe_gated_ffn* d, const void* x,
                            const vmoe_ffn_weights* w, const void* dy, int64_t lddy, void* dx,
                            const vmoe_ffn_grads* grads, const void* saved, size_t saved_bytes,
                            void* workspace, size_t workspace_bytes, void* stream) {
  if (!o) return VMOE_ERR_INVALID_ARG;
  if (!d || !grads) return ops_fail(o, VMOE_ERR_INVALID_ARG, "d and grads are required");
  size_t need = 0;
  TRY(vmoe_gated_ffn_workspace_size(o, d, 1, &need, nullptr));
  const size_t e = dtype_bytes(d->grad_dtype), m = d->hidden * d->inter * e;
  const struct { const char* name; void* p; size_t n; } out[6] = {
      {"d gate_w", grads->gate_w, m}, {"d up_w", grads->up_w, m}, {"d down_w", grads->down_w, m},
      {"d gate_b", grads->gate_b, d->inter * e}, {"d up_b", grads->up_b, d->inter * e},
      {"d down_b", grads->down_b, d->hidden * e}};
  for (const auto& q : out) TRY(check_elt(o, q.name, q.p, e));
  TRY(check_elt(o, "dx", dx, dtype_bytes(d->dtype)));
  DeviceGuard g(o->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->tokens == 0) {
    for (const auto& q : out) {
      const cudaError_t rc = q.p ? cudaMemsetAsync(q.p, 0, q.n, s) : cudaSuccess;
      if (rc != cudaSuccess) return ops_cuda_fail(o, rc, "zero gradients");
    }
    return VMOE_OK;
  }
  TRY(check_ffn_call(o, d, x, w));
  TRY(check_dy(o, dy, lddy, d->hidden, d->dtype));
  TRY(check_saved(o, d, saved, saved_bytes));
  TRY(check_workspace(o, workspace, workspace_bytes, need));
  Call c{o, {static_cast<char*>(workspace), 0}, s, false, d->dtype};
  FfnPtrs p{};
  p.x = x;
  p.w = *w;
  p.dy = dy;
  p.lddy = lddy;
  p.dx = dx;
  p.grads = *grads;
  p.saved = const_cast<char*>(static_cast<const char*>(saved));
  return ffn_backward(c, *d, p);
}

}  // extern "C"
