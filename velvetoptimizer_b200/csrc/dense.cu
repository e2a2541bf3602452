// C-ABI of the dense training operators: the vmoe_ops context, the fused linear and the gated
// feed-forward block (include/vesper_moe.h), forward and backward.
//
// Every call first lays its workspace out (Arena), then launches; the size functions run the
// same layout without a base.  Nothing is allocated and the host never waits.
#include <atomic>

#include "dense.h"
#include "ops_host.h"

namespace {

// Status words of the contexts, zero from the module's load on (contexts past this number
// share them).
constexpr int kStatusWords = 256;
__device__ int g_ops_status[kStatusWords];

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

  int ok(cudaError_t e, const char* what) {
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
    return ok(launch_pad_copy(src.p, src.ld, src.rows, src.cols, dst, ld, s), what);
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

struct Product {
  bool a_mn = false, b_mn = false;
  int epi = kEpiLinear;
  Mat a0, a1, b0, b1;
  int64_t M = 0, N = 0;
  int64_t k0 = 0, k1 = 0;  // reduction lengths of the operand pairs
  int groups = 1;
  DenseEpi e;
  const char* what = "";
};

int product_splits(const Call& c, const Product& p) {
  const int64_t m_tiles = (p.M + 255) / 256;
  const int64_t n_tiles = p.epi == kEpiGated ? (p.N + 127) / 128 : (p.N + 255) / 256;
  return choose_splits(m_tiles * n_tiles * p.groups,
                       static_cast<int>((p.k0 + 63) / 64 + (p.k1 + 63) / 64), c.o->num_sms / 2,
                       p.M * n_tiles * 1024 * p.groups);
}

// One bf16 product on the CTA pairs, split over k where its tiles leave SMs idle.
int run_product(Call& c, const Product& p) {
  const int64_t m_tiles = (p.M + 255) / 256;
  const int64_t n_tiles = p.epi == kEpiGated ? (p.N + 127) / 128 : (p.N + 255) / 256;
  if (m_tiles * n_tiles * p.groups * 16 > 0x7fffffff)
    return ops_fail(c.o, VMOE_ERR_UNSUPPORTED_SHAPE, "%s: too many output tiles", p.what);
  DenseGemm g;
  g.M = p.M;
  g.N = p.N;
  g.m_tiles = static_cast<int>(m_tiles);
  g.n_tiles = static_cast<int>(n_tiles);
  g.groups = p.groups;
  g.kb0 = static_cast<int>((p.k0 + 63) / 64);
  g.kb1 = static_cast<int>((p.k1 + 63) / 64);
  const int kb = g.kb0 + g.kb1;
  g.ldp = n_tiles * 256;
  const int64_t part = p.M * g.ldp * 4 * p.groups;
  g.splits = product_splits(c, p);
  g.kb_per_split = (kb + g.splits - 1) / g.splits;
  g.band = n_tiles < 8 ? static_cast<int>(n_tiles) : 8;
  g.epi = p.e;
  g.status = c.o->status;
  if (g.splits > 1) g.partial = c.ws.take<float>(static_cast<size_t>(part) * g.splits);
  if (c.dry) return VMOE_OK;
  DenseMaps maps;
  char why[256];
  const uint32_t abox = p.a_mn ? 64 : 128, bbox = p.b_mn ? 64 : 128;
  auto map = [&](CUtensorMap* m, const Mat& x, uint32_t box) {
    return make_tmap_bf16(m, x.p, static_cast<uint64_t>(x.rows), static_cast<uint64_t>(x.cols),
                          static_cast<uint64_t>(x.ld), box, why, sizeof(why));
  };
  bool good = map(&maps.a0, p.a0, abox) && map(&maps.b0, p.b0, bbox);
  if (good && p.a1.p) good = map(&maps.a1, p.a1, abox); else maps.a1 = maps.a0;
  if (good && p.b1.p) good = map(&maps.b1, p.b1, bbox); else maps.b1 = maps.b0;
  if (!good) return ops_fail(c.o, VMOE_ERR_CUDA, "%s: %s", p.what, why);
  TRY(c.ok(launch_gemm_dense(p.a_mn, p.b_mn, p.epi, maps, g, c.o->num_sms, c.s), p.what));
  if (g.splits > 1) return c.ok(launch_dense_finish(kBF16, p.epi, g, c.s), p.what);
  return VMOE_OK;
}

// The fp32 counterpart: partial sums of one or two operand pairs (or a gate and an up part),
// then the epilogue.
struct SimtPart {
  const float *a, *b;
  int64_t am, ak, bn, bk, K;
};

int run_simt(Call& c, int epi, const SimtPart* parts, int n_parts, int64_t M, int64_t N,
             const DenseEpi& e, const char* what) {
  const bool gated = epi == kEpiGated;
  const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128) * (gated ? 2 : 1);
  int64_t kmax = 1;
  for (int i = 0; i < n_parts; ++i) kmax = parts[i].K > kmax ? parts[i].K : kmax;
  // about two blocks per SM, each with 64 or more k
  int64_t splits = 2 * c.o->num_sms / (tiles > 0 ? tiles : 1);
  if (splits > kmax / 64) splits = kmax / 64;
  if (splits > 64) splits = 64;
  if (splits < 1) splits = 1;
  const int64_t per = round_up((kmax + splits - 1) / splits, 16);
  splits = (kmax + per - 1) / per;
  DenseGemm g;
  g.M = M;
  g.N = N;
  g.ldp = gated ? (N + 127) / 128 * 256 : round_up(N, 8);
  g.splits = static_cast<int>(gated ? splits : splits * n_parts);
  g.epi = e;
  const int64_t stride = M * g.ldp;
  g.partial = c.ws.take<float>(static_cast<size_t>(stride) * g.splits * 4);
  if (c.dry) return VMOE_OK;
  for (int i = 0; i < n_parts; ++i) {
    SimtGemm q{};
    q.a = parts[i].a;
    q.b = parts[i].b;
    q.am = parts[i].am;
    q.ak = parts[i].ak;
    q.bn = parts[i].bn;
    q.bk = parts[i].bk;
    q.M = M;
    q.N = N;
    q.K = parts[i].K;
    q.splits = static_cast<int>(splits);
    q.k_per_split = per;
    q.partial = g.partial + (gated ? 0 : static_cast<int64_t>(i) * splits * stride);
    q.ldp = g.ldp;
    q.split_stride = stride;
    q.gated_cols = gated ? 1 + i : 0;
    TRY(c.ok(launch_dense_simt(q, c.s), what));
  }
  return c.ok(launch_dense_finish(kF32, epi, g, c.s), what);
}

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
  int64_t rb = (6 * static_cast<int64_t>(c.o->num_sms) + strips - 1) / strips;
  if (rb > (T + 31) / 32) rb = (T + 31) / 32;
  if (rb > 128) rb = 128;
  if (rb < 1) rb = 1;
  a.rows_per_block = (T + rb - 1) / rb;
  a.row_blocks = static_cast<int>((T + a.rows_per_block - 1) / a.rows_per_block);
  if (db) a.colsum = c.ws.take<float>(static_cast<size_t>(a.row_blocks) * N * 4);
  if (c.dry) return VMOE_OK;
  TRY(c.ok(launch_dense_dz(c.dtype, a, c.s), "activation gradient"));
  if (db)
    return c.ok(launch_colsum_finish(a.colsum, a.row_blocks, N, db, db_f32, c.s), "bias gradient");
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
  if (dtype == VMOE_BF16 && !o->sm100)
    return ops_fail(o, VMOE_ERR_UNSUPPORTED_SHAPE, "the bf16 path needs an sm_100 GPU");
  return VMOE_OK;
}

int check_dim(vmoe_ops* o, const char* name, int64_t v) {
  if (v < 1 || v > kMaxDim)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "%s must be in [1, 2^31) (got %lld)", name,
                    static_cast<long long>(v));
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
  if (reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype))
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
  TRY(check_ld(o, "ldx", d->ldx, d->in_features));
  return check_ld(o, "ldw", d->ldw, d->in_features);
}

int check_ffn(vmoe_ops* o, const vmoe_gated_ffn* d) {
  TRY(check_common(o, d->tokens, d->dtype, d->activation, d->grad_dtype, d->gamma));
  if (d->activation == VMOE_ACT_NONE)
    return ops_fail(o, VMOE_ERR_INVALID_ARG, "the gated block needs an activation");
  TRY(check_dim(o, "hidden", d->hidden));
  TRY(check_dim(o, "inter", d->inter));
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
  if (d.dtype == VMOE_F32) {
    const SimtPart part{static_cast<const float*>(p.x), static_cast<const float*>(p.w), d.ldx, 1,
                        d.ldw, 1, K};
    return run_simt(c, kEpiLinear, &part, 1, T, N, e, "linear");
  }
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
    g.vec_in = K % 8 == 0 && pitch16(p.x, d.ldx, 2) && pitch16(p.w, d.ldw, 2);
    return c.ok(launch_dense_small(kEpiLinear, g, c.s), "linear");
  }
  Product q;
  q.a0 = {p.x, T, K, d.ldx};
  q.b0 = {p.w, N, K, d.ldw};
  TRY(c.tma_ready(q.a0, "linear"));
  TRY(c.tma_ready(q.b0, "linear"));
  q.M = T;
  q.N = N;
  q.k0 = K;
  q.e = e;
  q.what = "linear";
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
  if (f32) {
    const auto* fz = static_cast<const float*>(dz);
    const auto* fx = static_cast<const float*>(p.x);
    const auto* fw = static_cast<const float*>(p.w);
    if (c.dry || p.dx) {
      const SimtPart part{fz, fw, lddz, 1, 1, d.ldw, N};
      TRY(run_simt(c, kEpiLinear, &part, 1, T, K, ex, "linear dx"));
    }
    if (c.dry || p.dw) {
      const SimtPart part{fz, fx, 1, lddz, 1, d.ldx, T};
      TRY(run_simt(c, kEpiLinear, &part, 1, N, K, ew, "linear dW"));
    }
    return VMOE_OK;
  }
  const Mat z{dz, T, N, lddz};
  if (c.dry || p.dx) {
    Product q;
    q.b_mn = true;
    q.a0 = z;
    q.b0 = {p.w, N, K, d.ldw};
    TRY(c.tma_ready(q.b0, "linear dx"));
    q.M = T;
    q.N = K;
    q.k0 = N;
    q.e = ex;
    q.what = "linear dx";
    TRY(run_product(c, q));
  }
  if (c.dry || p.dw) {
    Product q;
    q.a_mn = q.b_mn = true;
    q.a0 = z;
    q.b0 = {p.x, T, K, d.ldx};
    TRY(c.tma_ready(q.b0, "linear dW"));
    q.M = N;
    q.N = K;
    q.k0 = T;
    q.e = ew;
    q.what = "linear dW";
    TRY(run_product(c, q));
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

struct FfnSaved {
  int64_t ld;
  size_t part, total;
};

FfnSaved ffn_saved(const vmoe_gated_ffn& d) {
  FfnSaved s;
  s.ld = round_up(d.inter, 8);
  s.part = (static_cast<size_t>(d.tokens) * s.ld * dtype_bytes(d.dtype) + 255) &
           ~static_cast<size_t>(255);
  s.total = 3 * s.part;
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
  if (d.dtype == VMOE_F32) {
    const auto* x = static_cast<const float*>(p.x);
    const SimtPart gu[2] = {{x, static_cast<const float*>(p.w.gate_w), d.ldx, 1, H, 1, H},
                            {x, static_cast<const float*>(p.w.up_w), d.ldx, 1, H, 1, H}};
    TRY(run_simt(c, kEpiGated, gu, 2, T, I, e1, "gate|up"));
    const SimtPart dn{static_cast<const float*>(h), static_cast<const float*>(p.w.down_w), sv.ld, 1,
                      I, 1, I};
    return run_simt(c, kEpiLinear, &dn, 1, T, H, e2, "down");
  }
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
    g.vec_in = H % 8 == 0 && pitch16(p.x, d.ldx, 2) && aligned16(p.w.gate_w) && aligned16(p.w.up_w);
    TRY(c.ok(launch_dense_small(kEpiGated, g, c.s), "gate|up"));
    SmallGemm q{};
    q.x = h;
    q.w = p.w.down_w;
    q.ldx = sv.ld;
    q.ldw = I;
    q.T = T;
    q.N = H;
    q.K = I;
    q.epi = e2;
    q.vec_in = I % 8 == 0 && aligned16(p.w.down_w);
    PdlScope pdl(true);  // its launch overlaps the gate|up kernel's end
    return c.ok(launch_dense_small(kEpiLinear, q, c.s), "down");
  }
  Product g;
  g.epi = kEpiGated;
  g.a0 = {p.x, T, H, d.ldx};
  g.b0 = {p.w.gate_w, I, H, H};
  g.b1 = {p.w.up_w, I, H, H};
  TRY(c.tma_ready(g.a0, "gate|up"));
  TRY(c.tma_ready(g.b0, "gate|up"));
  TRY(c.tma_ready(g.b1, "gate|up"));
  g.M = T;
  g.N = I;
  g.k0 = H;
  g.e = e1;
  g.what = "gate|up";
  TRY(run_product(c, g));
  Product q;
  q.a0 = {h, T, I, sv.ld};
  q.b0 = {p.w.down_w, H, I, I};
  TRY(c.tma_ready(q.b0, "down"));
  q.M = T;
  q.N = H;
  q.k0 = I;
  q.e = e2;
  q.what = "down";
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
  if (f32) {
    const auto* fx = static_cast<const float*>(p.x);
    const auto* fdy = static_cast<const float*>(p.dy);
    auto F = [](const void* q) { return static_cast<const float*>(q); };
    if (need_dgu) {
      const SimtPart part{fdy, F(p.w.down_w), p.lddy, 1, 1, I, H};
      TRY(run_simt(c, kEpiGluBwd, &part, 1, T, I, e, "dh"));
    }
    if (c.dry || p.dx) {
      const SimtPart parts[2] = {{F(dg), F(p.w.gate_w), sv.ld, 1, 1, H, I},
                                 {F(du), F(p.w.up_w), sv.ld, 1, 1, H, I}};
      TRY(run_simt(c, kEpiLinear, parts, 2, T, H, plain(p.dx, H, false), "dx"));
    }
    const struct { const void* a; int64_t lda; const float* b; int64_t ldb, M, N; void* out; } wg[3] = {
        {dg, sv.ld, fx, d.ldx, I, H, gr.gate_w},
        {du, sv.ld, fx, d.ldx, I, H, gr.up_w},
        {fdy, p.lddy, F(h), sv.ld, H, I, gr.down_w}};
    for (const auto& q : wg) {
      if (!c.dry && !q.out) continue;
      const SimtPart part{F(q.a), q.b, 1, q.lda, 1, q.ldb, T};
      TRY(run_simt(c, kEpiLinear, &part, 1, q.M, q.N, plain(q.out, q.N, true), "dW"));
    }
  } else {
    if (need_dgu) {
      Product q;
      q.b_mn = true;
      q.epi = kEpiGluBwd;
      q.a0 = dy;
      q.b0 = {p.w.down_w, H, I, I};
      TRY(c.tma_ready(q.b0, "dh"));
      q.M = T;
      q.N = I;
      q.k0 = H;
      q.e = e;
      q.what = "dh";
      // the gate's and the up's bias gradients: column sums in the epilogue, where it runs once
      if ((c.dry || gr.gate_b || gr.up_b) && product_splits(c, q) == 1) {
        q.e.colsum_stride = row_blocks * I;
        q.e.colsum = colsum = c.ws.take<float>(static_cast<size_t>(2 * row_blocks * I) * 4);
        summed = true;
      }
      TRY(run_product(c, q));
    }
    const Mat mdg{dg, T, I, sv.ld}, mdu{du, T, I, sv.ld};
    if (c.dry || p.dx) {
      Product q;
      q.b_mn = true;
      q.a0 = mdg;
      q.a1 = mdu;
      q.b0 = {p.w.gate_w, I, H, H};
      q.b1 = {p.w.up_w, I, H, H};
      TRY(c.tma_ready(q.b0, "dx"));
      TRY(c.tma_ready(q.b1, "dx"));
      q.M = T;
      q.N = H;
      q.k0 = q.k1 = I;
      q.e = plain(p.dx, H, false);
      q.what = "dx";
      TRY(run_product(c, q));
    }
    if (c.dry || gr.gate_w || gr.up_w) {
      Product q;
      q.a_mn = q.b_mn = true;
      q.b0 = {p.x, T, H, d.ldx};
      TRY(c.tma_ready(q.b0, "dW gate|up"));
      q.M = I;
      q.N = H;
      q.k0 = T;
      const bool both = c.dry || (gr.gate_w && gr.up_w);
      q.groups = both ? 2 : 1;
      q.a0 = both || gr.gate_w ? mdg : mdu;
      if (both) q.a1 = mdu;
      q.e = plain(both || gr.gate_w ? gr.gate_w : gr.up_w, H, true);
      if (both) {
        q.e.out2 = gr.up_w;
        if (!vec_ok(gr.up_w, H, H, gelt)) q.e.vec = 0;
      }
      q.what = "dW gate|up";
      TRY(run_product(c, q));
      if (c.dry) {  // one gradient alone may be split into more parts
        q.groups = 1;
        TRY(run_product(c, q));
      }
    }
    if (c.dry || gr.down_w) {
      Product q;
      q.a_mn = q.b_mn = true;
      q.a0 = dy;
      q.b0 = {h, T, I, sv.ld};
      q.M = H;
      q.N = I;
      q.k0 = T;
      q.e = plain(gr.down_w, I, true);
      q.what = "dW down";
      TRY(run_product(c, q));
    }
  }
  if (summed) {
    if (c.dry) return VMOE_OK;
    if (gr.gate_b) TRY(c.ok(launch_colsum_finish(colsum, row_blocks, I, gr.gate_b, gf32, c.s), "dbg"));
    if (gr.up_b)
      TRY(c.ok(launch_colsum_finish(colsum + row_blocks * I, row_blocks, I, gr.up_b, gf32, c.s), "dbu"));
    return VMOE_OK;
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
  // a status word of the library's own: a thread whose first call falls into a stream capture
  // (a captured backward on autograd's thread) must allocate and clear nothing
  static std::atomic<unsigned> next{0};
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  void* words = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&words, g_ops_status);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) {
    fprintf(stderr, "vmoe_ops_create: %s\n", cudaGetErrorString(e));
    delete o;
    return VMOE_ERR_CUDA;
  }
  o->status = static_cast<int*>(words) + next.fetch_add(1) % kStatusWords;
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
  DeviceGuard g(o->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->tokens == 0) {  // sums over no rows
    const size_t gelt = dtype_bytes(d->grad_dtype);
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
  DeviceGuard g(o->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->tokens == 0) {
    const size_t e = dtype_bytes(d->grad_dtype), m = d->hidden * d->inter * e;
    const struct { void* p; size_t n; } out[6] = {
        {grads->gate_w, m}, {grads->up_w, m}, {grads->down_w, m}, {grads->gate_b, d->inter * e},
        {grads->up_b, d->inter * e}, {grads->down_b, d->hidden * e}};
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
