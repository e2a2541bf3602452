// Host path of velvetoptimizer_b200.linear, .gated_ffn, .grad_norm and .clip_grad_norm_ for
// eager calls: argument checks, output and workspace tensors, the C-ABI call and the autograd
// node, in C++.  The same work
// done in Python and ctypes takes 30 us a forward and 100 us a backward, several times what
// the kernels of a one-token call take.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>
#include <unordered_set>

#include "vesper_moe.h"

namespace {

using at::Tensor;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// A status of the C ABI other than VMOE_OK; becomes _lib.VmoeError in Python.
struct AbiError : std::runtime_error {
  int code;
  AbiError(int c, const std::string& what) : std::runtime_error(what), code(c) {}
};

// The calling thread's contexts, one per device (calls on one context must not overlap).
struct Contexts {
  std::array<vmoe_ops*, 64> of{};
  ~Contexts() {
    for (vmoe_ops* o : of)
      if (o) vmoe_ops_destroy(o);
  }
};

vmoe_ops* context(const Tensor& x) {
  static thread_local Contexts contexts;
  const int d = x.get_device();
  TORCH_CHECK(d >= 0 && d < 64, "device index ", d, " is not supported");
  if (!contexts.of[d]) {
    const int rc = vmoe_ops_create(d, &contexts.of[d]);
    if (rc != VMOE_OK)
      throw AbiError(rc, std::string("vmoe_ops_create failed: ") + vmoe_status_string(rc));
  }
  return contexts.of[d];
}

void check(vmoe_ops* o, int rc, const char* what) {
  if (rc == VMOE_OK) return;
  throw AbiError(rc, std::string(what) + " failed: " + vmoe_status_string(rc) + " (" +
                         vmoe_ops_last_error(o) + ")");
}

int32_t dtype_of(at::ScalarType t) { return t == at::kFloat ? VMOE_F32 : VMOE_BF16; }
bool supported(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

bool misaligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) != 0; }

// A view whose elements are negated only when they are read (an imaginary part of a conjugate)
// as a tensor of its own
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// The matrix as the kernels read it, and its row pitch: itself where its rows are contiguous
// (and 16-byte aligned where the pitch is), else a contiguous copy.
Tensor rows(const Tensor& view, int64_t& ld) {
  const Tensor t = plain(view);
  const int64_t r = t.size(0), c = t.size(1), s0 = t.stride(0), s1 = t.stride(1);
  if ((s1 == 1 || c == 1) && (r <= 1 || s0 >= c)) {
    ld = r > 1 ? s0 : c;
    if (t.scalar_type() == at::kFloat || ld % 8 != 0 || !misaligned(t)) return t;
    ld = c;
    return t.clone(at::MemoryFormat::Contiguous);
  }
  ld = c;
  return t.contiguous();
}

// The same for an output's gradient, whose pitch is its row length or a multiple of 8.
Tensor grad_rows(const Tensor& t, int64_t& ld) {
  Tensor m = rows(t, ld);
  if (ld != t.size(1) && ld % 8 != 0 && t.scalar_type() == at::kBFloat16) {
    m = m.contiguous();
    ld = t.size(1);
  }
  return m;
}

Tensor packed(const Tensor& t) {
  Tensor m = plain(t).contiguous();
  return misaligned(m) ? m.clone(at::MemoryFormat::Contiguous) : m;
}

// Forward-mode derivatives are not computed: a tangent raises rather than being left out.
template <typename... T>
void no_tangents(const char* name, const T&... tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  auto dual = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Tensor>)
      return t.defined() && t._fw_grad(/*level=*/0).defined();
    else
      return t && t->defined() && t->_fw_grad(/*level=*/0).defined();
  };
  TORCH_CHECK_NOT_IMPLEMENTED(!(dual(tensors) || ...), name,
                              " has no forward-mode derivative: an argument carries a tangent");
}

const void* ptr(const OptTensor& t) { return t && t->defined() ? t->data_ptr() : nullptr; }

// An uninitialised CUDA tensor, past the dispatcher
Tensor fresh(at::IntArrayRef shape, const at::TensorOptions& like) {
  return at::detail::empty_cuda(shape, like);
}

struct Workspace {
  Tensor t;
  void* p = nullptr;
  size_t n = 0;
  Workspace(size_t bytes, const Tensor& like) {
    if (bytes == 0) return;
    t = fresh({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
    p = t.data_ptr();
    n = bytes;
  }
};

void* stream_of(const Tensor& x) {
  return c10::cuda::getCurrentCUDAStream(x.get_device()).stream();
}

OptTensor contiguous(const OptTensor& b) {
  return b && b->defined() ? OptTensor(plain(*b).contiguous()) : std::nullopt;
}

// ---- linear -----------------------------------------------------------------------------
// (y [T, N], z [T, N] or empty) for x [T, K]
std::tuple<Tensor, Tensor> linear_forward(const Tensor& x_in, const Tensor& w_in,
                                          const OptTensor& bias, const OptTensor& residual,
                                          int64_t act, double gamma, bool keep) {
  no_tangents("linear", x_in, w_in, bias, residual);
  vmoe_ops* o = context(x_in);
  vmoe_linear d{};
  d.tokens = x_in.size(0);
  d.in_features = x_in.size(1);
  d.out_features = w_in.size(0);
  const Tensor x = rows(x_in, d.ldx), w = rows(w_in, d.ldw);
  Tensor r;
  d.ldr = d.out_features;
  if (residual && residual->defined()) r = rows(*residual, d.ldr);
  const OptTensor b = contiguous(bias);
  d.dtype = d.grad_dtype = dtype_of(x.scalar_type());
  d.activation = static_cast<int32_t>(act);
  d.gamma = static_cast<float>(gamma);
  Tensor y = fresh({d.tokens, d.out_features}, x.options());
  Tensor z;
  if (keep) z = fresh({d.tokens, d.out_features}, x.options());
  size_t need = 0;
  check(o, vmoe_linear_workspace_size(o, &d, 0, &need), "vmoe_linear_workspace_size");
  const Workspace ws(need, x);
  check(o,
        vmoe_linear_forward(o, &d, x.data_ptr(), w.data_ptr(), ptr(b),
                            r.defined() ? r.data_ptr() : nullptr, y.data_ptr(),
                            keep ? z.data_ptr() : nullptr, ws.p, ws.n, stream_of(x)),
        "vmoe_linear_forward");
  return {y, z};
}

// (dx, dW, db), empty where not wanted
std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& x_in, const Tensor& w_in,
                                                   const Tensor& z, const Tensor& dy_in,
                                                   int64_t act, double gamma,
                                                   const std::vector<bool>& want, bool grad_f32) {
  no_tangents("linear's backward", x_in, w_in, z, dy_in);
  vmoe_ops* o = context(x_in);
  vmoe_linear d{};
  d.tokens = x_in.size(0);
  d.in_features = x_in.size(1);
  d.out_features = w_in.size(0);
  int64_t lddy = 0;
  const Tensor x = rows(x_in, d.ldx), w = rows(w_in, d.ldw), dy = grad_rows(dy_in, lddy);
  d.ldr = d.out_features;
  d.dtype = dtype_of(x.scalar_type());
  d.activation = static_cast<int32_t>(act);
  d.gamma = static_cast<float>(gamma);
  d.grad_dtype = grad_f32 ? VMOE_F32 : d.dtype;
  const auto xo = x.options();
  const auto go = grad_f32 ? xo.dtype(at::kFloat) : xo;
  Tensor dx = want[0] ? fresh({d.tokens, d.in_features}, xo) : fresh({0}, xo);
  Tensor dw = want[1] ? fresh({d.out_features, d.in_features}, go) : fresh({0}, go);
  Tensor db = want[2] ? fresh({d.out_features}, go) : fresh({0}, go);
  size_t need = 0;
  check(o, vmoe_linear_workspace_size(o, &d, 1, &need), "vmoe_linear_workspace_size");
  const Workspace ws(need, x);
  check(o,
        vmoe_linear_backward(o, &d, x.data_ptr(), w.data_ptr(),
                             z.defined() && z.numel() ? z.data_ptr() : nullptr, dy.data_ptr(), lddy,
                             want[0] ? dx.data_ptr() : nullptr, want[1] ? dw.data_ptr() : nullptr,
                             want[2] ? db.data_ptr() : nullptr, ws.p, ws.n, stream_of(x)),
        "vmoe_linear_backward");
  return {dx, dw, db};
}

// ---- gated feed-forward block -------------------------------------------------------------
vmoe_gated_ffn ffn_desc(const Tensor& x, int64_t inter, int64_t act, double gamma) {
  vmoe_gated_ffn d{};
  d.tokens = x.size(0);
  d.hidden = x.size(1);
  d.inter = inter;
  d.ldr = d.hidden;
  d.dtype = d.grad_dtype = dtype_of(x.scalar_type());
  d.activation = static_cast<int32_t>(act);
  d.gamma = static_cast<float>(gamma);
  return d;
}

// (y [T, H], what the backward reads, as bytes, or empty) for x [T, H]
std::tuple<Tensor, Tensor> gated_ffn_forward(const Tensor& x_in, const Tensor& gate_w,
                                             const Tensor& up_w, const Tensor& down_w,
                                             const OptTensor& gate_b, const OptTensor& up_b,
                                             const OptTensor& down_b, const OptTensor& residual,
                                             int64_t act, double gamma, bool keep) {
  no_tangents("gated_ffn", x_in, gate_w, up_w, down_w, gate_b, up_b, down_b, residual);
  vmoe_ops* o = context(x_in);
  vmoe_gated_ffn d = ffn_desc(x_in, gate_w.size(0), act, gamma);
  const Tensor x = rows(x_in, d.ldx);
  Tensor r;
  if (residual && residual->defined()) r = rows(*residual, d.ldr);
  const Tensor wg = packed(gate_w), wu = packed(up_w), wd = packed(down_w);
  const OptTensor bg = contiguous(gate_b), bu = contiguous(up_b), bd = contiguous(down_b);
  const vmoe_ffn_weights w{wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), ptr(bg), ptr(bu), ptr(bd)};
  size_t need = 0, saved_bytes = 0;
  check(o, vmoe_gated_ffn_workspace_size(o, &d, 0, &need, &saved_bytes),
        "vmoe_gated_ffn_workspace_size");
  Tensor y = fresh({d.tokens, d.hidden}, x.options());
  Tensor saved;
  if (keep) saved = fresh({static_cast<int64_t>(saved_bytes)}, x.options().dtype(at::kByte));
  const Workspace ws(need, x);
  const bool kept = keep && saved.numel() > 0;
  check(o,
        vmoe_gated_ffn_forward(o, &d, x.data_ptr(), &w, r.defined() ? r.data_ptr() : nullptr,
                               y.data_ptr(), kept ? saved.data_ptr() : nullptr,
                               kept ? saved_bytes : 0, ws.p, ws.n, stream_of(x)),
        "vmoe_gated_ffn_forward");
  return {y, saved};
}

// (dx, dWg, dWu, dWd, dbg, dbu, dbd), empty where not wanted
std::array<Tensor, 7> gated_ffn_backward_array(const Tensor& x_in, const Tensor& gate_w,
                                               const Tensor& up_w, const Tensor& down_w,
                                               const Tensor& saved, const Tensor& dy_in,
                                               int64_t act, double gamma,
                                               const std::vector<bool>& want, bool grad_f32) {
  no_tangents("gated_ffn's backward", x_in, gate_w, up_w, down_w, saved, dy_in);
  vmoe_ops* o = context(x_in);
  const int64_t I = gate_w.size(0), H = x_in.size(1);
  vmoe_gated_ffn d = ffn_desc(x_in, I, act, gamma);
  if (grad_f32) d.grad_dtype = VMOE_F32;
  int64_t lddy = 0;
  const Tensor x = rows(x_in, d.ldx), dy = grad_rows(dy_in, lddy);
  const Tensor wg = packed(gate_w), wu = packed(up_w), wd = packed(down_w);
  const vmoe_ffn_weights w{wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), nullptr, nullptr, nullptr};
  const std::array<std::vector<int64_t>, 7> shapes{
      {{d.tokens, H}, {I, H}, {I, H}, {H, I}, {I}, {I}, {H}}};
  std::array<Tensor, 7> out;
  std::array<void*, 7> p{};
  const auto xo = x.options();
  const auto go = grad_f32 ? xo.dtype(at::kFloat) : xo;
  for (size_t i = 0; i < 7; ++i) {
    out[i] = want[i] ? fresh(shapes[i], i ? go : xo) : fresh({0}, i ? go : xo);
    p[i] = want[i] ? out[i].data_ptr() : nullptr;
  }
  const vmoe_ffn_grads g{p[1], p[2], p[3], p[4], p[5], p[6]};
  size_t need = 0;
  check(o, vmoe_gated_ffn_workspace_size(o, &d, 1, &need, nullptr), "vmoe_gated_ffn_workspace_size");
  const Workspace ws(need, x);
  check(o,
        vmoe_gated_ffn_backward(o, &d, x.data_ptr(), &w, dy.data_ptr(), lddy, p[0], &g,
                                saved.data_ptr(), static_cast<size_t>(saved.numel()), ws.p, ws.n,
                                stream_of(x)),
        "vmoe_gated_ffn_backward");
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> gated_ffn_backward(
    const Tensor& x, const Tensor& gate_w, const Tensor& up_w, const Tensor& down_w,
    const Tensor& saved, const Tensor& dy, int64_t act, double gamma,
    const std::vector<bool>& want, bool grad_f32) {
  auto r = gated_ffn_backward_array(x, gate_w, up_w, down_w, saved, dy, act, gamma, want, grad_f32);
  return {r[0], r[1], r[2], r[3], r[4], r[5], r[6]};
}

// ---- autograd -----------------------------------------------------------------------------
using torch::autograd::SavedVariable;

OptTensor cast(const OptTensor& p, const Tensor& x) {
  return p && p->defined() ? OptTensor(p->to(x.scalar_type())) : std::nullopt;
}

// The gradients have no gradient: differentiating through them raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list fake;
  std::vector<size_t> at;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (!grads[i].defined()) continue;
    fake.push_back(grads[i].detach().set_requires_grad(true));
    at.push_back(i);
  }
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "the gradients of linear and gated_ffn cannot be differentiated", static_cast<int64_t>(fake.size()));
  variable_list out = (*node)(std::move(fake));
  for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = out[i];
  return grads;
}

// A gradient is accumulated on the stream that its leaf's accumulator was made on, and an eager
// graph that is still alive keeps the accumulators of its leaves.  Where those belong to the
// default stream, a captured backward would make that stream wait for the capture: not allowed,
// and the end of the process.  So the backward of a capture looks at the accumulators it leads to
// first, and raises.
void check_capture(const torch::autograd::Node* self) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto* exec = torch::autograd::get_current_graph_task_exec_info();
  std::unordered_set<const torch::autograd::Node*> seen{self};
  std::vector<const torch::autograd::Node*> todo{self};
  while (!todo.empty()) {
    const auto* node = todo.back();
    todo.pop_back();
    for (const auto& edge : node->next_edges()) {
      auto* next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (exec && !exec->empty()) {
        const auto it = exec->find(next);
        if (it == exec->end() || !it->second.should_execute()) continue;
      }
      if (dynamic_cast<torch::autograd::AccumulateGrad*>(next)) {
        const auto s = next->stream();
        TORCH_CHECK(!s || s->id() != 0,
                    "the backward of linear or gated_ffn is being captured while an earlier graph of "
                    "the same leaves, made on the default stream, is alive: delete the outputs or "
                    "losses that hold it before the capture, or make it on a side stream");
      }
      todo.push_back(next);
    }
  }
}

Tensor to_param(const Tensor& g, at::ScalarType type) {
  return g.scalar_type() == type ? g : g.to(type);
}

// A node with its inputs' edges in the order of `inputs` (absent ones have an empty edge).
template <typename N>
std::shared_ptr<N> make_node(std::initializer_list<const OptTensor*> inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  edges.reserve(inputs.size());
  for (const OptTensor* t : inputs)
    edges.push_back(*t && (*t)->defined() ? torch::autograd::impl::gradient_edge(**t)
                                          : torch::autograd::Edge());
  node->set_next_edges(std::move(edges));
  return node;
}

struct LinearBackward : public torch::autograd::Node {
  SavedVariable x, w, z;
  int64_t act = 0;
  double gamma = 0;
  at::ScalarType w_type = at::kFloat, b_type = at::kFloat;

  std::string name() const override { return "VesperLinearBackward"; }
  void release_variables() override {
    x.reset_data();
    w.reset_data();
    z.reset_data();
  }
  variable_list apply(variable_list&& dys) override {
    variable_list out(4);
    if (!dys[0].defined()) return out;
    check_capture(this);
    const bool nx = task_should_compute_output(0), nw = task_should_compute_output(1),
               nb = task_should_compute_output(2), nr = task_should_compute_output(3);
    if (nx || nw || nb) {
      const Tensor xs = x.unpack(), ws = w.unpack(), zs = z.unpack();
      at::AutoGradMode no_grad(false);
      auto [dx, dw, db] = linear_backward(xs, ws, zs, dys[0], act, gamma, {nx, nw, nb},
                                          w_type == at::kFloat || b_type == at::kFloat);
      if (nx) out[0] = dx;
      if (nw) out[1] = to_param(dw, w_type);
      if (nb) out[2] = to_param(db, b_type);
    }
    out = once(std::move(out));
    if (nr) out[3] = dys[0];
    return out;
  }
};

struct GatedFfnBackward : public torch::autograd::Node {
  SavedVariable x, wg, wu, wd, saved;
  int64_t act = 0;
  double gamma = 0;
  std::array<at::ScalarType, 6> types{};
  bool f32 = false;

  std::string name() const override { return "VesperGatedFfnBackward"; }
  void release_variables() override {
    for (SavedVariable* v : {&x, &wg, &wu, &wd, &saved}) v->reset_data();
  }
  variable_list apply(variable_list&& dys) override {
    variable_list out(8);
    if (!dys[0].defined()) return out;
    check_capture(this);
    std::vector<bool> want(7);
    bool any = false;
    for (size_t i = 0; i < 7; ++i) any |= (want[i] = task_should_compute_output(i));
    const bool nr = task_should_compute_output(7);
    if (any) {
      const Tensor xs = x.unpack(), g = wg.unpack(), u = wu.unpack(), d = wd.unpack(),
                   s = saved.unpack();
      at::AutoGradMode no_grad(false);
      auto got = gated_ffn_backward_array(xs, g, u, d, s, dys[0], act, gamma, want, f32);
      for (size_t i = 0; i < 7; ++i)
        if (want[i]) out[i] = i ? to_param(got[i], types[i - 1]) : got[i];
    }
    out = once(std::move(out));
    if (nr) out[7] = dys[0];
    return out;
  }
};

bool wants(const OptTensor& t) { return t && t->defined() && t->requires_grad(); }

Tensor linear_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                       const OptTensor& residual, int64_t act, double gamma) {
  const OptTensor ox(x), ow(weight);
  auto node = make_node<LinearBackward>({&ox, &ow, &bias, &residual});
  Tensor y;
  {
    at::AutoGradMode no_grad(false);
    const Tensor w = weight.to(x.scalar_type());
    const bool keep = act != VMOE_ACT_NONE && (wants(ox) || wants(ow) || wants(bias));
    auto [out, z] = linear_forward(x, w, cast(bias, x), residual, act, gamma, keep);
    y = out;
    node->x = SavedVariable(x, false);
    node->w = SavedVariable(w, false);
    node->z = SavedVariable(z, false);
  }
  node->act = act;
  node->gamma = gamma;
  node->w_type = weight.scalar_type();
  node->b_type = bias && bias->defined() ? bias->scalar_type() : weight.scalar_type();
  torch::autograd::set_history(y, node);
  return y;
}

Tensor gated_ffn_autograd(const Tensor& x, const Tensor& gate_w, const Tensor& up_w,
                          const Tensor& down_w, const OptTensor& gate_b, const OptTensor& up_b,
                          const OptTensor& down_b, const OptTensor& residual, int64_t act,
                          double gamma) {
  const OptTensor ox(x), og(gate_w), ou(up_w), od(down_w);
  auto node = make_node<GatedFfnBackward>({&ox, &og, &ou, &od, &gate_b, &up_b, &down_b, &residual});
  bool keep = wants(ox);
  size_t i = 0;
  for (const OptTensor* p : {&og, &ou, &od, &gate_b, &up_b, &down_b}) {
    const bool has = *p && (*p)->defined();
    keep = keep || wants(*p);
    node->f32 = node->f32 || (has && (*p)->scalar_type() == at::kFloat);
    node->types[i++] = has ? (*p)->scalar_type() : x.scalar_type();
  }
  Tensor y;
  {
    at::AutoGradMode no_grad(false);
    const auto t = x.scalar_type();
    const Tensor wg = gate_w.to(t), wu = up_w.to(t), wd = down_w.to(t);
    auto [out, saved] = gated_ffn_forward(x, wg, wu, wd, cast(gate_b, x), cast(up_b, x),
                                          cast(down_b, x), residual, act, gamma, keep);
    y = out;
    node->x = SavedVariable(x, false);
    node->wg = SavedVariable(wg, false);
    node->wu = SavedVariable(wu, false);
    node->wd = SavedVariable(wd, false);
    node->saved = SavedVariable(saved, false);
  }
  node->act = act;
  node->gamma = gamma;
  torch::autograd::set_history(y, node);
  return y;
}

// ---- the operators ------------------------------------------------------------------------
void check_x(const char* name, const Tensor& x) {
  TORCH_CHECK_TYPE(supported(x.scalar_type()), name, " supports float32 and bfloat16 inputs, not ",
                   x.scalar_type());
  TORCH_CHECK(x.is_cuda(), name, " runs on CUDA tensors only (there is no CPU path)");
  TORCH_CHECK_VALUE(x.dim() >= 1, name, ": x must have a feature dimension");
}

void check_param(const char* name, const char* label, const OptTensor& p, at::IntArrayRef shape,
                 const Tensor& x) {
  if (!p || !p->defined()) return;
  TORCH_CHECK_VALUE(p->sizes() == shape, name, ": ", label, " must have shape ", shape, ", not ",
                    p->sizes());
  TORCH_CHECK_VALUE(p->device() == x.device(), name, ": ", label, " is on ", p->device(),
                    ", x on ", x.device());
  TORCH_CHECK_TYPE(supported(p->scalar_type()), name, ": ", label,
                   " must be float32 or bfloat16, not ", p->scalar_type());
}

OptTensor check_residual(const char* name, const OptTensor& r, at::IntArrayRef shape,
                         const Tensor& x) {
  if (!r || !r->defined()) return std::nullopt;
  TORCH_CHECK_VALUE(r->sizes() == shape, name, ": residual must have shape ", shape, ", not ",
                    r->sizes());
  TORCH_CHECK_TYPE(r->device() == x.device() && r->scalar_type() == x.scalar_type(), name,
                   ": residual must be ", x.scalar_type(), " on ", x.device(), ", as x is");
  return r;
}

// [rows, features] of a tensor with any leading dimensions
Tensor flat(const Tensor& t) {
  return t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)});
}

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias,
              const OptTensor& residual, int64_t act, double gamma) {
  check_x("linear", x);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.numel() > 0,
                    "linear: weight must be [N, ", x.size(-1), "] with N and K at least 1, not ",
                    weight.sizes());
  const int64_t N = weight.size(0);
  check_param("linear", "weight", weight, weight.sizes(), x);
  check_param("linear", "bias", bias, {N}, x);
  auto shape = x.sizes().vec();
  shape.back() = N;
  OptTensor r = check_residual("linear", residual, shape, x);
  if (r) r = flat(*r);
  const Tensor x2 = flat(x);
  Tensor y;
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias) || wants(residual))) {
    y = linear_autograd(x2, weight, bias, r, act, gamma);
  } else {
    at::NoGradGuard no_grad;
    y = std::get<0>(linear_forward(x2, weight.to(x.scalar_type()), cast(bias, x), r, act, gamma, false));
  }
  return x.dim() == 2 ? y : y.reshape(shape);
}

Tensor gated_ffn(const Tensor& x, const Tensor& gate_w, const Tensor& up_w, const Tensor& down_w,
                 const OptTensor& gate_b, const OptTensor& up_b, const OptTensor& down_b,
                 const OptTensor& residual, int64_t act, double gamma) {
  const char* name = "gated_ffn";
  check_x(name, x);
  const int64_t H = x.size(-1);
  TORCH_CHECK_VALUE(gate_w.dim() == 2 && gate_w.size(1) == H && gate_w.numel() > 0, name,
                    ": gate_weight must be [I, ", H, "] with I and H at least 1, not ",
                    gate_w.sizes());
  const int64_t I = gate_w.size(0);
  check_param(name, "gate_weight", gate_w, {I, H}, x);
  check_param(name, "up_weight", up_w, {I, H}, x);
  check_param(name, "down_weight", down_w, {H, I}, x);
  check_param(name, "gate_bias", gate_b, {I}, x);
  check_param(name, "up_bias", up_b, {I}, x);
  check_param(name, "down_bias", down_b, {H}, x);
  OptTensor r = check_residual(name, residual, x.sizes(), x);
  if (r) r = flat(*r);
  const Tensor x2 = flat(x);
  Tensor y;
  if (at::GradMode::is_enabled() &&
      (wants(x) || wants(gate_w) || wants(up_w) || wants(down_w) || wants(gate_b) || wants(up_b) ||
       wants(down_b) || wants(residual))) {
    y = gated_ffn_autograd(x2, gate_w, up_w, down_w, gate_b, up_b, down_b, r, act, gamma);
  } else {
    at::NoGradGuard no_grad;
    const auto t = x.scalar_type();
    y = std::get<0>(gated_ffn_forward(x2, gate_w.to(t), up_w.to(t), down_w.to(t), cast(gate_b, x),
                                      cast(up_b, x), cast(down_b, x), r, act, gamma, false));
  }
  return x.dim() == 2 ? y : y.reshape(x.sizes());
}

// ---- gradient norm and clipping -----------------------------------------------------------
struct GradTable {
  std::vector<void*> ptrs;
  std::vector<int64_t> counts, bytes;
  std::vector<int32_t> dtypes;

  void add(const Tensor& t) {
    if (t.numel() == 0) return;
    ptrs.push_back(t.data_ptr());
    counts.push_back(t.numel());
    dtypes.push_back(dtype_of(t.scalar_type()));
    bytes.push_back(t.numel() * static_cast<int64_t>(t.element_size()));
  }

  // A tensor given twice is taken once; any other overlap raises (two warps would scale the
  // same element).
  void check_overlap() {
    const size_t n = ptrs.size();
    std::vector<size_t> order(n);
    for (size_t i = 0; i < n; ++i) order[i] = i;
    auto at = [&](size_t i) { return reinterpret_cast<uintptr_t>(ptrs[i]); };
    std::sort(order.begin(), order.end(),
              [&](size_t a, size_t b) { return at(a) != at(b) ? at(a) < at(b) : a < b; });
    std::vector<char> drop;
    size_t last = 0;
    uintptr_t end = 0;
    for (size_t k = 0; k < n; ++k) {
      const size_t i = order[k];
      if (k > 0 && at(i) < end) {
        TORCH_CHECK_VALUE(
            at(i) == at(last) && bytes[i] == bytes[last] && dtypes[i] == dtypes[last],
            "gradients overlap in memory");
        drop.resize(n);
        drop[i] = 1;
        continue;
      }
      end = at(i) + static_cast<uintptr_t>(bytes[i]);
      last = i;
    }
    if (drop.empty()) return;
    size_t m = 0;
    for (size_t i = 0; i < n; ++i) {
      if (drop[i]) continue;
      ptrs[m] = ptrs[i];
      counts[m] = counts[i];
      dtypes[m++] = dtypes[i];
    }
    ptrs.resize(m);
    counts.resize(m);
    dtypes.resize(m);
  }
};

// The bytes that a strided tensor covers: from `at` on, every sum of multiples of the strides,
// outermost first; the last dimension is the run of consecutive bytes.
struct Footprint {
  uintptr_t at = 0, end = 0;
  int64_t numel = 0;
  std::vector<std::pair<int64_t, int64_t>> dims;  // size, stride

  explicit Footprint(const Tensor& t)
      : at(reinterpret_cast<uintptr_t>(t.data_ptr())), numel(t.numel()) {
    const int64_t elt = static_cast<int64_t>(t.element_size());
    std::vector<std::pair<int64_t, int64_t>> d{{elt, 1}};
    for (int64_t k = 0; k < t.dim(); ++k)
      if (t.size(k) > 1 && t.stride(k) > 0) d.emplace_back(t.size(k), t.stride(k) * elt);
    std::sort(d.begin(), d.end(), [](const auto& a, const auto& b) { return a.second > b.second; });
    end = at + 1;
    for (const auto& q : d) {
      end += static_cast<uintptr_t>((q.first - 1) * q.second);
      if (!dims.empty() && dims.back().second == q.first * q.second)
        dims.back() = {dims.back().first * q.first, q.second};  // one run
      else
        dims.push_back(q);
    }
  }
  bool operator==(const Footprint& o) const { return at == o.at && numel == o.numel && dims == o.dims; }
};

// Whether two footprints share a byte: is there a sum of a's multiples minus b's that equals the
// distance of their starts?  Searched from the largest stride down; what the smaller strides can
// reach leaves one or two multiples to try for each stride of nested layouts.  A search that gets
// long (strides that interleave) counts as shared.
bool share_memory(const Footprint& a, const Footprint& b) {
  if (a.end <= b.at || b.end <= a.at) return false;
  struct Term {
    int64_t stride, lo, hi;  // multiples; then what the terms after this one reach
    int64_t reach_lo = 0, reach_hi = 0;
  };
  std::vector<Term> terms;
  for (const auto& q : a.dims) terms.push_back({q.second, 0, q.first - 1});
  for (const auto& q : b.dims) {
    auto same = std::find_if(terms.begin(), terms.end(), [&](const Term& t) { return t.stride == q.second; });
    if (same != terms.end()) same->lo -= q.first - 1;
    else terms.push_back({q.second, -(q.first - 1), 0});
  }
  std::sort(terms.begin(), terms.end(), [](const Term& x, const Term& y) { return x.stride > y.stride; });
  for (size_t i = terms.size() - 1; i-- > 0;) {
    const Term& n = terms[i + 1];
    terms[i].reach_lo = n.reach_lo + n.lo * n.stride;
    terms[i].reach_hi = n.reach_hi + n.hi * n.stride;
  }
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  int64_t steps = 0;
  auto search = [&](auto&& self, size_t i, int64_t d) -> bool {
    if (i == terms.size()) return d == 0;
    if (++steps > 100000) return true;
    const Term& t = terms[i];
    const int64_t from = std::max(t.lo, -floor_div(t.reach_hi - d, t.stride));
    const int64_t to = std::min(t.hi, floor_div(d - t.reach_lo, t.stride));
    for (int64_t m = from; m <= to; ++m)
      if (self(self, i + 1, d - m * t.stride)) return true;
    return false;
  };
  return search(search, 0, static_cast<int64_t>(b.at - a.at));
}

// Of the tensors that are not dense, those whose memory no other one has; raises where one
// shares some of its memory with another, dense ones among them.
std::vector<Tensor> distinct(const std::vector<Tensor>& gapped, const std::vector<Tensor>& dense) {
  struct Entry {
    Footprint f;
    size_t gapped;  // index, or -1
  };
  constexpr size_t kDense = static_cast<size_t>(-1);
  std::vector<Entry> all;
  all.reserve(gapped.size() + dense.size());
  for (size_t i = 0; i < gapped.size(); ++i) all.push_back({Footprint(gapped[i]), i});
  for (const Tensor& t : dense) all.push_back({Footprint(t), kDense});
  std::stable_sort(all.begin(), all.end(), [](const Entry& x, const Entry& y) { return x.f.at < y.f.at; });
  std::vector<char> keep(gapped.size(), 1);
  std::vector<const Entry*> open;  // begun before and not ended
  for (const Entry& e : all) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Entry* o) { return o->f.end <= e.f.at; }),
               open.end());
    bool again = false;
    for (const Entry* o : open) {
      if (o->gapped == kDense && e.gapped == kDense) continue;  // check_overlap's
      if (o->gapped != kDense && e.gapped != kDense && o->f == e.f &&
          gapped[o->gapped].scalar_type() == gapped[e.gapped].scalar_type()) {
        again = true;
        break;
      }
      TORCH_CHECK_VALUE(!share_memory(o->f, e.f), "gradients overlap in memory");
    }
    if (again) keep[e.gapped] = 0;
    else open.push_back(&e);
  }
  std::vector<Tensor> out;
  for (size_t i = 0; i < gapped.size(); ++i)
    if (keep[i]) out.push_back(gapped[i]);
  return out;
}

// The norm of the tensors of a list or tuple, or of their .grad where present (none: nothing),
// scaled in place when max_norm >= 0.
std::optional<Tensor> grad_norm(const py::object& items, bool use_grad, double max_norm, int norm) {
  TORCH_CHECK_TYPE(PyList_Check(items.ptr()) || PyTuple_Check(items.ptr()), "expected a list or tuple");
  // a tracer would take the norm for a constant and miss the scaling
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) &&
                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
              "grad_norm and clip_grad_norm_ cannot be traced");
  PyObject** p = PySequence_Fast_ITEMS(items.ptr());
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(items.ptr());
  GradTable table;
  std::vector<Tensor> gapped;  // not dense
  Tensor like;
  at::NoGradGuard no_grad;
  auto each = [&](auto&& f) {
    for (Py_ssize_t i = 0; i < n; ++i) {
      TORCH_CHECK_TYPE(THPVariable_Check(p[i]), "expected tensors");
      const Tensor& own = THPVariable_Unpack(p[i]);
      const Tensor& t = use_grad ? own.grad() : own;
      if (t.defined()) f(t);
    }
  };
  each([&](const Tensor& t) {
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, "sparse gradients are not supported");
    TORCH_CHECK_TYPE(supported(t.scalar_type()), "gradients must be float32 or bfloat16");
    no_tangents("grad_norm", t);
    TORCH_CHECK(t.is_cuda(), "gradients must be CUDA tensors (there is no CPU path)");
    if (!like.defined()) like = t;
    TORCH_CHECK_VALUE(t.device() == like.device(), "gradients must lie on one device");
    if (t.is_non_overlapping_and_dense()) {
      table.add(t);
      if (max_norm >= 0 && !t.is_inference()) torch::autograd::impl::bump_version(t);
      return;
    }
    if (t.numel() == 0) return;
    for (int64_t k = 0; max_norm >= 0 && k < t.dim(); ++k)
      TORCH_CHECK_VALUE(t.stride(k) != 0 || t.size(k) <= 1,
                        "a gradient whose elements share memory cannot be scaled in place");
    gapped.push_back(t);
  });
  if (!like.defined()) return std::nullopt;
  table.check_overlap();
  std::vector<std::pair<Tensor, Tensor>> copies;  // of those that are not dense: a dense copy each
  if (!gapped.empty()) {
    std::vector<Tensor> dense;
    each([&](const Tensor& t) {
      if (t.is_non_overlapping_and_dense() && t.numel() > 0) dense.push_back(t);
    });
    for (const Tensor& t : distinct(gapped, dense)) {
      copies.emplace_back(t, t.contiguous());
      table.add(copies.back().second);
    }
  }
  vmoe_ops* o = context(like);
  const int count = static_cast<int>(table.ptrs.size());
  size_t need = 0;
  check(o, vmoe_grad_norm_workspace_size(o, count, &need), "vmoe_grad_norm_workspace_size");
  const Workspace ws(need, like);
  Tensor out = fresh({}, like.options().dtype(at::kFloat));
  check(o,
        vmoe_grad_norm(o, table.ptrs.data(), table.counts.data(), table.dtypes.data(), count, norm,
                       static_cast<float>(max_norm), out.mutable_data_ptr<float>(), ws.p, ws.n,
                       stream_of(like)),
        "vmoe_grad_norm");
  if (max_norm >= 0)
    for (auto& c : copies) c.first.copy_(c.second);
  return out;
}

// Whether a call on these tensors may go past the dispatcher: none has a __torch_dispatch__ of its
// own, and no dispatch mode (make_fx, fake tensors, counters), pre-dispatch tracing or
// torch.jit.trace would miss the call.
template <typename... T>
bool eager(const T&... tensors) {
  auto own = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Tensor>)
      return t.key_set().has(c10::DispatchKey::Python);
    else
      return t && t->defined() && t->key_set().has(c10::DispatchKey::Python);
  };
  return !(own(tensors) || ...) && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) &&
         !torch::jit::tracer::isTracing();
}

}  // namespace

PYBIND11_MODULE(_dense_ops, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const AbiError& e) {
      py::object type = py::module_::import("velvetoptimizer_b200._lib").attr("VmoeError");
      py::object value = type(e.code, e.what());
      PyErr_SetObject(type.ptr(), value.ptr());
    }
  });
  using Release = py::call_guard<py::gil_scoped_release>;
  // None where the call is not the eager path's (see `eager`)
  m.def("linear", [](const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r, int64_t act,
                     double gamma) {
    return eager(x, w, b, r) ? OptTensor(linear(x, w, b, r, act, gamma)) : std::nullopt;
  }, Release());
  m.def("gated_ffn", [](const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                        const OptTensor& bg, const OptTensor& bu, const OptTensor& bd, const OptTensor& r,
                        int64_t act, double gamma) {
    return eager(x, wg, wu, wd, bg, bu, bd, r)
               ? OptTensor(gated_ffn(x, wg, wu, wd, bg, bu, bd, r, act, gamma))
               : std::nullopt;
  }, Release());
  m.def("eager", [](const Tensor& x, const Tensor& w) { return eager(x, w); });
  // the tracers' ops return a tensor in every place
  m.def("linear_forward", [](const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r,
                             int64_t act, double gamma, bool keep) {
    auto [y, z] = linear_forward(x, w, b, r, act, gamma, keep);
    return std::make_tuple(y, keep ? z : fresh({0}, x.options()));
  }, Release());
  m.def("linear_backward", &linear_backward, Release());
  m.def("gated_ffn_forward", [](const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                                const OptTensor& bg, const OptTensor& bu, const OptTensor& bd,
                                const OptTensor& r, int64_t act, double gamma, bool keep) {
    auto [y, saved] = gated_ffn_forward(x, wg, wu, wd, bg, bu, bd, r, act, gamma, keep);
    return std::make_tuple(y, keep ? saved : fresh({0}, x.options().dtype(at::kByte)));
  }, Release());
  m.def("gated_ffn_backward", &gated_ffn_backward, Release());
  m.def("grad_norm", &grad_norm);
  m.def("share_memory", [](const Tensor& a, const Tensor& b) {
    return share_memory(Footprint(a), Footprint(b));
  });
  m.def("device_status", [](const Tensor& x) {
    int32_t code = 0;
    vmoe_ops* o = context(x);
    check(o, vmoe_ops_device_status(o, &code, stream_of(x)), "vmoe_ops_device_status");
    return code;
  });
}
