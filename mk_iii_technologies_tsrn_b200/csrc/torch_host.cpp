// torch_host.cpp -- the host side of ops.embedding, ops.gated_scan(_step) and
// ops.residual_norm: outputs and workspaces, the call of the C entry point on the
// tensors' device and its current stream, and the autograd nodes.
//
// These operators are also called on single tokens and small batches, where the
// host's time is the call's.  A node written in Python takes the interpreter lock
// in the autograd engine's thread and builds its objects there: forward and
// backward of a 64 x 640 residual step 163 us so and 96 us here, of 32 tokens'
// embedding 96 and 60 us (a node that does nothing: 41 us); a decoding step of the
// embedding 15 and 6 us.
//
// The calls below return None for arguments that are not as the kernels take them;
// ops.py then converts them or raises what is wrong with them.  The other entries
// are called with checked arguments.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>

#include "tropical_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

Tensor or_none(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
int code_of(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? TP_DTYPE_BF16 : TP_DTYPE_F32;
}
void* at_(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return static_cast<float*>(at_(t)); }
void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}
// a status of the C ABI; _lib.TropicalLibraryError in Python
struct LibraryError : std::runtime_error {
  const char* what_failed;
  int status;
  LibraryError(const char* name, int st)
      : std::runtime_error(std::string(name) + " failed: " + tp_status_string(st)),
        what_failed(name), status(st) {}
};
void check(int status, const char* what) {
  if (status != TP_OK) throw LibraryError(what, status);
}
// The device as the current one, and pointers taken for what they are: torch's.
struct On {
  c10::cuda::CUDAGuard guard;
  const int checks = tp_set_thread_pointer_checks(0);
  explicit On(const Tensor& t) : guard(t.device()) {}
  ~On() { tp_set_thread_pointer_checks(checks); }
};
Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
// the last dimension contiguous, the others at any strides
Tensor channels(const Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
Tensor empty_as(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor bytes_on(const Tensor& t, int64_t n) {
  return at::empty({n > 16 ? n : 16}, t.options().dtype(at::kByte));
}
// Tensors that a transform looks into -- tangents of forward-mode derivatives, and the
// wrappers of torch.func -- would lose what it puts there: the nodes below know reverse
// mode alone.
void no_transforms(std::initializer_list<const Tensor*> ts, const char* what) {
  constexpr c10::DispatchKeySet wrapped =
      c10::DispatchKeySet(c10::DispatchKey::FuncTorchBatched) |
      c10::DispatchKeySet(c10::DispatchKey::FuncTorchGradWrapper);
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(!t->key_set().has_any(wrapped), what,
                                " does not run under the transforms of torch.func");
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined() ||
                                    !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
                                what, " has no forward-mode derivative");
  }
}
bool any_needs_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

bool is_float(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}
bool is_index(const Tensor& t) {
  return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong;
}
// t, where there is one: on `like`'s device, of its shape and type
bool alike(const Tensor& t, const Tensor& like) {
  return !t.defined() || (t.device() == like.device() &&
                          t.scalar_type() == like.scalar_type() && t.sizes() == like.sizes());
}

// The gradients that `make` returns, which cannot be differentiated again.  They depend on
// the incoming gradients, and on inputs that require a gradient if `on_inputs`: where
// create_graph=True records a graph of the former, differentiating it raises; of constant
// incoming gradients no graph is kept, and a warning says so where one was due.
template <typename F>
variable_list once(const char* what, const variable_list& grads, bool on_inputs, F make) {
  bool record = false;
  for (const Tensor& g : grads)
    record |= at::GradMode::is_enabled() && g.defined() && g.requires_grad();
  if (at::GradMode::is_enabled() && on_inputs && !record)
    TORCH_WARN(what, " has first derivatives only: its gradients, asked for with "
               "create_graph=True, count as constants in what is differentiated next");
  at::NoGradGuard off;
  variable_list out = make();
  if (!record) return out;
  at::AutoGradMode on(true);
  for (Tensor& t : out) {
    if (!t.defined()) continue;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "this operator's backward is not differentiable", 1);
    variable_list one{t.detach().set_requires_grad(true)};
    t = (*error)(std::move(one))[0];
  }
  return out;
}

// ---------------------------------------------------------------- residual norm
struct Rows {
  Tensor t;
  int64_t ld = 0;
};
Rows rows_of(const Tensor& t, int64_t D) {
  if (!t.defined()) return {};
  if (t.is_contiguous()) return {t, D};
  Tensor r = channels(t.reshape({-1, D}));
  const int64_t ld = r.stride(0);
  return {r, ld};
}

struct ResidualIn {
  Tensor x, branch, gate, scale, weight, bias, bw, bb;
  double eps;
  int64_t norm;
  bool branch_norm;
};
int params_code(const ResidualIn& a) {
  for (const Tensor* t : {&a.scale, &a.weight, &a.bias, &a.bw, &a.bb})
    if (t->defined()) return code_of(*t);
  return TP_DTYPE_F32;
}

std::tuple<Tensor, Tensor, Tensor> residual_run(const ResidualIn& a, bool normalize,
                                                bool need_stats) {
  const On device(a.x);
  const int64_t D = a.x.size(-1), rows = a.x.numel() / D;
  const Rows x = rows_of(a.x, D), b = rows_of(a.branch, D), g = rows_of(a.gate, D);
  const Tensor w = contiguous(a.weight), bias = contiguous(a.bias), bw = contiguous(a.bw),
               bb = contiguous(a.bb), sc = contiguous(a.scale);
  Tensor y = empty_as(a.x), n, stats;
  if (normalize) n = empty_as(a.x);
  if (need_stats) stats = at::empty({rows, 4}, a.x.options().dtype(at::kFloat));
  check(tp_residual_norm_fwd(code_of(a.x), params_code(a), (int)a.norm, rows, D, at_(x.t), x.ld,
                             at_(b.t), b.ld, at_(g.t), g.ld, at_(sc),
                             sc.defined() && sc.numel() > 1, a.branch_norm, at_(bw), at_(bb),
                             at_(w), at_(bias), (float)a.eps, at_(y), at_(n), floats(stats),
                             stream_of(a.x)),
        "tp_residual_norm_fwd");
  return {y, n, stats};
}

// gradients of x, branch, gate, then float32 ones of the wanted of scale, weight, bias,
// branch weight and branch bias (views of one buffer)
variable_list residual_back(const ResidualIn& a, const Tensor& stats, const Tensor& dy_,
                            const Tensor& dn_, const std::array<bool, 5>& wanted) {
  const On device(a.x);
  const int64_t D = a.x.size(-1), rows = a.x.numel() / D;
  const Rows x = rows_of(a.x, D), b = rows_of(a.branch, D), g = rows_of(a.gate, D);
  const Tensor w = contiguous(a.weight), bias = contiguous(a.bias), bw = contiguous(a.bw),
               bb = contiguous(a.bb), sc = contiguous(a.scale), dy = contiguous(dy_),
               dn = contiguous(dn_);
  variable_list out(8);
  out[0] = empty_as(a.x);
  out[1] = empty_as(a.branch);
  if (a.gate.defined()) out[2] = empty_as(a.gate);
  const Tensor* params[5] = {&a.scale, &a.weight, &a.bias, &a.bw, &a.bb};
  int64_t total = 0, at = 0;
  for (int i = 0; i < 5; ++i)
    if (wanted[i]) total += params[i]->numel();
  if (total > 0) {
    const Tensor all = at::empty({total}, a.x.options().dtype(at::kFloat));
    for (int i = 0; i < 5; ++i) {
      if (!wanted[i]) continue;
      out[3 + i] = all.narrow(0, at, params[i]->numel());
      at += params[i]->numel();
    }
  }
  const int64_t need = tp_residual_norm_bwd_workspace_bytes(rows, D);
  const Tensor ws = bytes_on(a.x, need);
  check(tp_residual_norm_bwd(code_of(a.x), params_code(a), (int)a.norm, rows, D, at_(x.t), x.ld,
                             at_(b.t), b.ld, at_(g.t), g.ld, at_(sc),
                             sc.defined() && sc.numel() > 1, a.branch_norm, at_(bw), at_(bb),
                             at_(w), at_(bias), (float)a.eps, floats(stats), at_(dy), at_(dn),
                             at_(out[0]), at_(out[1]), at_(out[2]), floats(out[3]),
                             floats(out[6]), floats(out[7]), floats(out[4]), floats(out[5]),
                             at_(ws), need, stream_of(a.x)),
        "tp_residual_norm_bwd");
  for (int i = 0; i < 5; ++i)
    if (out[3 + i].defined() && params[i]->dim() != 1)
      out[3 + i] = out[3 + i].view(params[i]->sizes());
  return out;
}

// (y, n): the backward recomputes y from x and takes the row statistics from the forward
struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor branch, Maybe gate,
                               Maybe scale, Maybe weight, Maybe bias, Maybe bw, Maybe bb,
                               double eps, int64_t norm, bool branch_norm, bool normalize) {
    ctx->set_materialize_grads(false);
    const ResidualIn a{x, branch, or_none(gate), or_none(scale), or_none(weight), or_none(bias),
                       or_none(bw), or_none(bb), eps, norm, branch_norm};
    auto [y, n, stats] = residual_run(a, normalize, true);
    ctx->save_for_backward({x, branch, a.gate, a.scale, a.weight, a.bias, a.bw, a.bb, stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["branch_norm"] = branch_norm;
    // bit i: input i is there; bit 8 + i: it requires a gradient
    int64_t bits = 0, i = 0;
    for (const Tensor* t : {&a.x, &a.branch, &a.gate, &a.scale, &a.weight, &a.bias, &a.bw, &a.bb}) {
      if (t->defined()) bits |= (int64_t)1 << i | (int64_t)t->requires_grad() << (8 + i);
      ++i;
    }
    ctx->saved_data["inputs"] = bits;
    return normalize ? variable_list{y, n} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t bits = ctx->saved_data["inputs"].toInt();
    std::array<bool, 8> need, grad;
    for (int i = 0, place = 0; i < 8; ++i) {      // (what is not there has no place)
      need[i] = (bits >> i & 1) && ctx->needs_input_grad(place++);
      grad[i] = bits >> (8 + i) & 1;
    }
    // x, branch, gate, scale, bw and bb enter the second norm's derivative; without it the
    // product scale * sigmoid(gate) * (N(branch) * bw + bb) is left, linear in each but the
    // gate and a normalised branch
    const bool branch_norm = ctx->saved_data["branch_norm"].toBool();
    const bool in_norm = grads.size() > 1 && grads[1].defined() &&
                         (grad[0] || grad[1] || grad[2] || grad[3] || grad[6] || grad[7]);
    const bool in_product = grad[2] || (grad[1] && branch_norm) ||
                            (grad[3] && (grad[1] || grad[6] || grad[7]));
    return once("residual_norm", grads, in_norm || in_product, [&] {
      const Tensor dy = grads[0], dn = grads.size() > 1 ? grads[1] : Tensor();
      if (!dy.defined() && !dn.defined()) return variable_list(12);
      const variable_list s = ctx->get_saved_variables();
      variable_list out =
          residual_back({s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7],
                         ctx->saved_data["eps"].toDouble(), ctx->saved_data["norm"].toInt(),
                         branch_norm}, s[8], dy, dn,
                        {need[3], need[4], need[5], need[6], need[7]});
      for (int i = 0; i < 3; ++i)
        if (!need[i]) out[i] = Tensor();
      for (int i = 3; i < 8; ++i)
        if (out[i].defined() && s[i].scalar_type() != at::kFloat)
          out[i] = out[i].to(s[i].scalar_type());
      out.resize(12);
      return out;
    });
  }
};

bool residual_ok(const ResidualIn& a, bool normalize) {
  if (!a.x.is_cuda() || !is_float(a.x) || a.x.dim() == 0) return false;
  const int64_t D = a.x.size(-1);
  if (D < 1 || D > 8192 || !alike(a.branch, a.x) || !alike(a.gate, a.x)) return false;
  if (!a.branch_norm && (a.bw.defined() || a.bb.defined())) return false;
  if (!normalize && (a.weight.defined() || a.bias.defined())) return false;
  const Tensor* one = nullptr;      // the parameters' type
  for (const Tensor* t : {&a.scale, &a.weight, &a.bias, &a.bw, &a.bb}) {
    if (!t->defined()) continue;
    if (!(t->dim() == 1 && t->size(0) == D) && !(t == &a.scale && t->numel() == 1)) return false;
    if (t->device() != a.x.device()) return false;
    if (t->scalar_type() != at::kFloat && t->scalar_type() != a.x.scalar_type()) return false;
    if (one != nullptr && one->scalar_type() != t->scalar_type()) return false;
    one = t;
  }
  return true;
}

std::optional<std::tuple<Tensor, Tensor>> residual_norm(Tensor x, Tensor branch, Maybe gate, Maybe scale,
                                         Maybe weight, Maybe bias, Maybe bw, Maybe bb, double eps,
                                         int64_t norm, bool branch_norm, bool normalize) {
  const ResidualIn a{x, branch, or_none(gate), or_none(scale), or_none(weight), or_none(bias),
                     or_none(bw), or_none(bb), eps, norm, branch_norm};
  no_transforms({&a.x, &a.branch, &a.gate, &a.scale, &a.weight, &a.bias, &a.bw, &a.bb},
                "residual_norm");
  if (!residual_ok(a, normalize)) return std::nullopt;
  if (any_needs_grad({&a.x, &a.branch, &a.gate, &a.scale, &a.weight, &a.bias, &a.bw, &a.bb})) {
    variable_list out = ResidualNorm::apply(x, branch, gate, scale, weight, bias, bw, bb, eps,
                                            norm, branch_norm, normalize);
    return std::make_tuple(out[0], normalize ? out[1] : Tensor());
  }
  auto [y, n, stats] = residual_run(a, normalize, false);
  return std::make_tuple(y, n);
}

std::tuple<Tensor, Tensor, Tensor> residual_norm_fwd(
    Tensor x, Tensor branch, Maybe gate, Maybe scale, Maybe weight, Maybe bias, Maybe bw, Maybe bb,
    double eps, int64_t norm, bool branch_norm, bool normalize, bool need_stats) {
  at::NoGradGuard off;
  return residual_run({x, branch, or_none(gate), or_none(scale), or_none(weight), or_none(bias),
                       or_none(bw), or_none(bb), eps, norm, branch_norm}, normalize, need_stats);
}

variable_list residual_norm_bwd(Tensor stats, Maybe dy, Maybe dn, Tensor x, Tensor branch,
                                Maybe gate, Maybe scale, Maybe weight, Maybe bias, Maybe bw,
                                Maybe bb, double eps, int64_t norm, bool branch_norm) {
  at::NoGradGuard off;
  const ResidualIn a{x, branch, or_none(gate), or_none(scale), or_none(weight), or_none(bias),
                     or_none(bw), or_none(bb), eps, norm, branch_norm};
  return residual_back(a, stats, or_none(dy), or_none(dn),
                       {a.scale.defined(), a.weight.defined(), a.bias.defined(), a.bw.defined(),
                        a.bb.defined()});
}

// ---------------------------------------------------------------- gated scan
Tensor scan_workspace(const Tensor& x, int64_t& need) {
  need = tp_gated_scan_workspace_bytes(x.size(0), x.size(1), x.size(2));
  return need > 0 ? bytes_on(x, need) : Tensor();
}

std::tuple<Tensor, Tensor, Tensor> scan_run(const Tensor& gate_, const Tensor& x_,
                                            const Tensor& h0_, const Tensor& lengths, int64_t form,
                                            bool need_states, bool need_last) {
  const On device(x_);
  const int64_t B = x_.size(0), T = x_.size(1), C = x_.size(2);
  const Tensor gate = channels(gate_), x = channels(x_), h0 = contiguous(h0_);
  const auto f32 = x_.options().dtype(at::kFloat);
  Tensor h = empty_as(x_), last, states;
  if (need_last) last = at::empty({B, C}, f32);
  if (need_states) states = at::empty({B, (T + 63) / 64, C}, f32);
  int64_t need;
  const Tensor ws = scan_workspace(x_, need);
  check(tp_gated_scan_fwd(code_of(x), (int)form, B, T, C, at_(gate), gate.stride(0),
                          gate.stride(1), at_(x), x.stride(0), x.stride(1), floats(h0),
                          (const int32_t*)at_(lengths), at_(h), floats(last), floats(states),
                          at_(ws), need, stream_of(x)),
        "tp_gated_scan_fwd");
  return {h, last, states};
}

std::tuple<Tensor, Tensor, Tensor> scan_back(const Tensor& states, const Tensor& dh_,
                                             const Tensor& dlast_, const Tensor& gate_,
                                             const Tensor& x_, const Tensor& lengths, int64_t form,
                                             bool need_dh0) {
  const On device(x_);
  const int64_t B = x_.size(0), T = x_.size(1), C = x_.size(2);
  const Tensor gate = channels(gate_), x = channels(x_), dh = contiguous(dh_),
               dlast = contiguous(dlast_);
  Tensor dgate = empty_as(x_), dx = empty_as(x_), dh0;
  if (need_dh0) dh0 = at::empty({B, C}, x_.options().dtype(at::kFloat));
  int64_t need;
  const Tensor ws = scan_workspace(x_, need);
  check(tp_gated_scan_bwd(code_of(x), (int)form, B, T, C, at_(gate), gate.stride(0),
                          gate.stride(1), at_(x), x.stride(0), x.stride(1),
                          (const int32_t*)at_(lengths), floats(states), at_(dh), floats(dlast),
                          at_(dgate), at_(dx), floats(dh0), at_(ws), need, stream_of(x)),
        "tp_gated_scan_bwd");
  return {dgate, dx, dh0};
}

// (h, h_last): keeps gate, x and one fp32 state per 64 steps
struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, Tensor gate, Tensor x, Maybe h0,
                               Maybe lengths, int64_t form) {
    ctx->set_materialize_grads(false);
    const Tensor ends = or_none(lengths);
    auto [h, last, states] = scan_run(gate, x, or_none(h0), ends, form, true, true);
    ctx->save_for_backward({gate, x, ends, states});
    ctx->saved_data["form"] = form;
    ctx->saved_data["h0"] = h0.has_value();
    ctx->saved_data["gate"] = gate.requires_grad();
    return {h, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    // (linear in x and h0: only the gate is in the others' derivatives)
    return once("gated_scan", grads, ctx->saved_data["gate"].toBool(), [&] {
      if (!grads[0].defined() && !grads[1].defined()) return variable_list(5);
      const variable_list s = ctx->get_saved_variables();
      const bool need_h0 = ctx->saved_data["h0"].toBool() && ctx->needs_input_grad(2);
      auto [dgate, dx, dh0] = scan_back(s[3], grads[0], grads[1], s[0], s[1], s[2],
                                        ctx->saved_data["form"].toInt(), need_h0);
      return variable_list{ctx->needs_input_grad(0) ? dgate : Tensor(),
                           ctx->needs_input_grad(1) ? dx : Tensor(), dh0, Tensor(), Tensor()};
    });
  }
};

std::optional<std::tuple<Tensor, Tensor>> gated_scan(Tensor gate, Tensor x, Maybe h0,
                                                     Maybe lengths, int64_t form,
                                                     bool need_last) {
  const Tensor first = or_none(h0), ends = or_none(lengths);
  no_transforms({&gate, &x, &first, &ends}, "gated_scan");
  if (!x.is_cuda() || !is_float(x) || x.dim() != 3 || !alike(gate, x)) return std::nullopt;
  if (first.defined() &&
      (first.device() != x.device() || first.scalar_type() != at::kFloat || first.dim() != 2 ||
       first.size(0) != x.size(0) || first.size(1) != x.size(2)))
    return std::nullopt;
  if (ends.defined() &&
      (ends.device() != x.device() || ends.scalar_type() != at::kInt || ends.dim() != 1 ||
       ends.size(0) != x.size(0) || !ends.is_contiguous()))
    return std::nullopt;
  if (any_needs_grad({&gate, &x, &first})) {
    variable_list out = GatedScan::apply(gate, x, h0, lengths, form);
    return std::make_tuple(out[0], out[1]);
  }
  auto [h, last, states] = scan_run(gate, x, first, ends, form, false, need_last);
  return std::make_tuple(h, last);
}

std::tuple<Tensor, Tensor, Tensor> gated_scan_fwd(Tensor gate, Tensor x, Maybe h0, Maybe lengths,
                                                  int64_t form, bool need_states, bool need_last) {
  at::NoGradGuard off;
  return scan_run(gate, x, or_none(h0), or_none(lengths), form, need_states, need_last);
}

std::tuple<Tensor, Tensor, Tensor> gated_scan_bwd(Tensor states, Maybe dh, Maybe dlast,
                                                  Tensor gate, Tensor x, Maybe lengths,
                                                  int64_t form, bool need_dh0) {
  at::NoGradGuard off;
  return scan_back(states, or_none(dh), or_none(dlast), gate, x, or_none(lengths), form, need_dh0);
}

Maybe gated_scan_step(Tensor gate_, Tensor x_, Tensor state, int64_t form) {
  no_transforms({&gate_, &x_, &state}, "gated_scan_step");
  if (!x_.is_cuda() || !is_float(x_) || x_.dim() != 2 || !alike(gate_, x_)) return std::nullopt;
  if (state.device() != x_.device() || state.scalar_type() != at::kFloat ||
      state.sizes() != x_.sizes() || (x_.size(1) > 1 && state.stride(1) != 1) ||
      (x_.size(0) > 1 && state.stride(0) < x_.size(1)))
    return std::nullopt;
  if (any_needs_grad({&gate_, &x_, &state})) return std::nullopt;
  at::NoGradGuard off;
  const On device(x_);
  const Tensor gate = channels(gate_), x = channels(x_);
  Tensor h = empty_as(x_);
  check(tp_gated_scan_step(code_of(x), (int)form, x.size(0), x.size(1), at_(gate), gate.stride(0),
                           at_(x), x.stride(0), floats(state), state.stride(0), at_(h),
                           stream_of(x)),
        "tp_gated_scan_step");
  state.unsafeGetTensorImpl()->bump_version();
  return h;
}

// ---------------------------------------------------------------- embedding
int bits_of(const Tensor& t) { return t.scalar_type() == at::kInt ? 32 : 64; }

Tensor embed_run(const Tensor& ids_, const Tensor& weight, const Tensor& pos, const Tensor& at,
                 double scale) {
  const On device(weight);
  const Tensor ids = ids_.contiguous(), w = channels(weight),
               p = pos.defined() ? channels(pos) : pos;
  const int64_t D = w.size(1), T = ids.dim() ? ids.size(-1) : 1;
  c10::DimVector shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(D);
  Tensor out = at::empty(shape, w.options());
  check(tp_embedding_fwd(code_of(w), bits_of(ids), ids.numel(), T, D, at_(ids), at_(w), w.size(0),
                         w.stride(0), (float)scale, at_(p), p.defined() ? p.size(0) : 0,
                         p.defined() ? p.stride(0) : 0, at_(at), at_(out), stream_of(w)),
        "tp_embedding_fwd");
  return out;
}

// other: the tokens' indices in the other table, of other_rows rows, where there is one
Tensor embed_back(const Tensor& ids_, const Tensor& dout_, int64_t rows, double scale,
                  int64_t padding, const Tensor& other_, int64_t other_rows) {
  const On device(dout_);
  const Tensor ids = ids_.contiguous(), dout = dout_.contiguous(), other = contiguous(other_);
  const int64_t N = ids.numel(), D = dout.size(-1);
  const int64_t need = tp_embedding_bwd_workspace_bytes(N, rows, D);
  TORCH_CHECK_VALUE(need >= 0, "embedding_bwd takes fewer than 2^31 tokens and rows, got ", N,
                    " and ", rows);
  Tensor dw = at::empty({rows, D}, dout.options());
  const Tensor ws = bytes_on(dout, need);
  check(tp_embedding_bwd_both(code_of(dout), bits_of(ids), N, D, at_(ids), at_(dout), rows,
                              (float)scale, padding, at_(other), other_rows, at_(dw), at_(ws),
                              ws.numel(), stream_of(dout)),
        "tp_embedding_bwd_both");
  return dw;
}

// ids: the tokens' rows in a table of id_rows, where there is one
Tensor embed_pos_back(const Tensor& dout_, int64_t rows, const Tensor& ids_, int64_t id_rows) {
  const On device(dout_);
  const Tensor dout = dout_.contiguous(), ids = contiguous(ids_);
  const int64_t D = dout.size(-1), T = dout.dim() > 1 ? dout.size(-2) : 1;
  Tensor dp = at::empty({rows, D}, dout.options());
  check(tp_embedding_pos_bwd_both(code_of(dout), D ? dout.numel() / D : 0, T, D, at_(dout), rows,
                                  at_(ids), ids.defined() ? bits_of(ids) : 64, id_rows, at_(dp),
                                  stream_of(dout)),
        "tp_embedding_pos_bwd_both");
  return dp;
}

// the gradients of the tables are dense; a token outside either table adds to neither
struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, Tensor weight, Maybe pos_weight, Tensor ids,
                        Maybe positions, double scale, int64_t padding) {
    const Tensor pos = or_none(pos_weight), at = or_none(positions);
    ctx->save_for_backward({ids, at});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["pos"] = pos.defined();
    ctx->saved_data["positions"] = pos.defined() ? pos.size(0) : 0;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed_run(ids, weight, pos, at, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return once("embedding", grads, false, [&] {
      const variable_list s = ctx->get_saved_variables();
      const Tensor dout = grads[0].contiguous();
      variable_list out(6);
      const int64_t rows = ctx->saved_data["rows"].toInt(),
                    positions = ctx->saved_data["positions"].toInt();
      if (ctx->needs_input_grad(0))
        out[0] = embed_back(s[0], dout, rows, ctx->saved_data["scale"].toDouble(),
                            ctx->saved_data["padding"].toInt(), s[1], positions);
      if (ctx->saved_data["pos"].toBool() && ctx->needs_input_grad(1))
        out[1] = s[1].defined() ? embed_back(s[1], dout, positions, 1.0, -1, s[0], rows)
                                : embed_pos_back(dout, positions, s[0], rows);
      return out;
    });
  }
};

Maybe embedding(Tensor ids, Tensor weight, Maybe pos_weight, Maybe positions, double scale,
                int64_t padding) {
  const Tensor pos = or_none(pos_weight), at = or_none(positions);
  no_transforms({&ids, &weight, &pos, &at}, "embedding");
  if (!weight.is_cuda() || !is_float(weight) || weight.dim() != 2 || !is_index(ids) ||
      ids.device() != weight.device())
    return std::nullopt;
  if (pos.defined() &&
      (pos.device() != weight.device() || pos.scalar_type() != weight.scalar_type() ||
       pos.dim() != 2 || pos.size(1) != weight.size(1)))
    return std::nullopt;
  if (at.defined() && (!pos.defined() || !alike(at, ids) || !at.is_contiguous()))
    return std::nullopt;
  if (pos.defined() && !at.defined() && (ids.dim() ? ids.size(-1) : 1) > pos.size(0))
    return std::nullopt;
  if (any_needs_grad({&weight, &pos}))
    return Embedding::apply(weight, pos_weight, ids, positions, scale, padding);
  return embed_run(ids, weight, pos, at, scale);
}

Tensor embedding_fwd(Tensor ids, Tensor weight, Maybe pos_weight, Maybe positions, double scale) {
  at::NoGradGuard off;
  return embed_run(ids, weight, or_none(pos_weight), or_none(positions), scale);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const LibraryError& e) {
      const py::object cls = py::module_::import("mk_iii_technologies_tsrn_b200._lib")
                                 .attr("TropicalLibraryError");
      PyErr_SetObject(cls.ptr(), cls(e.what_failed, e.status, tp_status_string(e.status)).ptr());
    }
  });
  m.def("residual_norm", &residual_norm);
  m.def("residual_norm_fwd", &residual_norm_fwd);
  m.def("residual_norm_bwd", &residual_norm_bwd);
  m.def("gated_scan", &gated_scan);
  m.def("gated_scan_fwd", &gated_scan_fwd);
  m.def("gated_scan_bwd", &gated_scan_bwd);
  m.def("gated_scan_step", &gated_scan_step);
  m.def("embedding", &embedding);
  m.def("embedding_fwd", &embedding_fwd);
  m.def("embedding_bwd", [](Tensor ids, Tensor dout, int64_t rows, double scale, int64_t padding) {
    at::NoGradGuard off;
    return embed_back(ids, dout, rows, scale, padding, Tensor(), 0);
  });
  m.def("embedding_pos_bwd", [](Tensor dout, int64_t rows) {
    at::NoGradGuard off;
    return embed_pos_back(dout, rows, Tensor(), 0);
  });
}
