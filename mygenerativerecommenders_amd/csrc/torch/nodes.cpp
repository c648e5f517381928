// Autograd nodes and the optimizer's list call over the C-ABI entries, as torch operators
// (gr_amd::*).  A backward pass runs on one of torch's own threads: written in Python it takes
// the interpreter there and back, some 45 us a call, more than the kernels of a small batch.
// The C-ABI library is not linked: gr_torch_bind() takes the addresses of its functions, so that both
// sides use the one that is loaded (no operator, or a trace that makes the first call would hold
// them).  Arguments are checked by the Python entry points.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <cstring>
#include <vector>

#include "../../../include/gr_hstu.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entries {
  decltype(&gr_last_error) last_error;
  decltype(&gr_layer_norm_fwd) layer_norm_fwd;
  decltype(&gr_layer_norm_bwd_workspace_size) layer_norm_bwd_workspace_size;
  decltype(&gr_layer_norm_bwd) layer_norm_bwd;
  decltype(&gr_jagged_attn_fwd) jagged_attn_fwd;
  decltype(&gr_jagged_attn_bwd_workspace_size) jagged_attn_bwd_workspace_size;
  decltype(&gr_jagged_attn_bwd) jagged_attn_bwd;
  decltype(&gr_adamw8_step) adamw8_step;
};
Entries e{};

void bound() { TORCH_CHECK(e.last_error, "gr_amd: import mygenerativerecommenders_amd and call _lib.nodes() first"); }
void done(int status, const char* what) {
  TORCH_CHECK(status == 0, what, " failed (status ", status, "): ", e.last_error());
}
void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
bool is16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
Tensor floats(const Tensor& like, at::IntArrayRef size) { return at::empty(size, like.options().dtype(at::kFloat)); }
Tensor bytes(const Tensor& like, size_t n) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
Tensor plain(const Tensor& like) { return at::empty(like.sizes(), like.options()); }

// The kernels read memory: forward-mode tangents, transforms and traces would go on without the
// operator, so they raise.  Wrapped tensors show by their dispatch keys, a trace of plain ones by its mode.
bool has_tangent(const Tensor& t) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined();
}
void plain_call(const char* what, std::initializer_list<const Tensor*> inputs) {
  bound();
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped{DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::FuncTorchBatched,
                                        DispatchKey::FuncTorchGradWrapper, DispatchKey::Batched};
  for (const Tensor* t : inputs) {
    if (!t->defined()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(*t), what, ": no forward-mode derivative");
    TORCH_CHECK_NOT_IMPLEMENTED(!t->key_set().has_any(wrapped), what, ": plain tensors only, no transformed or traced ones");
  }
  TORCH_CHECK_NOT_IMPLEMENTED(!c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY), what,
                              ": cannot be traced");
}

// ---------------------------------------------------------------- layer norm
// x as (rows, D) with contiguous columns and rows that are D apart, or one: a view wherever its
// strides allow
Tensor rows_of(const Tensor& x) {
  const int64_t d = x.size(-1);
  const Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, d});
  const bool apart = x2.size(0) <= 1 || x2.stride(0) == 0 || x2.stride(0) >= d;
  return (d == 1 || x2.stride(1) == 1) && apart ? x2 : x2.contiguous();
}

int norm_types(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  const Tensor& p = weight.defined() ? weight : bias;
  return (is16(x) ? 1 : 0) + (p.defined() && is16(p) ? 2 : 0);
}

Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const Tensor x2 = rows_of(x), y = plain(x);
  const int64_t d = x.size(-1);
  if (stats) *stats = floats(x, {x2.size(0), 2});
  done(e.layer_norm_fwd(x2.data_ptr(), x2.stride(0), x2.size(0), (int)d, ptr(weight), ptr(bias),
                        norm_types(x, weight, bias), (float)eps, y.data_ptr(), d, stats ? fptr(*stats) : nullptr,
                        stream(x)),
       "gr_layer_norm_fwd");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    Tensor stats;
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    const Tensor y = norm_forward(x, w, b, eps, &stats);
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3], &dy = grads[0];
    // inputs that are not given have no number
    const bool want_x = ctx->needs_input_grad(0), want_w = weight.defined() && ctx->needs_input_grad(1),
               want_b = bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
    const int64_t d = x.size(-1);
    if (at::GradMode::is_enabled()) {  // create_graph: differentiable operations
      const Tensor xf = x.to(at::kFloat), g = dy.to(at::kFloat), c = xf - xf.mean(-1, true);
      const Tensor r = (c.square().mean(-1, true) + ctx->saved_data["eps"].toDouble()).rsqrt(), xh = c * r;
      const Tensor gw = weight.defined() ? g * weight.to(at::kFloat) : g;
      Tensor dx, dw, db;
      if (want_x) dx = (r * (gw - gw.mean(-1, true) - xh * (gw * xh).mean(-1, true))).to(x.scalar_type());
      if (want_w) dw = (g * xh).reshape({-1, d}).sum(0).to(weight.scalar_type());
      if (want_b) db = g.reshape({-1, d}).sum(0).to(bias.scalar_type());
      return {dx, dw, db, Tensor()};
    }
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = rows_of(x), g = rows_of(dy);
    const int types = norm_types(x, weight, bias);
    Tensor dx, dw, db, ws;
    if (want_x) dx = plain(x);
    if (want_w) dw = plain(weight);
    if (want_b) db = plain(bias);
    const size_t n = want_w || want_b ? e.layer_norm_bwd_workspace_size(x2.size(0), (int)d, types) : 0;
    if (n) ws = bytes(x, n);
    done(e.layer_norm_bwd(g.data_ptr(), g.stride(0), x2.data_ptr(), x2.stride(0), x2.size(0), (int)d, ptr(weight), types,
                          fptr(stats), ptr(dx), d, ptr(dw), ptr(db), ptr(ws), n, stream(x)),
         "gr_layer_norm_bwd");
    return {dx, dw, db, Tensor()};
  }
};

bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  plain_call("layer_norm", {&x, &w, &b});
  if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b))) return LayerNorm::apply(x, weight, bias, eps);
  return norm_forward(x, w, b, eps, nullptr);
}

// ---------------------------------------------------------------- jagged attention
// bfloat16 rows are read as pairs: from a start on a 4-byte boundary on
bool pairs(const Tensor& x) { return !is16(x) || (uintptr_t)x.data_ptr() % 4 == 0; }
// (not contiguous(), which returns what torch counts as contiguous wherever it starts, and with any
// stride where a size is 1)
Tensor copied(const Tensor& x) { return plain(x).copy_(x); }
// x itself where the kernels read it in place: contiguous columns, row strides below 2^22, for
// bfloat16 even strides and a start on a 4-byte boundary; else a contiguous copy.  `apart`: rows
// must not share elements either (the backward pass's queries).
Tensor columns(const Tensor& x, bool apart = false) {
  const int64_t s0 = x.stride(0), s1 = x.stride(1);
  bool ok = x.stride(2) == 1 && s0 >= (apart ? x.size(2) : 0) && s0 < (1 << 22) && pairs(x);
  if (is16(x)) ok = ok && s0 % 2 == 0 && s1 % 2 == 0;
  return ok ? x : copied(x);
}

Tensor attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, bool causal, double scale,
                         Tensor* low, Tensor* lse) {
  const c10::DeviceGuard guard(q.device());
  const int64_t rows = q.size(0), h = q.size(1), dv = v.size(2);
  const Tensor out = at::empty({rows, h, dv}, q.options());
  if (lse) *lse = floats(q, {h, rows});
  if (low && is16(q)) *low = plain(out);
  done(e.jagged_attn_fwd(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                         v.stride(0), v.stride(1), offsets.data_ptr<int64_t>(), (int)offsets.numel() - 1, rows, (int)h,
                         (int)k.size(1), (int)q.size(2), (int)dv, causal, (float)scale, is16(q), out.data_ptr(),
                         low ? ptr(*low) : nullptr, lse ? fptr(*lse) : nullptr, stream(q)),
       "gr_jagged_attn_fwd");
  return out;
}

// The history of gradients made under create_graph: its edges are what they depend on (q, k, v and
// the output's gradient), so that every way to a second derivative meets it.
struct NoSecondDerivative : torch::autograd::Node {
  explicit NoSecondDerivative(torch::autograd::edge_list&& edges) : Node(std::move(edges)) {}
  variable_list apply(variable_list&&) override { TORCH_CHECK(false, "jagged_attention: no second derivative"); }
};

struct JaggedAttention : torch::autograd::Function<JaggedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& offsets,
                        bool causal, double scale) {
    const Tensor q = columns(q0, true), k = columns(k0), v = columns(v0);
    Tensor low, lse;
    const Tensor out = attention_forward(q, k, v, offsets, causal, scale, &low, &lse);
    ctx->save_for_backward({q, k, v, offsets, out, low, lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &offsets = saved[3], &out = saved[4], &low = saved[5],
                 &lse = saved[6];
    variable_list got(6);
    {
      const at::NoGradGuard off;
      const c10::DeviceGuard guard(q.device());
      const Tensor dout = grads[0].is_contiguous() && pairs(grads[0]) ? grads[0] : copied(grads[0]);
      for (int i = 0; i < 3; ++i) got[i] = plain(saved[i]);
      const int64_t rows = q.size(0), h = q.size(1);
      const size_t n = e.jagged_attn_bwd_workspace_size(rows, (int)h);
      const Tensor ws = bytes(q, n);
      done(e.jagged_attn_bwd(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                             v.stride(0), v.stride(1), offsets.data_ptr<int64_t>(), (int)offsets.numel() - 1, rows, (int)h,
                             (int)k.size(1), (int)q.size(2), (int)v.size(2), ctx->saved_data["causal"].toBool(),
                             (float)ctx->saved_data["scale"].toDouble(), is16(q), out.data_ptr(), ptr(low), fptr(lse),
                             dout.data_ptr(), got[0].data_ptr(), got[1].data_ptr(), got[2].data_ptr(), ws.data_ptr(), n,
                             stream(q)),
           "gr_jagged_attn_bwd");
    }
    if (at::GradMode::is_enabled()) {  // create_graph
      auto edges = torch::autograd::get_current_node()->next_edges();
      edges.push_back(torch::autograd::impl::gradient_edge(grads[0]));
      const auto node = std::make_shared<NoSecondDerivative>(std::move(edges));
      for (int i = 0; i < 3; ++i) torch::autograd::set_history(got[i], node);
    }
    return got;
  }
};

Tensor jagged_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets, bool causal, double scale) {
  plain_call("jagged_attention", {&q, &k, &v, &offsets});
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v)))
    return JaggedAttention::apply(q, k, v, offsets, causal, scale);
  return attention_forward(columns(q), columns(k), columns(v), offsets, causal, scale, nullptr, nullptr);
}

// ---------------------------------------------------------------- AdamW over a list
// One step for the parameters that have a gradient; tensor i's moments start at the sum of the
// sizes before it, each rounded up to 64 elements.
void adamw8_step(at::TensorList params, const Tensor& exp_avg, const Tensor& exp_avg_scale, const Tensor& exp_avg_sq,
                 const Tensor& exp_avg_sq_scale, const Tensor& step, const Tensor& counters, double lr, double beta1,
                 double beta2, double eps, double weight_decay) {
  bound();
  const size_t n = params.size();
  std::vector<float*> p(n);
  std::vector<const float*> g(n);
  std::vector<int64_t> offs(n), numel(n);
  int64_t at = 0;
  for (size_t i = 0; i < n; ++i) {
    const Tensor &t = params[i], &grad = t.grad();
    offs[i] = at;
    at += (t.numel() + 63) / 64 * 64;
    if (!grad.defined()) continue;
    TORCH_CHECK_TYPE(!grad.is_sparse() && grad.scalar_type() == at::kFloat && grad.is_contiguous() && grad.sizes() == t.sizes() &&
                         grad.device() == t.device() && t.scalar_type() == at::kFloat && t.is_contiguous() &&
                         t.device() == step.device(),
                     "FlatAdamW: dense contiguous fp32 parameters and gradients expected");
    p[i] = t.data_ptr<float>();
    g[i] = grad.data_ptr<float>();
    numel[i] = t.numel();
  }
  TORCH_CHECK(at == exp_avg.numel(), "FlatAdamW: the group's parameters no longer have the sizes of its moments");
  const c10::DeviceGuard guard(step.device());
  done(e.adamw8_step(p.data(), g.data(), offs.data(), numel.data(), (int)n, (uint8_t*)exp_avg.data_ptr(),
                     fptr(exp_avg_scale), (uint8_t*)exp_avg_sq.data_ptr(), fptr(exp_avg_sq_scale), fptr(step),
                     (uint32_t*)counters.data_ptr(), lr, beta1, beta2, eps, weight_decay, stream(step)),
       "gr_adamw8_step");
  // a graph that saved a parameter before must not go on with what it is now
  for (size_t i = 0; i < n; ++i)
    if (p[i]) params[i].unsafeGetTensorImpl()->bump_version();
}

}  // namespace

TORCH_LIBRARY(gr_amd, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", layer_norm);
  m.def("jagged_attention(Tensor q, Tensor k, Tensor v, Tensor offsets, bool causal, float scale) -> Tensor",
        jagged_attention);
  m.def(
      "adamw8_step(Tensor[] params, Tensor exp_avg, Tensor exp_avg_scale, Tensor exp_avg_sq, Tensor exp_avg_sq_scale, "
      "Tensor step, Tensor counters, float lr, float beta1, float beta2, float eps, float weight_decay) -> ()",
      adamw8_step);
}

extern "C" __attribute__((visibility("default"))) int gr_torch_bind(const void* const* addresses, int n) {
  if (n * sizeof(void*) != sizeof(Entries)) return 1;
  std::memcpy(&e, addresses, sizeof(Entries));
  return 0;
}
