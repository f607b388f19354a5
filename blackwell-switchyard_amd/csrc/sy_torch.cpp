// The autograd operators as native torch functions over the C ABI: what the Python
// functions of hip_op.py, table_op.py and stats_op.py do on their ordinary inputs,
// without the interpreter. A small forward + backward is bound by the host: the
// Python bodies and their ctypes calls take 16 + 19 us, and twice that when autograd
// alternates between the caller's thread and its own. Forward + backward, N=4 T=256
// D=512 fp32 (14 us on the device): 122-133 us, here 40-59; N=9 T=4096 D=2048 bf16
// 135, here 88 (the device's time); a forward of 8 tokens 15.0, here 6.3.
//
// Every function here returns nullopt (None) instead of a result for a call that is
// not ordinary -- anything its checks refuse, no tokens, transforms, modes, tracing,
// forward-mode tangents -- and the caller then takes the Python path, which raises or
// handles it. Nothing is cached between calls.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <utility>
#include <vector>

#include "../../include/switchyard.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SY_F32;
    case at::kHalf: return SY_F16;
    case at::kBFloat16: return SY_BF16;
    default: return -1;
  }
}

void check(int64_t rc, const char* what) {
  if (rc != 0)
    throw std::runtime_error(std::string(what) + " failed (" + std::to_string(rc) +
                             "): " + sy_strerror((int)rc));
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// A dense GPU tensor of a supported dtype that nothing intercepts: no tensor subclass
// with its own dispatch, no transform's wrapper, no lazy negation or conjugation, no
// forward-mode tangent.
bool plain(const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped{DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                        DispatchKey::Batched, DispatchKey::Functionalize};
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && code_of(t) >= 0 &&
         !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.key_set().has_any(wrapped) && !t.is_neg() &&
         !t.is_conj() && !t._fw_grad(0).defined();
}

// No function transform (vmap, grad, jvp), torch dispatch or function mode, nor tracer
// is active on this thread.
bool ordinary() {
  return !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled() &&
         !torch::jit::tracer::isTracing();
}

Tensor dense(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

// A dense copy in `like`'s dtype where the gradient is not already that.
Tensor grad_like(const Tensor& g, const Tensor& like) {
  return dense(g.scalar_type() == like.scalar_type() ? g : g.to(like.scalar_type()));
}

bool needs_grad(const Tensor& a, const Tensor& b) {
  return at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad());
}

bool tracked(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

at::TensorOptions f32_on(const Tensor& t) { return t.options().dtype(at::kFloat).requires_grad(false); }

// Sizes of stacked sources; `ok` false where the Python path has to see the call.
struct Stacked {
  int64_t n = 0, b = 0, t = 0, d = 0, tok = 0;
  bool ok = false;
};
Stacked sizes_of(const Tensor& v, const Tensor& w, int64_t w_dim) {
  Stacked s;
  if (!plain(v) || !plain(w) || v.dim() != 4 || w.dim() != w_dim || w.device() != v.device()) return s;
  s.n = v.size(0), s.b = v.size(1), s.t = v.size(2), s.d = v.size(3), s.tok = s.b * s.t;
  s.ok = w.size(w_dim - 1) == s.d && s.n > 0 && s.tok > 0 && s.d > 0 && ordinary();
  return s;
}

Tensor bwd_workspace(const Tensor& like, int64_t n, int64_t tok, int64_t d, int vt, int wt) {
  const int64_t bytes = sy_bwd_workspace_bytes(n, tok, d, vt, wt);
  if (bytes < 0) check(bytes, "sy_bwd_workspace_bytes");
  return at::empty({std::max<int64_t>(1, (bytes + 3) / 4)}, f32_on(like));
}

// ------------------------------------------------------------------ operator

Tensor operator_forward(const Tensor& v, const Tensor& w, const Stacked& s, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(v.device());
  Tensor out = at::empty({s.b, s.t, s.d}, v.options().requires_grad(false));
  if (stats != nullptr) *stats = at::empty({2, s.n, s.tok}, f32_on(v));
  check(sy_fwd(v.data_ptr(), w.data_ptr(), out.data_ptr(),
               stats != nullptr ? stats->data_ptr<float>() : nullptr, s.n, s.tok, s.d, s.tok * s.d,
               code_of(v), code_of(w), (float)eps, stream_of(v)),
        "sy_fwd");
  return out;
}

// (dv, dw) of the operator from dense v and w and the forward's statistics.
variable_list operator_backward(const Tensor& v, const Tensor& w, const Tensor& stats, const Tensor& grad,
                                double eps) {
  const c10::DeviceGuard guard(v.device());
  const int64_t n = v.size(0), d = v.size(3), tok = v.size(1) * v.size(2);
  const int vt = code_of(v), wt = code_of(w);
  const Tensor g = grad_like(grad, v);
  Tensor dv = at::empty(v.sizes(), v.options().requires_grad(false));
  Tensor dw = at::empty({d}, w.options().requires_grad(false));
  const Tensor ws = bwd_workspace(v, n, tok, d, vt, wt);
  check(sy_bwd(v.data_ptr(), w.data_ptr(), g.data_ptr(), stats.data_ptr<float>(), dv.data_ptr(),
               dw.data_ptr(), ws.data_ptr(), ws.numel() * 4, n, tok, d, tok * d, vt, wt, (float)eps,
               stream_of(v)),
        "sy_bwd");
  return {dv, dw};
}

struct BlockAttnResHIP : torch::autograd::Function<BlockAttnResHIP> {
  static Tensor forward(AutogradContext* ctx, const Tensor& v_in, const Tensor& w_in, double eps) {
    const Tensor v = dense(v_in), w = dense(w_in);
    Stacked s{v.size(0), v.size(1), v.size(2), v.size(3), v.size(1) * v.size(2), true};
    Tensor stats;
    Tensor out = operator_forward(v, w, s, eps, &stats);
    ctx->save_for_backward({v, w, stats});
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto r = operator_backward(saved[0], saved[1], saved[2], grads[0], ctx->saved_data["eps"].toDouble());
    return {r[0], r[1], Tensor()};
  }
};

std::optional<Tensor> block_attn_res(const Tensor& v, const Tensor& w, double eps) {
  const Stacked s = sizes_of(v, w, 1);
  if (!s.ok) return std::nullopt;
  if (needs_grad(v, w)) return BlockAttnResHIP::apply(v, w, eps);
  return operator_forward(dense(v), dense(w), s, eps, nullptr);
}

// ------------------------------------------- the module: a query and its gain

Tensor gain_forward(const Tensor& v, const Tensor& w, const Tensor& g, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(v.device());
  const int64_t n = v.size(0), b = v.size(1), t = v.size(2), d = v.size(3), tok = b * t;
  Tensor out = at::empty({b, t, d}, v.options().requires_grad(false));
  if (stats != nullptr) *stats = at::empty({2, n, tok}, f32_on(v));
  check(sy_fwd_gain(v.data_ptr(), w.data_ptr(), g.data_ptr(), out.data_ptr(),
                    stats != nullptr ? stats->data_ptr<float>() : nullptr, n, tok, d, tok * d, code_of(v),
                    code_of(w), (float)eps, stream_of(v)),
        "sy_fwd_gain");
  return out;
}

struct BlockAttnResGain : torch::autograd::Function<BlockAttnResGain> {
  static Tensor forward(AutogradContext* ctx, const Tensor& v_in, const Tensor& w_in, const Tensor& g_in,
                        double eps) {
    const Tensor v = dense(v_in), w = dense(w_in), g = dense(g_in);
    Tensor stats;
    Tensor out = gain_forward(v, w, g, eps, &stats);
    ctx->save_for_backward({v, w, g, stats});
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &v = saved[0], &w = saved[1];
    const c10::DeviceGuard guard(v.device());
    if (at::GradMode::is_enabled()) {
      // Recorded: the product's own gradients are torch operations, through which the
      // factors can be differentiated again (the operator's carry no graph).
      const Tensor wf = w.to(at::kFloat), gf = saved[2].to(at::kFloat);
      const auto r = operator_backward(v, (wf * gf).detach(), saved[3], grads[0],
                                       ctx->saved_data["eps"].toDouble());
      return {r[0], (r[1] * gf).to(w.scalar_type()), (r[1] * wf).to(w.scalar_type()), Tensor()};
    }
    const int64_t n = v.size(0), d = v.size(3), tok = v.size(1) * v.size(2);
    const int vt = code_of(v), wt = code_of(w);
    const Tensor go = grad_like(grads[0], v);
    Tensor dv = at::empty(v.sizes(), v.options().requires_grad(false));
    Tensor dw = at::empty({d}, w.options().requires_grad(false));
    Tensor dg = at::empty({d}, w.options().requires_grad(false));
    const Tensor ws = bwd_workspace(v, n, tok, d, vt, wt);
    check(sy_bwd_gain(v.data_ptr(), w.data_ptr(), saved[2].data_ptr(), go.data_ptr(),
                      saved[3].data_ptr<float>(), dv.data_ptr(), dw.data_ptr(), dg.data_ptr(), ws.data_ptr(),
                      ws.numel() * 4, n, tok, d, tok * d, vt, wt, (float)ctx->saved_data["eps"].toDouble(),
                      stream_of(v)),
          "sy_bwd_gain");
    return {dv, dw, dg, Tensor()};
  }
};

std::optional<Tensor> block_attn_res_gain(const Tensor& v, const Tensor& w, const Tensor& g, double eps) {
  if (!sizes_of(v, w, 1).ok || !plain(g) || g.sizes() != w.sizes() || g.scalar_type() != w.scalar_type() ||
      g.device() != w.device())
    return std::nullopt;
  if (needs_grad(v, w) || (at::GradMode::is_enabled() && g.requires_grad()))
    return BlockAttnResGain::apply(v, w, g, eps);
  return gain_forward(dense(v), dense(w), dense(g), eps, nullptr);
}

// --------------------------------------------------- sources as separate tensors

struct BlockAttnResSources : torch::autograd::Function<BlockAttnResSources> {
  static Tensor forward(AutogradContext* ctx, const Tensor& w_in, double eps, at::TensorList sources);
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

Tensor sources_forward(const Tensor& w, const variable_list& rows, double eps, Tensor* stats) {
  const Tensor& first = rows[0];
  const c10::DeviceGuard guard(first.device());
  const int64_t n = (int64_t)rows.size(), d = first.size(2), tok = first.size(0) * first.size(1);
  Tensor out = at::empty(first.sizes(), first.options().requires_grad(false));
  if (stats != nullptr) *stats = at::empty({2, n, tok}, f32_on(first));
  const void* p[SY_MAX_TABLE_ROWS];
  for (int64_t k = 0; k < n; ++k) p[k] = rows[k].data_ptr();
  check(sy_fwd_table(p, w.data_ptr(), out.data_ptr(), stats != nullptr ? stats->data_ptr<float>() : nullptr,
                     n, tok, d, code_of(first), code_of(w), (float)eps, stream_of(first)),
        "sy_fwd_table");
  return out;
}

Tensor BlockAttnResSources::forward(AutogradContext* ctx, const Tensor& w_in, double eps,
                                    at::TensorList sources) {
  const Tensor w = dense(w_in);
  variable_list rows;
  rows.reserve(sources.size() + 2);
  for (const Tensor& s : sources) rows.push_back(dense(s));
  Tensor stats;
  Tensor out = sources_forward(w, rows, eps, &stats);
  rows.push_back(w);
  rows.push_back(stats);
  ctx->save_for_backward(std::move(rows));
  ctx->saved_data["eps"] = eps;
  return out;
}

variable_list BlockAttnResSources::backward(AutogradContext* ctx, variable_list grads) {
  const auto saved = ctx->get_saved_variables();
  const int64_t n = (int64_t)saved.size() - 2;
  const Tensor &first = saved[0], &w = saved[n], &stats = saved[n + 1];
  const c10::DeviceGuard guard(first.device());
  const int64_t d = first.size(2), tok = first.size(0) * first.size(1);
  const int vt = code_of(first), wt = code_of(w);
  const Tensor g = grad_like(grads[0], first);
  // One allocation; each source's gradient is a slice of it.
  const variable_list dvs =
      at::empty({n, first.size(0), first.size(1), d}, first.options().requires_grad(false)).unbind(0);
  Tensor dw = at::empty({d}, w.options().requires_grad(false));
  const Tensor ws = bwd_workspace(first, n, tok, d, vt, wt);
  const void* p[SY_MAX_TABLE_ROWS];
  void* q[SY_MAX_TABLE_ROWS];
  for (int64_t k = 0; k < n; ++k) {
    p[k] = saved[k].data_ptr();
    q[k] = dvs[k].data_ptr();
  }
  check(sy_bwd_table(p, w.data_ptr(), g.data_ptr(), stats.data_ptr<float>(), q, dw.data_ptr(),
                     ws.data_ptr(), ws.numel() * 4, n, tok, d, vt, wt,
                     (float)ctx->saved_data["eps"].toDouble(), stream_of(first)),
        "sy_bwd_table");
  variable_list r{dw, Tensor()};
  r.insert(r.end(), dvs.begin(), dvs.end());
  return r;
}

std::optional<Tensor> block_attn_res_sources(const std::vector<Tensor>& sources, const Tensor& w,
                                             double eps) {
  if (sources.empty() || sources.size() > SY_MAX_TABLE_ROWS || !ordinary()) return std::nullopt;
  const Tensor& first = sources[0];
  if (!plain(first) || !plain(w) || first.dim() != 3 || first.numel() == 0 || w.dim() != 1 ||
      w.size(0) != first.size(2) || w.device() != first.device())
    return std::nullopt;
  bool grad = w.requires_grad();
  for (const Tensor& s : sources) {
    if (!plain(s) || s.sizes() != first.sizes() || s.device() != first.device() ||
        s.scalar_type() != first.scalar_type())
      return std::nullopt;
    grad = grad || s.requires_grad();
  }
  if (grad && at::GradMode::is_enabled()) return BlockAttnResSources::apply(w, eps, at::TensorList(sources));
  variable_list rows;
  for (const Tensor& s : sources) rows.push_back(dense(s));
  return sources_forward(dense(w), rows, eps, nullptr);
}

// ----------------------------------------------------------------- two phases

Tensor two_phase_forward(const Tensor& v, const Tensor& w, int64_t split, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(v.device());
  const int64_t n = v.size(0), b = v.size(1), t = v.size(2), d = v.size(3), tok = b * t;
  Tensor out = at::empty({b, t, d}, v.options().requires_grad(false));
  if (stats != nullptr) *stats = at::empty({2, n, tok}, f32_on(v));
  const Tensor o1 = at::empty_like(out), ml = at::empty({4, tok}, f32_on(v));
  check(sy_two_phase(v.data_ptr(), w.data_ptr(), o1.data_ptr(), ml.data_ptr<float>(), out.data_ptr(),
                     stats != nullptr ? stats->data_ptr<float>() : nullptr, n, split, tok, d, tok * d,
                     code_of(v), code_of(w), (float)eps, stream_of(v)),
        "sy_two_phase");
  return out;
}

struct TwoPhase : torch::autograd::Function<TwoPhase> {
  static Tensor forward(AutogradContext* ctx, const Tensor& v_in, const Tensor& w_in, int64_t split,
                        double eps) {
    const Tensor v = dense(v_in), w = dense(w_in);
    Tensor stats;
    Tensor out = two_phase_forward(v, w, split, eps, &stats);
    ctx->save_for_backward({v, w, stats});
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto r = operator_backward(saved[0], saved[1], saved[2], grads[0], ctx->saved_data["eps"].toDouble());
    return {r[0], r[1], Tensor(), Tensor()};
  }
};

std::optional<Tensor> block_attn_res_two_phase(const Tensor& v, const Tensor& w, int64_t split, double eps) {
  const Stacked s = sizes_of(v, w, 1);
  if (!s.ok || split < 1 || split >= s.n) return std::nullopt;
  if (needs_grad(v, w)) return TwoPhase::apply(v, w, split, eps);
  return two_phase_forward(dense(v), dense(w), split, eps, nullptr);
}

// -------------------------------------------------------------------- batched

Tensor batched_forward(const Tensor& v, const Tensor& q, double eps) {
  const c10::DeviceGuard guard(v.device());
  const int64_t n = v.size(0), b = v.size(1), t = v.size(2), d = v.size(3), s = q.size(0);
  Tensor out = at::empty({s, b, t, d}, v.options().requires_grad(false));
  check(sy_fwd_batched(v.data_ptr(), q.data_ptr(), out.data_ptr(), n, s, b * t, d, b * t * d, code_of(v),
                       (float)eps, stream_of(v)),
        "sy_fwd_batched");
  return out;
}

struct BlockAttnResBatched : torch::autograd::Function<BlockAttnResBatched> {
  static Tensor forward(AutogradContext* ctx, const Tensor& v_in, const Tensor& q_in, double eps) {
    const Tensor v = dense(v_in), q = dense(q_in);
    ctx->save_for_backward({v, q});
    ctx->saved_data["eps"] = eps;
    return batched_forward(v, q, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &v = saved[0], &q = saved[1];
    const c10::DeviceGuard guard(v.device());
    const int64_t n = v.size(0), d = v.size(3), tok = v.size(1) * v.size(2), s = q.size(0);
    const int dt = code_of(v);
    const Tensor g = grad_like(grads[0], v);
    Tensor dv = at::empty(v.sizes(), v.options().requires_grad(false));
    Tensor dq = at::empty(q.sizes(), q.options().requires_grad(false));
    const int64_t bytes = sy_bwd_batched_workspace_bytes(n, s, tok, d, dt);
    if (bytes < 0) check(bytes, "sy_bwd_batched_workspace_bytes");
    const Tensor ws = at::empty({std::max<int64_t>(1, (bytes + 3) / 4)}, f32_on(v));
    check(sy_bwd_batched(v.data_ptr(), q.data_ptr(), g.data_ptr(), dv.data_ptr(), dq.data_ptr(),
                         ws.data_ptr(), ws.numel() * 4, n, s, tok, d, tok * d, dt,
                         (float)ctx->saved_data["eps"].toDouble(), stream_of(v)),
          "sy_bwd_batched");
    return {dv, dq, Tensor()};
  }
};

bool batched_ok(const Tensor& v, const Tensor& q) {
  return sizes_of(v, q, 2).ok && q.size(0) > 0 && v.scalar_type() == q.scalar_type();
}

std::optional<Tensor> block_attn_res_batched(const Tensor& v, const Tensor& q, double eps) {
  if (!batched_ok(v, q) || v.requires_grad() || q.requires_grad()) return std::nullopt;
  return batched_forward(dense(v), dense(q), eps);
}

std::optional<Tensor> block_attn_res_batched_train(const Tensor& v, const Tensor& q, double eps) {
  if (!batched_ok(v, q)) return std::nullopt;
  if (needs_grad(v, q)) return BlockAttnResBatched::apply(v, q, eps);
  return batched_forward(dense(v), dense(q), eps);
}

// ------------------------------------------------------------ decoder sublayers

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
int64_t chunk(const Tensor& t) { return 16 / (int64_t)t.element_size(); }

// Whether a backward may launch its kernel. A recorded one (create_graph) may not, as
// the kernels' results carry no graph, nor one inside a transform or mode or given a
// wrapped gradient (is_grads_batched): those evaluate the same gradient from torch
// operations in fp32.
bool kernel_backward(const variable_list& grads) {
  if (at::GradMode::is_enabled() || !ordinary()) return false;
  for (const Tensor& g : grads)
    if (!plain(g)) return false;
  return true;
}

Tensor norm_forward(const Tensor& x, const Tensor& w, double eps, Tensor* rinv) {
  const c10::DeviceGuard guard(x.device());
  const int64_t d = w.size(0), tok = x.numel() / d;
  Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
  if (rinv != nullptr) *rinv = at::empty({tok}, f32_on(x));
  check(sy_rms_norm(x.data_ptr(), w.data_ptr(), out.data_ptr(),
                    rinv != nullptr ? rinv->data_ptr<float>() : nullptr, tok, d, code_of(x), (float)eps,
                    stream_of(x)),
        "sy_rms_norm");
  return out;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, double eps) {
    Tensor rinv;
    Tensor out = norm_forward(x, w, eps, &rinv);
    ctx->save_for_backward({x, w, rinv});
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    const c10::DeviceGuard guard(x.device());
    if (!kernel_backward(grads)) {
      const Tensor xf = x.to(at::kFloat), gf = grads[0].to(at::kFloat), gw = gf * w.to(at::kFloat);
      const Tensor r = xf.square().mean(-1, /*keepdim=*/true).add(ctx->saved_data["eps"].toDouble()).rsqrt();
      const Tensor dx = r * gw - xf * (r.pow(3) * (gw * xf).mean(-1, /*keepdim=*/true));
      const Tensor dw = (gf * xf * r).reshape({-1, w.size(0)}).sum(0);
      return {dx.to(x.scalar_type()), dw.to(w.scalar_type()), Tensor()};
    }
    const int64_t d = w.size(0), tok = x.numel() / d;
    Tensor g = grad_like(grads[0], x);
    if (!aligned16(g)) g = g.clone();
    Tensor dx = at::empty(x.sizes(), x.options().requires_grad(false));
    Tensor dw = at::empty({d}, w.options().requires_grad(false));
    const int64_t bytes = sy_rms_norm_bwd_bytes(tok, d);
    if (bytes < 0) check(bytes, "sy_rms_norm_bwd_bytes");
    const Tensor ws = at::empty({std::max<int64_t>(1, bytes / 4)}, f32_on(x));
    check(sy_rms_norm_bwd(x.data_ptr(), w.data_ptr(), g.data_ptr(), saved[2].data_ptr<float>(), dx.data_ptr(),
                          dw.data_ptr(), ws.data_ptr(), ws.numel() * 4, tok, d, code_of(x), stream_of(x)),
          "sy_rms_norm_bwd");
    return {dx, dw, Tensor()};
  }
};

std::optional<Tensor> rms_norm(const Tensor& x, const Tensor& w, double eps) {
  if (!ordinary() || !plain(x) || !plain(w) || w.dim() != 1 || x.dim() < 1 || x.numel() == 0 ||
      x.size(-1) != w.size(0) || x.scalar_type() != w.scalar_type() || x.device() != w.device() ||
      !x.is_contiguous() || !w.is_contiguous() || !aligned16(x) || !aligned16(w) ||
      w.size(0) % chunk(x) != 0 || w.size(0) / chunk(x) > 512)
    return std::nullopt;
  if (needs_grad(x, w)) return RmsNorm::apply(x, w, eps);
  return norm_forward(x, w, eps, nullptr);
}

variable_list rope_forward(const Tensor& qkv, const Tensor& cosv, const Tensor& sinv) {
  const c10::DeviceGuard guard(qkv.device());
  const int64_t b = qkv.size(0), t = qkv.size(1), h = qkv.size(3), hd = qkv.size(4);
  variable_list r;
  for (int k = 0; k < 3; ++k) r.push_back(at::empty({b, h, t, hd}, qkv.options().requires_grad(false)));
  check(sy_rope_qkv(qkv.data_ptr(), r[0].data_ptr(), r[1].data_ptr(), r[2].data_ptr(),
                    cosv.data_ptr<float>(), sinv.data_ptr<float>(), b * t, t, h, hd, code_of(qkv), 0,
                    stream_of(qkv)),
        "sy_rope_qkv");
  return r;
}

struct RopeQkv : torch::autograd::Function<RopeQkv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& cosv,
                               const Tensor& sinv) {
    ctx->save_for_backward({cosv, sinv});
    return rope_forward(qkv, cosv, sinv);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!kernel_backward(grads)) {  // the kernel's inverse rotation
      const int64_t t = grads[0].size(2), half = grads[0].size(3) / 2;
      const Tensor c = saved[0].reshape({-1, half}).slice(0, 0, t), s = saved[1].reshape({-1, half}).slice(0, 0, t);
      variable_list d;
      for (int k = 0; k < 3; ++k) {
        Tensor g = grads[k];
        if (k < 2) {
          const auto p = g.to(at::kFloat).chunk(2, -1);
          g = at::cat({p[0] * c + p[1] * s, p[1] * c - p[0] * s}, -1).to(g.scalar_type());
        }
        d.push_back(g.transpose(1, 2));
      }
      return {at::stack(d, 2), Tensor(), Tensor()};
    }
    for (Tensor& g : grads) {
      g = dense(g);
      if (!aligned16(g)) g = g.clone();
    }
    const Tensor& q = grads[0];
    const c10::DeviceGuard guard(q.device());
    const int64_t b = q.size(0), h = q.size(1), t = q.size(2), hd = q.size(3);
    Tensor dqkv = at::empty({b, t, 3, h, hd}, q.options().requires_grad(false));
    check(sy_rope_qkv(dqkv.data_ptr(), q.data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(),
                      saved[0].data_ptr<float>(), saved[1].data_ptr<float>(), b * t, t, h, hd, code_of(q), 1,
                      stream_of(q)),
          "sy_rope_qkv");
    return {dqkv, Tensor(), Tensor()};
  }
};

// qkv [B, T, 3, H, hd], tables [>= T, 1, hd/2] -> (q, k, v), each [B, H, T, hd].
std::optional<variable_list> rope_qkv(const Tensor& qkv, const Tensor& cosv, const Tensor& sinv) {
  if (!ordinary() || !plain(qkv) || !plain(cosv) || !plain(sinv) || qkv.dim() != 5 || qkv.size(2) != 3 ||
      qkv.numel() == 0 || !qkv.is_contiguous() || !aligned16(qkv) || qkv.size(4) % (2 * chunk(qkv)) != 0 ||
      qkv.size(3) > 0xffff || qkv.size(4) > 0xffff)
    return std::nullopt;
  for (const Tensor* t : {&cosv, &sinv})
    if (t->scalar_type() != at::kFloat || t->device() != qkv.device() || !t->is_contiguous() ||
        t->requires_grad() || t->dim() != 3 || t->size(1) != 1 || t->size(2) != qkv.size(4) / 2 ||
        t->size(0) < qkv.size(1))
      return std::nullopt;
  if (at::GradMode::is_enabled() && qkv.requires_grad()) return RopeQkv::apply(qkv, cosv, sinv);
  return rope_forward(qkv, cosv, sinv);
}

// A projection as the kernels read it: dense, from a 16-byte boundary on.
Tensor rows_of(const Tensor& qkv) {
  const Tensor x = dense(qkv);
  return aligned16(x) ? x : x.clone();
}

// The gains of a norm over heads of hd: of the activations' dtype or fp32, both the same.
bool gains_ok(const Tensor& q_gain, const Tensor& k_gain, const Tensor& like, int64_t hd) {
  for (const Tensor* g : {&q_gain, &k_gain})
    if (!plain(*g) || g->dim() != 1 || g->size(0) != hd || g->device() != like.device() ||
        g->scalar_type() != q_gain.scalar_type() ||
        (g->scalar_type() != like.scalar_type() && g->scalar_type() != at::kFloat))
      return false;
  return true;
}

variable_list head_norm_forward(const Tensor& qkv, const Tensor& gq, const Tensor& gk, const Tensor& cosv,
                                const Tensor& sinv, int64_t kv, double eps) {
  const c10::DeviceGuard guard(qkv.device());
  const int64_t b = qkv.size(0), t = qkv.size(1), h = qkv.size(2) - 2 * kv, hd = qkv.size(3);
  variable_list r;
  for (int k = 0; k < 3; ++k)
    r.push_back(at::empty({b, k == 0 ? h : kv, t, hd}, qkv.options().requires_grad(false)));
  check(sy_qk_norm_rope(qkv.data_ptr(), gq.data_ptr(), gk.data_ptr(), cosv.data_ptr<float>(), sinv.data_ptr<float>(),
                        r[0].data_ptr(), r[1].data_ptr(), r[2].data_ptr(), b * t, t, h, kv, hd, code_of(qkv),
                        code_of(gq), (float)eps, stream_of(qkv)),
        "sy_qk_norm_rope");
  return r;
}

// Under capture, what a backward hands to nodes of a stream outside of it (those of the leaves,
// where an eager graph of them lives) would take that stream into the capture, which ends the
// process.
void check_capture(const Tensor& t) {
  const auto now = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index());
  const auto captures = [](hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return s != nullptr && hipStreamIsCapturing(s, &status) == hipSuccess && status != hipStreamCaptureStatusNone;
  };
  if (!captures(now.stream())) return;
  const auto node = torch::autograd::get_current_node();
  if (node == nullptr) return;
  for (const auto& edge : node->next_edges()) {
    if (!edge.function) continue;
    const auto other = edge.function->stream();
    TORCH_CHECK(!other.has_value() || *other == now.unwrap() ||
                    captures(c10::hip::HIPStreamMasqueradingAsCUDA(*other).stream()),
                "qk_norm_rope: a backward is captured while an eager graph of the same leaves lives; drop its outputs "
                "before the capture");
  }
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv_in, const Tensor& gq_in, const Tensor& gk_in,
                               const Tensor& cosv, const Tensor& sinv, int64_t kv, double eps) {
    // The inputs themselves, not the copies: a recorded backward's derivative leads to them.
    ctx->save_for_backward({qkv_in, gq_in, gk_in, cosv, sinv});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["kv"] = kv;
    return head_norm_forward(rows_of(qkv_in), dense(gq_in), dense(gk_in), cosv, sinv, kv, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor qkv = saved[0], gq = saved[1], gk = saved[2];
    const c10::DeviceGuard guard(qkv.device());
    check_capture(qkv);
    const double eps = ctx->saved_data["eps"].toDouble();
    const int64_t b = qkv.size(0), t = qkv.size(1), kv = ctx->saved_data["kv"].toInt(), h = qkv.size(2) - 2 * kv,
                  hd = qkv.size(3);
    if (!kernel_backward(grads)) {  // the same from torch operations
      const Tensor c = saved[3].reshape({-1, hd / 2}).slice(0, 0, t), s = saved[4].reshape({-1, hd / 2}).slice(0, 0, t);
      const auto parts = qkv.transpose(1, 2).split_with_sizes({h, kv, kv}, 1);
      variable_list dx, dg;
      for (int k = 0; k < 2; ++k) {
        const Tensor x = parts[k].to(at::kFloat), gain = (k == 0 ? gq : gk).to(at::kFloat);
        const auto p = grads[k].to(at::kFloat).chunk(2, -1);
        const Tensor e = at::cat({p[0] * c + p[1] * s, p[1] * c - p[0] * s}, -1);
        const Tensor r = x.square().mean(-1, /*keepdim=*/true).add(eps).rsqrt(), u = x * r;
        dx.push_back((r * (e * gain - u * (e * gain * u).mean(-1, /*keepdim=*/true))).to(qkv.scalar_type()));
        dg.push_back((e * u).sum(at::IntArrayRef{0, 1, 2}).to(gq.scalar_type()));
      }
      dx.push_back(grads[2]);
      return {at::cat(dx, 1).transpose(1, 2), dg[0], dg[1], Tensor(), Tensor(), Tensor(), Tensor()};
    }
    qkv = rows_of(qkv), gq = dense(gq), gk = dense(gk);
    int64_t strides[9];
    for (int k = 0; k < 3; ++k) {
      Tensor& g = grads[k];
      bool fits = g.stride(3) == 1 && aligned16(g);
      for (int d = 0; d < 3; ++d) fits = fits && g.stride(d) >= 0 && g.stride(d) % chunk(g) == 0;
      if (!fits) g = g.clone(at::MemoryFormat::Contiguous);
      for (int d = 0; d < 3; ++d) strides[3 * k + d] = g.stride(d);
    }
    Tensor dqkv = at::empty(qkv.sizes(), qkv.options().requires_grad(false));
    Tensor dgq = at::empty({hd}, gq.options().requires_grad(false));
    Tensor dgk = at::empty({hd}, gk.options().requires_grad(false));
    const int64_t bytes = sy_qk_norm_rope_bwd_bytes(b * t, h, kv, hd, code_of(qkv));
    if (bytes < 0) check(bytes, "sy_qk_norm_rope_bwd_bytes");
    const Tensor ws = at::empty({std::max<int64_t>(1, bytes / 4)}, f32_on(qkv));
    check(sy_qk_norm_rope_bwd(qkv.data_ptr(), gq.data_ptr(), gk.data_ptr(), saved[3].data_ptr<float>(),
                              saved[4].data_ptr<float>(), grads[0].data_ptr(), grads[1].data_ptr(),
                              grads[2].data_ptr(), strides, dqkv.data_ptr(), dgq.data_ptr(), dgk.data_ptr(),
                              ws.data_ptr(), ws.numel() * 4, b * t, t, h, kv, hd, code_of(qkv), code_of(gq),
                              (float)eps, stream_of(qkv)),
          "sy_qk_norm_rope_bwd");
    return {dqkv, dgq, dgk, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// qkv [B, T, heads + 2 kv, hd] (kv 0: a third of the heads), gains [hd], tables [>= T, (1,) hd/2]
// -> (q, k, v), each [B, heads of it, T, hd].
std::optional<variable_list> qk_norm_rope(const Tensor& qkv_in, const Tensor& gq, const Tensor& gk, const Tensor& cosv,
                                          const Tensor& sinv, int64_t kv, double eps) {
  if (!ordinary() || !plain(qkv_in) || qkv_in.dim() != 4 || qkv_in.numel() == 0 || !plain(cosv) || !plain(sinv))
    return std::nullopt;
  const int64_t rows = qkv_in.size(2), hd = qkv_in.size(3);
  if (kv == 0) {
    if (rows % 3 != 0) return std::nullopt;
    kv = rows / 3;
  }
  if (kv < 1 || rows - 2 * kv < 1 || rows > 0xffff || hd % 8 != 0 || hd > 256 || !gains_ok(gq, gk, qkv_in, hd))
    return std::nullopt;
  for (const Tensor* t : {&cosv, &sinv})
    if (t->scalar_type() != at::kFloat || t->device() != qkv_in.device() || !t->is_contiguous() || tracked(*t) ||
        (t->dim() != 2 && t->dim() != 3) || t->size(-1) != hd / 2 || t->numel() != t->size(0) * t->size(-1) ||
        t->size(0) < qkv_in.size(1))
      return std::nullopt;
  if (tracked(qkv_in) || tracked(gq) || tracked(gk)) return QkNormRope::apply(qkv_in, gq, gk, cosv, sinv, kv, eps);
  return head_norm_forward(rows_of(qkv_in), dense(gq), dense(gk), cosv, sinv, kv, eps);
}

struct SwiGlu : torch::autograd::Function<SwiGlu> {
  static Tensor run(const Tensor& gu) {
    const c10::DeviceGuard guard(gu.device());
    auto sizes = gu.sizes().vec();
    const int64_t f = sizes.back() / 2;
    sizes.back() = f;
    Tensor out = at::empty(sizes, gu.options().requires_grad(false));
    check(sy_swiglu(gu.data_ptr(), out.data_ptr(), out.numel() / f, f, code_of(gu), stream_of(gu)), "sy_swiglu");
    return out;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& gu) {
    ctx->save_for_backward({gu});
    return run(gu);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor gu = ctx->get_saved_variables()[0];
    const c10::DeviceGuard guard(gu.device());
    if (!kernel_backward(grads)) {
      const auto p = gu.to(at::kFloat).chunk(2, -1);
      const Tensor gf = grads[0].to(at::kFloat), s = at::sigmoid(p[0]);
      return {at::cat({gf * p[1] * s * (1 + p[0] * (1 - s)), gf * p[0] * s}, -1).to(gu.scalar_type())};
    }
    Tensor g = grad_like(grads[0], gu);
    if (!aligned16(g)) g = g.clone();
    Tensor d = at::empty(gu.sizes(), gu.options().requires_grad(false));
    const int64_t f = gu.size(-1) / 2;
    check(sy_swiglu_bwd(gu.data_ptr(), g.data_ptr(), d.data_ptr(), g.numel() / f, f, code_of(gu),
                        stream_of(gu)),
          "sy_swiglu_bwd");
    return {d};
  }
};

std::optional<Tensor> swiglu(const Tensor& gu) {
  if (!ordinary() || !plain(gu) || gu.dim() < 1 || gu.numel() == 0 || !gu.is_contiguous() || !aligned16(gu) ||
      gu.size(-1) % (2 * chunk(gu)) != 0)
    return std::nullopt;
  if (at::GradMode::is_enabled() && gu.requires_grad()) return SwiGlu::apply(gu);
  return SwiGlu::run(gu);
}

// -------------------------------------------------------------------- serving

// A dense GPU tensor of another type that nothing intercepts.
bool whole_of(const Tensor& t, at::ScalarType type) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped{DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                        DispatchKey::Batched, DispatchKey::Functionalize};
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == type &&
         !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.key_set().has_any(wrapped);
}
bool whole(const Tensor& t) { return whole_of(t, at::kInt); }

void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

constexpr int64_t kMostTokens = (int64_t)1 << 30;  // in a sequence's pages, and in a prefix

// The cache and the sequences of a call with n_tok packed rows and `heads` query heads;
// false where the Python function has to see the call.
bool paged_of(const Tensor& like, int64_t heads, const Tensor& k, const Tensor& v, const Tensor& table,
              const Tensor& lengths, const std::optional<Tensor>& starts, sy_paged* c) {
  if (!ordinary() || !plain(like) || !plain(k) || !plain(v) || !whole(table) || !whole(lengths) || k.dim() != 4 ||
      k.sizes() != v.sizes() || k.strides() != v.strides() || like.scalar_type() != k.scalar_type() ||
      v.scalar_type() != k.scalar_type() || table.dim() != 2 || lengths.dim() != 1 ||
      table.size(0) != lengths.size(0) || !lengths.is_contiguous() || lengths.size(0) < 1 ||
      (table.size(1) > 1 && table.stride(1) != 1) || table.size(1) < 1 || k.size(2) < 1 ||
      table.size(1) > kMostTokens / k.size(2))
    return false;
  for (const Tensor* t : {&k, &v, &table, &lengths})
    if (t->device() != like.device()) return false;
  const int64_t chunk_of = chunk(k), page = k.size(2), hd = k.size(3);
  if (k.size(0) < 1 || k.size(1) < 1 || page < 1 || (page & (page - 1)) != 0 || hd < 8 || hd > 256 || hd % 8 != 0 ||
      k.stride(3) != 1 || heads < 1 || heads % k.size(1) != 0 || heads > 0xffff || !aligned16(k) || !aligned16(v))
    return false;
  for (int d = 0; d < 3; ++d)
    if (k.stride(d) < 0 || k.stride(d) % chunk_of != 0) return false;
  const int64_t span = ((int64_t)1 << 32) / (int64_t)k.element_size();
  if (k.stride(0) >= span || k.stride(2) >= span / page) return false;
  const int64_t n_seq = lengths.size(0), n_tok = like.size(0);
  if (starts.has_value()) {
    if (!whole(*starts) || starts->dim() != 1 || starts->size(0) != n_seq + 1 || !starts->is_contiguous() ||
        starts->device() != like.device())
      return false;
  } else if (n_tok % n_seq != 0) {
    return false;
  }
  *c = sy_paged{k.data_ptr(), v.data_ptr(), table.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(),
                starts.has_value() ? starts->data_ptr<int32_t>() : nullptr, k.stride(0), k.stride(1), k.stride(2),
                table.stride(0), n_seq, n_tok, k.size(0), table.size(1), (int32_t)page, (int32_t)heads,
                (int32_t)k.size(1), (int32_t)hd, code_of(k)};
  return true;
}

// The caller's output, if it is one the kernels can write.
bool out_ok(const std::optional<Tensor>& out, const Tensor& like, int64_t n_tok, int64_t heads, int64_t hd) {
  return !out.has_value() ||
         (plain(*out) && out->dim() == 3 && out->size(0) == n_tok && out->size(1) == heads && out->size(2) == hd &&
          out->is_contiguous() && aligned16(*out) && out->scalar_type() == like.scalar_type() &&
          out->device() == like.device() && !tracked(*out));
}

std::optional<Tensor> paged_append(const Tensor& qkv_in, const Tensor& cosv, const Tensor& sinv, const Tensor& k,
                                   const Tensor& v, const Tensor& table, const Tensor& lengths,
                                   const std::optional<Tensor>& starts, int64_t prefix_len,
                                   const std::optional<Tensor>& out, const std::optional<Tensor>& q_gain,
                                   const std::optional<Tensor>& k_gain, double eps) {
  sy_paged c;
  if (qkv_in.dim() != 3 || qkv_in.size(0) < 1 || k.dim() != 4) return std::nullopt;
  const int64_t heads = qkv_in.size(1) - 2 * k.size(1);
  if (!paged_of(qkv_in, heads, k, v, table, lengths, starts, &c) || qkv_in.size(2) != c.hd || tracked(qkv_in) ||
      tracked(k) || tracked(v) || prefix_len < 0 || prefix_len > kMostTokens ||
      !out_ok(out, qkv_in, c.n_tok, heads, c.hd))
    return std::nullopt;
  for (const Tensor* t : {&cosv, &sinv})
    if (!plain(*t) || t->scalar_type() != at::kFloat || t->device() != qkv_in.device() || !t->is_contiguous() ||
        t->dim() < 2 || t->size(-1) * 2 != c.hd || t->numel() != t->size(0) * t->size(-1) || tracked(*t))
      return std::nullopt;
  if (cosv.sizes() != sinv.sizes() || q_gain.has_value() != k_gain.has_value()) return std::nullopt;
  const bool norm = q_gain.has_value();
  if (norm && (!gains_ok(*q_gain, *k_gain, qkv_in, c.hd) || tracked(*q_gain) || tracked(*k_gain))) return std::nullopt;
  const c10::DeviceGuard guard(qkv_in.device());
  const bool fits = qkv_in.stride(2) == 1 && qkv_in.stride(0) >= 0 && qkv_in.stride(1) >= 0 &&
                    (!norm || (qkv_in.stride(0) % 4 == 0 && qkv_in.stride(1) % 4 == 0 &&
                               reinterpret_cast<uintptr_t>(qkv_in.data_ptr()) % (4 * qkv_in.element_size()) == 0));
  const Tensor qkv = fits ? qkv_in : qkv_in.clone(at::MemoryFormat::Contiguous);
  Tensor q = out.has_value() ? *out : at::empty({c.n_tok, heads, c.hd}, qkv.options().requires_grad(false));
  if (norm) {
    const Tensor gq = dense(*q_gain), gk = dense(*k_gain);
    check(sy_paged_append_norm(&c, qkv.data_ptr(), qkv.stride(0), qkv.stride(1), gq.data_ptr(), gk.data_ptr(),
                               code_of(gq), (float)eps, cosv.data_ptr<float>(), sinv.data_ptr<float>(), cosv.size(0),
                               prefix_len, q.data_ptr(), out.has_value() ? 0 : 1, stream_of(qkv)),
          "sy_paged_append_norm");
  } else {
    check(sy_paged_append(&c, qkv.data_ptr(), qkv.stride(0), qkv.stride(1), cosv.data_ptr<float>(),
                          sinv.data_ptr<float>(), cosv.size(0), prefix_len, q.data_ptr(), out.has_value() ? 0 : 1,
                          stream_of(qkv)),
          "sy_paged_append");
  }
  changed(k);
  changed(v);
  if (out.has_value()) changed(q);
  return q;
}

std::optional<Tensor> paged_attention(const Tensor& q_in, const Tensor& k, const Tensor& v, const Tensor& table,
                                      const Tensor& lengths, const std::optional<Tensor>& starts,
                                      const std::optional<Tensor>& prefix_pages, int64_t prefix_len, double scale,
                                      const std::optional<Tensor>& out) {
  sy_paged c;
  if (q_in.dim() != 3 || q_in.size(0) < 1) return std::nullopt;
  const int64_t heads = q_in.size(1);
  if (!paged_of(q_in, heads, k, v, table, lengths, starts, &c) || q_in.size(2) != c.hd || tracked(q_in) ||
      tracked(k) || tracked(v) || prefix_len < 0 || prefix_len > kMostTokens ||
      !out_ok(out, q_in, c.n_tok, heads, c.hd))
    return std::nullopt;
  if (prefix_len > 0 && (!prefix_pages.has_value() || !whole(*prefix_pages) || prefix_pages->dim() != 1 ||
                         !prefix_pages->is_contiguous() || prefix_pages->device() != q_in.device() ||
                         prefix_pages->size(0) * c.page < prefix_len))
    return std::nullopt;
  const c10::DeviceGuard guard(q_in.device());
  const int64_t ce = chunk(q_in);
  const bool fits = q_in.stride(2) == 1 && q_in.stride(0) >= 0 && q_in.stride(1) >= 0 && q_in.stride(0) % ce == 0 &&
                    q_in.stride(1) % ce == 0 && aligned16(q_in);
  const Tensor q = fits ? q_in : q_in.clone(at::MemoryFormat::Contiguous);
  Tensor o = out.has_value() ? *out : at::empty({c.n_tok, heads, c.hd}, q.options().requires_grad(false));
  const int64_t bytes = sy_paged_attention_workspace_bytes(&c, prefix_len);
  if (bytes < 0) return std::nullopt;
  Tensor ws;
  if (bytes > 0) ws = at::empty({bytes / 4}, f32_on(q));
  check(sy_paged_attention(&c, q.data_ptr(), q.stride(0), q.stride(1), o.data_ptr(),
                           prefix_len > 0 ? prefix_pages->data_ptr<int32_t>() : nullptr, prefix_len, (float)scale,
                           out.has_value() ? 0 : 1, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
        "sy_paged_attention");
  if (out.has_value()) changed(o);
  return o;
}

// Settings as numbers, each replaced by a tensor of one a row where that is given.
std::optional<Tensor> sample_tokens(const Tensor& logits_in, const Tensor& u, double temperature, int64_t top_k,
                                    double top_p, double min_p, const std::optional<Tensor>& temperatures,
                                    const std::optional<Tensor>& top_ks, const std::optional<Tensor>& top_ps,
                                    const std::optional<Tensor>& min_ps) {
  if (!ordinary() || !plain(logits_in) || !plain(u) || logits_in.dim() != 2 || logits_in.numel() == 0 ||
      logits_in.size(1) > (1 << 18) || u.dim() != 1 || u.size(0) != logits_in.size(0) ||
      u.scalar_type() != at::kFloat || !u.is_contiguous() || u.device() != logits_in.device())
    return std::nullopt;
  sy_sampling how{temperature, top_p, min_p, top_k, nullptr, nullptr, nullptr, nullptr};
  const auto row_of = [&](const std::optional<Tensor>& t, at::ScalarType dtype) {
    return (dtype == at::kInt ? whole(*t) : plain(*t)) && t->dim() == 1 && t->size(0) == u.size(0) &&
           t->scalar_type() == dtype && t->is_contiguous() && t->device() == u.device();
  };
  const std::pair<const std::optional<Tensor>*, const float**> floats[] = {
      {&temperatures, &how.temperatures}, {&top_ps, &how.top_ps}, {&min_ps, &how.min_ps}};
  for (const auto& [t, p] : floats)
    if (t->has_value()) {
      if (!row_of(*t, at::kFloat)) return std::nullopt;
      *p = (*t)->data_ptr<float>();
    }
  if (top_ks.has_value()) {
    if (!row_of(top_ks, at::kInt)) return std::nullopt;
    how.top_ks = top_ks->data_ptr<int32_t>();
  }
  const c10::DeviceGuard guard(u.device());
  const bool rows = (logits_in.stride(1) == 1 || logits_in.size(1) == 1) && logits_in.stride(0) >= 0;
  const Tensor logits = rows ? logits_in : logits_in.contiguous();
  Tensor tokens = at::empty({logits.size(0)}, logits.options().dtype(at::kLong).requires_grad(false));
  check(sy_sample(logits.data_ptr(), u.data_ptr<float>(), tokens.data_ptr<int64_t>(), &how, logits.size(0),
                  logits.size(1), logits.stride(0), code_of(logits), stream_of(logits)),
        "sy_sample");
  return tokens;
}

std::optional<Tensor> adjust_logits(const Tensor& logits_in, double repetition, double presence, double frequency,
                                    const std::optional<Tensor>& tokens, const std::optional<Tensor>& lengths,
                                    const std::optional<Tensor>& prompts, const std::optional<Tensor>& repetitions,
                                    const std::optional<Tensor>& presences, const std::optional<Tensor>& frequencies,
                                    const std::optional<Tensor>& bias, const std::optional<Tensor>& allowed,
                                    const std::optional<Tensor>& out) {
  if (!ordinary() || !plain(logits_in) || tracked(logits_in) || logits_in.dim() != 2 || logits_in.numel() == 0 ||
      logits_in.size(1) > (1 << 30))
    return std::nullopt;
  const int64_t b = logits_in.size(0), v = logits_in.size(1);
  const auto dev = logits_in.device();
  sy_adjusting how{};
  how.repetition = repetition, how.presence = presence, how.frequency = frequency;
  how.tokens_bytes = 8;
  if (tokens.has_value()) {
    const Tensor& t = *tokens;
    if (!(whole_of(t, at::kLong) || whole(t)) || t.device() != dev || t.dim() != 2 || t.size(0) != b ||
        t.size(1) > (1 << 30) || t.stride(0) < 0 || (t.size(1) > 1 && t.stride(1) != 1))
      return std::nullopt;
    how.tokens = t.data_ptr(), how.tokens_stride = t.stride(0), how.n_tokens = t.size(1);
    how.tokens_bytes = (int32_t)t.element_size();
  } else if (lengths.has_value() || prompts.has_value()) {
    return std::nullopt;
  }
  const std::pair<const std::optional<Tensor>*, const int32_t**> ints[] = {{&lengths, &how.lengths},
                                                                          {&prompts, &how.prompt_lengths}};
  for (const auto& [t, p] : ints)
    if (t->has_value()) {
      if (!whole(**t) || (*t)->dim() != 1 || (*t)->size(0) != b || !(*t)->is_contiguous() || (*t)->device() != dev)
        return std::nullopt;
      *p = (*t)->data_ptr<int32_t>();
    }
  const std::pair<const std::optional<Tensor>*, const float**> floats[] = {
      {&repetitions, &how.repetitions}, {&presences, &how.presences}, {&frequencies, &how.frequencies}};
  for (const auto& [t, p] : floats)
    if (t->has_value()) {
      if (!plain(**t) || tracked(**t) || (*t)->scalar_type() != at::kFloat || (*t)->dim() != 1 || (*t)->size(0) != b ||
          !(*t)->is_contiguous() || (*t)->device() != dev)
        return std::nullopt;
      *p = (*t)->data_ptr<float>();
    }
  if (bias.has_value()) {
    const Tensor& t = *bias;
    if (!plain(t) || tracked(t) || (t.scalar_type() != at::kFloat && t.scalar_type() != logits_in.scalar_type()) ||
        t.device() != dev || t.dim() < 1 || t.dim() > 2 || t.size(-1) != v || (v > 1 && t.stride(-1) != 1) ||
        (t.dim() == 2 && (t.size(0) != b || t.stride(0) < 0)))
      return std::nullopt;
    how.bias = t.data_ptr(), how.bias_dtype = code_of(t), how.bias_stride = t.dim() == 2 ? t.stride(0) : 0;
  }
  if (allowed.has_value()) {
    const Tensor& t = *allowed;
    const bool words = whole(t);
    const int64_t n = words ? (v + 31) / 32 : v;
    if ((!words && !whole_of(t, at::kBool)) || t.device() != dev || t.dim() < 1 || t.dim() > 2 || t.size(-1) != n ||
        (n > 1 && t.stride(-1) != 1) || (t.dim() == 2 && (t.size(0) != b || t.stride(0) < 0)))
      return std::nullopt;
    how.mask = t.data_ptr(), how.mask_kind = words ? 1 : 2, how.mask_stride = t.dim() == 2 ? t.stride(0) : 0;
  }
  if (out.has_value() && (!plain(*out) || tracked(*out) || out->sizes() != logits_in.sizes() || out->device() != dev ||
                          out->scalar_type() != logits_in.scalar_type() || (v > 1 && out->stride(1) != 1) ||
                          (b > 1 && out->stride(0) < v)))
    return std::nullopt;
  const c10::DeviceGuard guard(dev);
  const bool rows = (logits_in.stride(1) == 1 || v == 1) && logits_in.stride(0) >= 0;
  const Tensor x = rows ? logits_in : logits_in.contiguous();
  Tensor y = out.has_value() ? *out : at::empty({b, v}, x.options().requires_grad(false));
  check(sy_adjust(x.data_ptr(), y.data_ptr(), &how, b, v, x.stride(0), y.stride(0), code_of(x), stream_of(x)),
        "sy_adjust");
  if (out.has_value()) changed(y);
  return y;
}

std::optional<Tensor> linear4(const Tensor& x_in, const Tensor& tiles, const Tensor& scales,
                              const std::optional<Tensor>& zeros, int64_t n, int64_t k, int64_t group) {
  if (!ordinary() || !plain(x_in) || tracked(x_in) || x_in.dim() < 1 || x_in.numel() == 0 || x_in.size(-1) != k ||
      !whole(tiles) || !plain(scales) || tracked(scales) || scales.scalar_type() != x_in.scalar_type() ||
      tiles.device() != x_in.device() || scales.device() != x_in.device() || !tiles.is_contiguous() ||
      !scales.is_contiguous() || !aligned16(tiles) || !aligned16(scales) || (group != 32 && group != 64 && group != 128) || n < 1 ||
      tiles.numel() != (n + 15) / 16 * ((k + 127) / 128) * 256 || scales.numel() != tiles.numel() * 8 / group ||
      x_in.numel() / k > 0x7fffffff)
    return std::nullopt;
  if (zeros.has_value() && (!whole_of(*zeros, at::kByte) || zeros->device() != x_in.device() ||
                            !zeros->is_contiguous() || zeros->numel() != scales.numel() ||
                            reinterpret_cast<uintptr_t>(zeros->data_ptr()) % 4 != 0))
    return std::nullopt;
  const c10::DeviceGuard guard(x_in.device());
  Tensor x = x_in.dim() == 2 ? x_in : x_in.reshape({-1, k});
  if ((k > 1 && x.stride(1) != 1) || x.stride(0) < 0) x = x.contiguous();
  auto sizes = x_in.sizes().vec();
  sizes.back() = n;
  Tensor out = at::empty(sizes, x.options().requires_grad(false));
  check(sy_linear4(x.data_ptr(), x.stride(0), tiles.data_ptr(), scales.data_ptr(),
                   zeros.has_value() ? zeros->data_ptr<uint8_t>() : nullptr, out.data_ptr(), x.size(0), n, k, group,
                   code_of(x), stream_of(x)),
        "sy_linear4");
  return out;
}

}  // namespace

// The interpreter's lock is released during a call, as ctypes does.
PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const auto free_lock = py::call_guard<py::gil_scoped_release>();
  m.def("block_attn_res", &block_attn_res, free_lock);
  m.def("block_attn_res_gain", &block_attn_res_gain, free_lock);
  m.def("block_attn_res_sources", &block_attn_res_sources, free_lock);
  m.def("block_attn_res_two_phase", &block_attn_res_two_phase, free_lock);
  m.def("block_attn_res_batched", &block_attn_res_batched, free_lock);
  m.def("block_attn_res_batched_train", &block_attn_res_batched_train, free_lock);
  m.def("rms_norm", &rms_norm, free_lock);
  m.def("rope_qkv", &rope_qkv, free_lock);
  m.def("swiglu", &swiglu, free_lock);
  m.def("qk_norm_rope", &qk_norm_rope, free_lock);
  m.def("paged_append", &paged_append, free_lock);
  m.def("paged_attention", &paged_attention, free_lock);
  m.def("adjust_logits", &adjust_logits, free_lock);
  m.def("sample_tokens", &sample_tokens, free_lock);
  m.def("linear4", &linear4, free_lock);
}
