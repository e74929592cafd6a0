// The training operators' host side in native code: autograd functions over the C ABI's
// router and block norm, and the AdamW step's lists of tensors. As Python autograd functions
// a forward and backward of a small batch spent 60-70 us on the host, most of it there.
// Included by tmoe_torch.cpp. The functions check their arguments themselves (shapes and
// dtypes before devices, so that a machine without a GPU refuses them alike) and run on
// the current stream of their tensors' device.
#pragma once

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "tmoe.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

struct TrainEntry {
  decltype(&tmoe_last_error) last_error;
  decltype(&tmoe_router_workspace_bytes) router_workspace_bytes;
  decltype(&tmoe_router_forward) router_forward;
  decltype(&tmoe_router_backward) router_backward;
  decltype(&tmoe_block_norm_workspace_bytes) norm_workspace_bytes;
  decltype(&tmoe_block_norm_forward) norm_forward;
  decltype(&tmoe_block_norm_backward) norm_backward;
  decltype(&tmoe_adamw_step) adamw_step;
} g_train{};

void check_rc(int rc) { TORCH_CHECK(rc >= 0, "tmoe error ", rc, ": ", g_train.last_error()); }
void* current_stream(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
void check_hip(const at::Tensor& t, const char* who) {
  TORCH_CHECK(t.device().is_cuda(), who, " runs on HIP devices only; input is on ", t.device());
}
int32_t dtype_of(const at::Tensor& t, const char* who) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kBFloat16 || s == at::kFloat, who, ": dtype ", s,
              ": supported are bfloat16 and float32");
  return s == at::kBFloat16 ? TMOE_BF16 : TMOE_F32;
}
const void* ptr_of(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }
void* out_ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool wants_grad(std::initializer_list<const OptTensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const OptTensor* t : ts)
    if (*t && (*t)->requires_grad()) return true;
  return false;
}

// A leaf's accumulator lives as long as a graph that holds it and runs on the stream that
// this graph was made on. Under capture a backward that meets one of another stream would
// take that stream into the capture, which ends the process: refused here instead.
void check_capture(std::initializer_list<const OptTensor*> ts, const char* who) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const OptTensor* t : ts) {
    if (!*t || !(*t)->requires_grad() || (*t)->grad_fn()) continue;
    const auto acc = torch::autograd::impl::try_get_grad_accumulator(**t);
    if (!acc || !acc->stream()) continue;
    TORCH_CHECK(acc->stream()->id() == c10::hip::getCurrentHIPStream((*t)->device().index()).id(), who,
                ": a graph that was made outside this capture, on another stream, still holds one of "
                "these leaves; delete its outputs before the capture");
  }
}

// The kernels carry no tangents: an operand that has one would lose it without a word. Only
// inside a level of forward-mode derivatives does a tensor have one.
bool tangents_live() {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
         torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
}
void check_tangent(const at::Tensor& t, const char* who) {
  TORCH_CHECK(!t._fw_grad(0).defined(), who, " has no forward-mode derivative");
}

// The rows (..., d) of t at one stride; a contiguous copy where they have none.
struct Rows {
  at::Tensor t;
  int64_t stride = 0;
};
Rows rows_of(const at::Tensor& t) {
  const int64_t n = t.dim(), d = t.size(n - 1);
  bool ok = d <= 1 || t.stride(n - 1) == 1;
  int64_t stride = -1, next = -1;   // of a row; what the next outer axis has to step by
  for (int64_t i = n - 2; i >= 0 && ok; --i) {
    if (t.size(i) == 1) continue;
    if (stride < 0) stride = t.stride(i);
    else ok = t.stride(i) == next;
    next = t.stride(i) * t.size(i);
  }
  if (stride < 0) stride = d;        // one row
  if (!ok || stride < d) return {t.contiguous(), d};
  return {t, stride};
}

// A backward that ran with gradients on (create_graph) has gradients of its own that nobody
// computed: asking for them is an error, not zero.
variable_list once(variable_list grads, const char* who) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (const at::Tensor& g : grads)
    if (g.defined()) given.push_back(g.detach().requires_grad_(true));
  if (given.empty()) return grads;
  auto err = std::make_shared<torch::autograd::DelayedError>(
      std::string(who) + ": its backward cannot be differentiated", (int64_t)given.size());
  given = (*err)(std::move(given));
  size_t i = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = given[i++];
  return grads;
}

// ---- router --------------------------------------------------------------------

constexpr const char* kRouter = "fused_router";

struct RouterCall {
  at::Tensor raw;
  OptTensor mask, tau_dev;
  double tau = 0, cap = 0;
  int64_t k = 0;
  tmoe_router args() const {
    tmoe_router r{};
    r.raw = raw.const_data_ptr();
    r.B = raw.size(0);
    r.E = raw.size(1);
    r.row_stride = r.B > 1 ? raw.stride(0) : r.E;
    r.k = k;
    r.dtype = raw.scalar_type() == at::kBFloat16 ? TMOE_BF16 : TMOE_F32;
    r.cap = (float)cap;
    r.temperature = (float)tau;
    r.temperature_dev = static_cast<const float*>(ptr_of(tau_dev));
    r.mask = static_cast<const uint8_t*>(ptr_of(mask));
    return r;
  }
};

// idx, w, lb, z, counts, tokens
variable_list router_forward(const RouterCall& c) {
  const c10::DeviceGuard guard(c.raw.device());
  const tmoe_router r = c.args();
  const auto o = c.raw.options();
  at::Tensor idx = at::empty({r.B, r.k}, o.dtype(at::kLong));
  at::Tensor w = at::empty({r.B, r.k}, o.dtype(at::kFloat));
  at::Tensor lb = at::empty({}, o.dtype(at::kFloat)), z = at::empty({}, o.dtype(at::kFloat));
  at::Tensor tokens = at::empty({}, o.dtype(at::kFloat));
  at::Tensor counts = at::empty({r.E}, o.dtype(at::kLong));
  const size_t nws = g_train.router_workspace_bytes(r.B, r.E);
  at::Tensor ws = bytes_like(c.raw, nws);
  check_rc(g_train.router_forward(&r, idx.data_ptr<int64_t>(), w.data_ptr<float>(),
                                  lb.data_ptr<float>(), z.data_ptr<float>(), tokens.data_ptr<float>(),
                                  counts.data_ptr<int64_t>(), ws.data_ptr(), nws,
                                  current_stream(c.raw)));
  return {idx, w, lb, z, counts, tokens};
}

struct Router : torch::autograd::Function<Router> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& raw, RouterCall c) {
    variable_list o = router_forward(c);
    const at::Tensor tokens = o.back();
    o.pop_back();
    ctx->mark_non_differentiable({o[0], o[4]});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({raw.is_same(c.raw) ? raw : c.raw, c.mask.value_or(at::Tensor()),
                            c.tau_dev.value_or(at::Tensor()), o[0], tokens, o[4]});
    ctx->saved_data["tau"] = c.tau;
    ctx->saved_data["cap"] = c.cap;
    ctx->saved_data["k"] = c.k;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    RouterCall c;
    c.raw = s[0];
    if (s[1].defined()) c.mask = s[1];
    if (s[2].defined()) c.tau_dev = s[2];
    c.tau = ctx->saved_data["tau"].toDouble();
    c.cap = ctx->saved_data["cap"].toDouble();
    c.k = ctx->saved_data["k"].toInt();
    if (!g[1].defined() && !g[2].defined() && !g[3].defined()) return {at::Tensor(), at::Tensor()};
    const c10::DeviceGuard guard(c.raw.device());
    const tmoe_router r = c.args();
    at::Tensor dw = g[1].defined() ? g[1].contiguous() : g[1];
    at::Tensor draw = at::empty({r.B, r.E}, c.raw.options());
    auto f = [](const at::Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; };
    check_rc(g_train.router_backward(&r, s[3].const_data_ptr<int64_t>(), f(s[4]),
                                     s[5].const_data_ptr<int64_t>(), f(dw), f(g[2]), f(g[3]),
                                     draw.data_ptr(), current_stream(c.raw)));
    return once({draw, at::Tensor()}, kRouter);
  }
};

// router(raw, k, temperature: number or None, its device tensor or None, cap, mask or None):
// (idx, w, lb, z, counts)
PyObject* router(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (bad_args(n, 6, "router")) return nullptr;
  const at::Tensor& raw = tensor(a[0]);
  RouterCall c;
  c.k = integer(a[1]);
  c.cap = PyFloat_AsDouble(a[4]);
  if (a[3] == Py_None) c.tau = PyFloat_AsDouble(a[2]);
  if (PyErr_Occurred()) return nullptr;
  dtype_of(raw, kRouter);
  TORCH_CHECK(raw.dim() == 2, kRouter, ": raw logits (B, E) expected, got ", raw.sizes());
  TORCH_CHECK(raw.size(1) >= 1 && c.k >= 1 && c.k <= raw.size(1), kRouter, ": top_k ", c.k, " of ",
              raw.size(1), " experts");
  TORCH_CHECK(raw.size(1) <= 256 && c.k <= 16, kRouter, ": at most 256 experts and top_k 16, got ",
              raw.size(1), " and ", c.k);
  if (a[5] != Py_None) {
    const at::Tensor& m = tensor(a[5]);
    TORCH_CHECK(m.scalar_type() == at::kBool && m.dim() == 1 && m.size(0) == raw.size(0), kRouter,
                ": mask (", raw.size(0), ") of bool expected, got ", m.sizes(), " of ", m.scalar_type());
    TORCH_CHECK(m.device() == raw.device(), kRouter, ": mask on ", m.device(), ", logits on ",
                raw.device());
    c.mask = m.contiguous();
  }
  if (a[3] != Py_None) {
    const at::Tensor& t = tensor(a[3]);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == 1 && !t.requires_grad(), kRouter,
                ": temperature: a number, or a float32 tensor of one value that needs no gradient");
    TORCH_CHECK(t.device() == raw.device(), kRouter, ": temperature on ", t.device(), ", logits on ",
                raw.device());
    c.tau_dev = t;
  } else {
    TORCH_CHECK(c.tau > 0 && std::isfinite((float)c.tau), kRouter, ": temperature ", c.tau);
  }
  TORCH_CHECK(c.cap > 0 && std::isfinite((float)c.cap), kRouter, ": scale ", c.cap);
  if (tangents_live()) {
    check_tangent(raw, kRouter);
    if (c.tau_dev) check_tangent(*c.tau_dev, kRouter);
  }
  check_hip(raw, kRouter);
  variable_list o;
  {
    pybind11::gil_scoped_release nogil;
    {
      const at::NoGradGuard no_grad;
      c.raw = rows_of(raw).t;
    }
    if (at::GradMode::is_enabled() && raw.requires_grad()) {
      const c10::DeviceGuard guard(raw.device());
      const OptTensor leaf = raw;
      check_capture({&leaf}, kRouter);
      o = Router::apply(raw, c);
    } else {
      o = router_forward(c);
    }
  }
  PyObject* r = PyTuple_New(5);
  if (!r) return nullptr;
  for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(o[i]));
  return r;
  END_HANDLE_TH_ERRORS
}

// ---- block norm ----------------------------------------------------------------

constexpr const char* kNorm = "fused_block_norm";

struct NormCall {
  OptTensor x, gate, post, gamma, next;
  at::Tensor y;
  double eps = 0;
  bool want_r = true;
};

struct NormRows {
  Rows x, y, gate;
  OptTensor post, gamma, next;
  tmoe_block_norm n{};
};
void fill(NormRows& k, double eps) {
  const at::Tensor& y = k.y.t;
  k.n.y = y.const_data_ptr();
  k.n.y_stride = k.y.stride;
  if (k.x.t.defined()) { k.n.x = k.x.t.const_data_ptr(); k.n.x_stride = k.x.stride; }
  if (k.gate.t.defined()) { k.n.gate = k.gate.t.const_data_ptr(); k.n.gate_stride = k.gate.stride; }
  k.n.post_weight = ptr_of(k.post);
  k.n.gamma = ptr_of(k.gamma);
  k.n.next_weight = ptr_of(k.next);
  k.n.d = y.size(y.dim() - 1);
  k.n.T = k.n.d ? y.numel() / k.n.d : 0;
  k.n.dtype = y.scalar_type() == at::kBFloat16 ? TMOE_BF16 : TMOE_F32;
  k.n.eps = (float)eps;
}
OptTensor contiguous(const OptTensor& t) { return t ? OptTensor(t->contiguous()) : t; }

// r, h, inv (undefined where not wanted)
variable_list norm_forward(const NormCall& c, NormRows& k, bool want_inv) {
  const c10::DeviceGuard guard(c.y.device());
  k.y = rows_of(c.y);
  if (c.x) k.x = rows_of(*c.x);
  if (c.gate) k.gate = rows_of(*c.gate);
  k.post = contiguous(c.post);
  k.gamma = contiguous(c.gamma);
  k.next = contiguous(c.next);
  fill(k, c.eps);
  const auto o = c.y.options();
  at::Tensor r, h, inv;
  if (c.want_r) r = at::empty(c.y.sizes(), o);
  if (c.next) h = at::empty(c.y.sizes(), o);
  if (want_inv && (c.post || c.next)) inv = at::empty({2, k.n.T}, o.dtype(at::kFloat));
  check_rc(g_train.norm_forward(&k.n, out_ptr(r), out_ptr(h),
                                static_cast<float*>(out_ptr(inv)), current_stream(c.y)));
  return {r, h, inv};
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const OptTensor& x, const at::Tensor& y,
                               const OptTensor& gate, const OptTensor& post, const OptTensor& gamma,
                               const OptTensor& next, double eps, bool want_r) {
    NormRows k;
    variable_list o = norm_forward({x, gate, post, gamma, next, y, eps, want_r}, k, true);
    ctx->set_materialize_grads(false);
    auto given = [](const OptTensor& t) { return t ? *t : at::Tensor(); };
    ctx->save_for_backward({k.x.t, k.y.t, k.gate.t, given(k.post), given(k.gamma), given(k.next),
                            o[2]});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["r"] = want_r;
    variable_list outs;
    if (want_r) outs.push_back(o[0]);
    if (o[1].defined()) outs.push_back(o[1]);
    return outs;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const bool want_r = ctx->saved_data["r"].toBool();
    NormRows k;
    k.y = rows_of(s[1]);
    if (s[0].defined()) k.x = rows_of(s[0]);
    if (s[2].defined()) k.gate = rows_of(s[2]);
    if (s[3].defined()) k.post = s[3];
    if (s[4].defined()) k.gamma = s[4];
    if (s[5].defined()) k.next = s[5];
    fill(k, ctx->saved_data["eps"].toDouble());
    const at::Tensor dr = want_r ? g[0] : at::Tensor();
    const at::Tensor dh = k.next ? g[want_r ? 1 : 0] : at::Tensor();
    variable_list d(8);
    if (!dr.defined() && !dh.defined()) return d;
    const at::Tensor& y = k.y.t;
    const c10::DeviceGuard guard(y.device());
    Rows drr, dhr;
    if (dr.defined()) drr = rows_of(dr);
    if (dh.defined()) dhr = rows_of(dh);
    size_t edge = 0;
    bool weights = false;
    for (int i = 0; i < 6; ++i) {   // arguments and saved tensors are in one order
      if (!s[i].defined()) continue;
      if (!ctx->needs_input_grad(edge++)) continue;
      d[i] = at::empty(s[i].sizes(), y.options());
      weights |= i >= 3;
    }
    if (!weights && !d[0].defined() && !d[1].defined() && !d[2].defined()) return d;
    const size_t nws = weights ? g_train.norm_workspace_bytes(k.n.T, k.n.d, k.n.dtype) : 0;
    at::Tensor ws;
    if (nws) ws = bytes_like(y, nws);
    check_rc(g_train.norm_backward(
        &k.n, static_cast<const float*>(out_ptr(s[6])), out_ptr(drr.t), drr.stride, out_ptr(dhr.t),
        dhr.stride, out_ptr(d[0]), out_ptr(d[1]), out_ptr(d[2]), out_ptr(d[3]), out_ptr(d[4]),
        out_ptr(d[5]), out_ptr(ws), nws, current_stream(y)));
    return once(std::move(d), kNorm);
  }
};

OptTensor opt_tensor(PyObject* o) { return o == Py_None ? OptTensor() : OptTensor(tensor(o)); }

// block_norm(x, y, gate, post_weight, gamma, next_weight (each None or a tensor), eps): (r, h);
// y None: r is not computed (it is x) and None comes back for it, h = x / rms(x) next_weight
PyObject* block_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (bad_args(n, 7, "block_norm")) return nullptr;
  OptTensor x = opt_tensor(a[0]), y = opt_tensor(a[1]);
  const OptTensor gate = opt_tensor(a[2]), post = opt_tensor(a[3]), gamma = opt_tensor(a[4]),
                  next = opt_tensor(a[5]);
  const double eps = PyFloat_AsDouble(a[6]);
  if (PyErr_Occurred()) return nullptr;
  TORCH_CHECK(x || y, kNorm, ": x or y expected");
  TORCH_CHECK(y || (!gate && !post && !gamma && next), kNorm,
              ": without y there is next_weight alone");
  const bool want_r = y.has_value();
  if (!y) std::swap(x, y);
  dtype_of(*y, kNorm);
  TORCH_CHECK(y->dim() >= 1, kNorm, ": (..., d) expected");
  const int64_t d = y->size(y->dim() - 1);
  TORCH_CHECK(d >= 1 && d <= 16384, kNorm, ": rows of ", d, " elements (1 to 16384)");
  TORCH_CHECK(eps >= 0 && std::isfinite((float)eps), kNorm, ": eps ", eps);
  for (const OptTensor* t : std::initializer_list<const OptTensor*>{&x, &gate}) {
    if (!*t) continue;
    TORCH_CHECK((*t)->sizes() == y->sizes(), kNorm, ": shapes ", (*t)->sizes(), " and ", y->sizes());
  }
  for (const OptTensor* t : {&post, &gamma, &next})
    if (*t)
      TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == d, kNorm, ": a weight of shape ",
                  (*t)->sizes(), " for rows of ", d);
  for (const OptTensor* t : std::initializer_list<const OptTensor*>{&x, &gate, &post, &gamma, &next}) {
    if (!*t) continue;
    TORCH_CHECK((*t)->scalar_type() == y->scalar_type(), kNorm, ": dtypes ", (*t)->scalar_type(),
                " and ", y->scalar_type());
    TORCH_CHECK((*t)->device() == y->device(), kNorm, ": tensors on ", (*t)->device(), " and ",
                y->device());
  }
  if (tangents_live())
    for (const OptTensor* t : std::initializer_list<const OptTensor*>{&x, &y, &gate, &post, &gamma, &next})
      if (*t) check_tangent(**t, kNorm);
  check_hip(*y, kNorm);
  at::Tensor r, h;
  {
    pybind11::gil_scoped_release nogil;
    if (wants_grad({&x, &y, &gate, &post, &gamma, &next})) {
      const c10::DeviceGuard guard(y->device());
      check_capture({&x, &y, &gate, &post, &gamma, &next}, kNorm);
      const variable_list o = BlockNorm::apply(x, *y, gate, post, gamma, next, eps, want_r);
      if (want_r) r = o[0];
      if (next) h = o.back();
    } else {
      NormRows k;
      const variable_list o = norm_forward({x, gate, post, gamma, next, *y, eps, want_r}, k, false);
      r = o[0];
      h = o[1];
    }
  }
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, r.defined() ? THPVariable_Wrap(r) : none());
  PyTuple_SET_ITEM(t, 1, h.defined() ? THPVariable_Wrap(h) : none());
  return t;
  END_HANDLE_TH_ERRORS
}

// ---- AdamW ---------------------------------------------------------------------

constexpr const char* kAdamw = "adamw_step";

std::vector<at::Tensor> tensors_of(PyObject* o, const char* what, size_t want) {
  if (!PyList_Check(o) && !PyTuple_Check(o))
    throw torch::TypeError(std::string(kAdamw) + ": a list of tensors expected for " + what);
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  TORCH_CHECK(want == (size_t)-1 || (size_t)n == want, kAdamw, ": ", n, " ", what, " for ", want,
              " parameters");
  std::vector<at::Tensor> v;
  v.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) v.push_back(tensor(PySequence_Fast_GET_ITEM(o, i)));
  return v;
}

// adamw(params, grads, m, v, m_scales or None, v_scales or None, step, its device tensor or
// None, lr, beta1, beta2, eps, weight_decay, seed)
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (bad_args(nargs, 14, "adamw")) return nullptr;
  const bool q8 = a[4] != Py_None;
  const std::vector<at::Tensor> p = tensors_of(a[0], "parameters", (size_t)-1);
  const size_t n = p.size();
  std::vector<at::Tensor> g = tensors_of(a[1], "gradients", n);
  const std::vector<at::Tensor> m = tensors_of(a[2], "first moments", n);
  const std::vector<at::Tensor> v = tensors_of(a[3], "second moments", n);
  std::vector<at::Tensor> ms, vs;
  if (q8) {
    ms = tensors_of(a[4], "scales of first moments", n);
    vs = tensors_of(a[5], "scales of second moments", n);
  }
  tmoe_adamw_step_args s{};
  double num[5];
  for (int i = 0; i < 5; ++i) {
    num[i] = PyFloat_AsDouble(a[8 + i]);
    if (PyErr_Occurred()) return nullptr;
  }
  s.lr = num[0]; s.beta1 = num[1]; s.beta2 = num[2]; s.eps = num[3]; s.weight_decay = num[4];
  s.seed = (uint32_t)PyLong_AsUnsignedLongMask(a[13]);
  if (PyErr_Occurred()) return nullptr;
  s.state_bits = q8 ? 8 : 32;
  if (n == 0) return none();
  const at::Device dev = p[0].device();
  const auto dt = p[0].scalar_type();
  s.dtype = dtype_of(p[0], kAdamw);
  OptTensor step_dev;
  if (a[7] != Py_None) {
    step_dev = tensor(a[7]);
    TORCH_CHECK(step_dev->scalar_type() == at::kLong && step_dev->numel() == 1 &&
                    step_dev->device() == dev,
                kAdamw, ": step: a number, or an int64 tensor of one value on the parameters' device");
  } else {
    s.step = integer(a[6]);
    TORCH_CHECK(s.step >= 1, kAdamw, ": step ", s.step, " (the first is 1)");
  }
  struct Span { uintptr_t at, end; };
  std::vector<Span> written, read;
  written.reserve(5 * n);
  read.reserve(n);
  auto span = [](const at::Tensor& t, std::vector<Span>& list) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    if (t.numel()) list.push_back({at, at + (uintptr_t)t.numel() * t.element_size()});
  };
  const bool tangents = tangents_live();
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor& q = p[i];
    TORCH_CHECK(q.scalar_type() == dt && g[i].scalar_type() == dt, kAdamw, ": tensor ", i,
                ": parameter of ", q.scalar_type(), ", gradient of ", g[i].scalar_type(),
                ", the first parameter of ", dt);
    TORCH_CHECK(g[i].layout() == at::kStrided && g[i].sizes() == q.sizes(), kAdamw, ": tensor ", i,
                ": parameter ", q.sizes(), ", gradient ", g[i].sizes(), " (sparse ones are refused)");
    TORCH_CHECK(q.is_non_overlapping_and_dense(), kAdamw, ": tensor ", i,
                ": its elements have gaps or overlap");
    const int64_t blocks = (q.numel() + 255) / 256;
    if (q8) {
      const auto ok = [](const at::Tensor& t, int64_t len) {
        return (t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte) &&
               t.numel() == len && t.is_contiguous();
      };
      const auto sc = [](const at::Tensor& t, int64_t len) {
        return t.scalar_type() == at::kFloat && t.numel() == len && t.is_contiguous();
      };
      TORCH_CHECK(ok(m[i], q.numel()) && ok(v[i], q.numel()), kAdamw, ": tensor ", i,
                  ": states of ", q.numel(), " contiguous float8_e4m3fn (or uint8) codes expected");
      TORCH_CHECK(sc(ms[i], blocks) && sc(vs[i], blocks), kAdamw, ": tensor ", i, ": ", blocks,
                  " contiguous float32 scales expected");
      TORCH_CHECK(ms[i].device() == dev && vs[i].device() == dev, kAdamw, ": tensor ", i,
                  ": not all on ", dev);
    } else {
      for (const at::Tensor* t : {&m[i], &v[i]})
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->sizes() == q.sizes() &&
                        t->strides() == q.strides(),
                    kAdamw, ": tensor ", i, ": moments of float32 laid out as the parameter expected");
    }
    TORCH_CHECK(q.device() == dev && g[i].device() == dev && m[i].device() == dev &&
                    v[i].device() == dev,
                kAdamw, ": tensor ", i, ": not all on ", dev);
    if (tangents)
      for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &g[i], &m[i], &v[i]})
        check_tangent(*t, kAdamw);
    const size_t first = written.size();
    for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &m[i], &v[i]}) span(*t, written);
    // a gradient that the kernels read where it lies (one in another order is copied first);
    // the very elements that its own thread writes it may be
    if (g[i].strides() == q.strides()) {
      span(g[i], read);
      for (size_t j = first; j < written.size(); ++j)
        if (written[j].at == read.back().at && written[j].end == read.back().end) {
          read.pop_back();
          break;
        }
    }
    if (q8) {
      span(ms[i], written);
      span(vs[i], written);
    }
  }
  std::sort(written.begin(), written.end(), [](Span x, Span y) { return x.at < y.at; });
  for (size_t i = 1; i < written.size(); ++i)
    TORCH_CHECK(written[i - 1].end <= written[i].at, kAdamw,
                ": two of the parameters and states share memory");
  for (const Span& r : read) {      // the last written one that begins before r ends
    const auto w = std::lower_bound(written.begin(), written.end(), r.end,
                                    [](const Span& x, uintptr_t end) { return x.at < end; });
    TORCH_CHECK(w == written.begin() || (w - 1)->end <= r.at, kAdamw,
                ": a gradient shares memory with another element's parameter or state");
  }
  check_hip(p[0], kAdamw);
  {
    pybind11::gil_scoped_release nogil;
    const c10::DeviceGuard guard(dev);
    const at::AutoDispatchBelowADInplaceOrView below;
    std::vector<tmoe_adamw_tensor> t(n);
    for (size_t i = 0; i < n; ++i) {
      if (g[i].strides() != p[i].strides()) {
        at::Tensor same = at::empty_like(p[i]);     // the parameter's order of elements
        same.copy_(g[i]);
        g[i] = same;
      }
      t[i].p = p[i].data_ptr();
      t[i].g = g[i].const_data_ptr();
      t[i].m = m[i].data_ptr();
      t[i].v = v[i].data_ptr();
      t[i].m_scale = q8 ? static_cast<float*>(ms[i].data_ptr()) : nullptr;
      t[i].v_scale = q8 ? static_cast<float*>(vs[i].data_ptr()) : nullptr;
      t[i].n = p[i].numel();
    }
    s.step_dev = step_dev ? step_dev->const_data_ptr<int64_t>() : nullptr;
    check_rc(g_train.adamw_step(t.data(), (int64_t)n, &s, current_stream(p[0])));
    // what a graph saved of a parameter before this step is not its value any more
    const std::vector<at::Tensor>* const lists[] = {&p, &m, &v, &ms, &vs};
    for (const auto* list : lists)
      for (const at::Tensor& q : *list)
        if (!q.is_inference()) q.unsafeGetTensorImpl()->bump_version();
  }
  return none();
  END_HANDLE_TH_ERRORS
}

}  // namespace
