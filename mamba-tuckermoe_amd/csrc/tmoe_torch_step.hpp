// The wider training operators' host side in native code: autograd functions over the C ABI's
// expert router and 8-bit products, and the Muon step's lists of tensors. Included by
// tmoe_torch.cpp after tmoe_torch_train.hpp, whose conventions hold here too.
#pragma once

#include "tmoe.h"

namespace {

struct StepEntry {
  decltype(&tmoe_expert_router_workspace_bytes) expert_router_workspace_bytes;
  decltype(&tmoe_expert_router_forward) expert_router_forward;
  decltype(&tmoe_expert_router_backward) expert_router_backward;
} g_step{};

// ---- expert router ---------------------------------------------------------------

constexpr const char* kExpertRouter = "fused_expert_router";

struct ExpertRouterCall {
  at::Tensor raw;
  OptTensor bias, mask;
  int64_t k = 0, groups = 1, top_groups = 1, score = 0;
  double scale = 1;
  bool renormalize = true;
  tmoe_expert_router args() const {
    tmoe_expert_router r{};
    r.raw = raw.const_data_ptr();
    r.B = raw.size(0);
    r.E = raw.size(1);
    r.row_stride = r.B > 1 ? raw.stride(0) : r.E;
    r.k = k;
    r.groups = groups;
    r.top_groups = top_groups;
    r.bias = static_cast<const float*>(ptr_of(bias));
    r.mask = static_cast<const uint8_t*>(ptr_of(mask));
    r.dtype = raw.scalar_type() == at::kBFloat16 ? TMOE_BF16 : TMOE_F32;
    r.score = (int32_t)score;
    r.renormalize = renormalize;
    r.scale = (float)scale;
    return r;
  }
};

// idx, w, counts
variable_list expert_router_forward(const ExpertRouterCall& c) {
  const c10::DeviceGuard guard(c.raw.device());
  const tmoe_expert_router r = c.args();
  const auto o = c.raw.options();
  at::Tensor idx = at::empty({r.B, r.k}, o.dtype(at::kLong));
  at::Tensor w = at::empty({r.B, r.k}, o.dtype(at::kFloat));
  at::Tensor counts = at::empty({r.E}, o.dtype(at::kLong));
  const size_t nws = g_step.expert_router_workspace_bytes(r.B, r.E);
  at::Tensor ws = bytes_like(c.raw, nws);
  check_rc(g_step.expert_router_forward(&r, idx.data_ptr<int64_t>(), w.data_ptr<float>(),
                                        counts.data_ptr<int64_t>(), ws.data_ptr(), nws,
                                        current_stream(c.raw)));
  return {idx, w, counts};
}

struct ExpertRouter : torch::autograd::Function<ExpertRouter> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& raw, ExpertRouterCall c) {
    variable_list o = expert_router_forward(c);
    ctx->mark_non_differentiable({o[0], o[2]});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({raw.is_same(c.raw) ? raw : c.raw, c.mask.value_or(at::Tensor()), o[0], o[1]});
    ctx->saved_data["k"] = c.k;
    ctx->saved_data["score"] = c.score;
    ctx->saved_data["scale"] = c.scale;
    ctx->saved_data["renormalize"] = c.renormalize;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[1].defined()) return {at::Tensor(), at::Tensor()};
    const variable_list s = ctx->get_saved_variables();
    ExpertRouterCall c;
    c.raw = s[0];
    if (s[1].defined()) c.mask = s[1];
    c.k = ctx->saved_data["k"].toInt();
    c.score = ctx->saved_data["score"].toInt();
    c.scale = ctx->saved_data["scale"].toDouble();
    c.renormalize = ctx->saved_data["renormalize"].toBool();
    const c10::DeviceGuard guard(c.raw.device());
    const tmoe_expert_router r = c.args();
    const at::Tensor dw = g[1].contiguous();
    at::Tensor draw = at::empty({r.B, r.E}, c.raw.options());
    check_rc(g_step.expert_router_backward(&r, s[2].const_data_ptr<int64_t>(), s[3].const_data_ptr<float>(),
                                           dw.const_data_ptr<float>(), draw.data_ptr(),
                                           current_stream(c.raw)));
    return once({draw, at::Tensor()}, kExpertRouter);
  }
};

// expert_router(raw, k, sigmoid, bias or None, groups, top_groups, renormalize, scale, mask or None):
// (idx, w, counts)
PyObject* expert_router(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (bad_args(n, 9, "expert_router")) return nullptr;
  const at::Tensor& raw = tensor(a[0]);
  ExpertRouterCall c;
  c.k = integer(a[1]);
  c.score = PyObject_IsTrue(a[2]) ? TMOE_SCORE_SIGMOID : TMOE_SCORE_SOFTMAX;
  c.bias = opt_tensor(a[3]);
  c.groups = integer(a[4]);
  c.top_groups = integer(a[5]);
  c.renormalize = PyObject_IsTrue(a[6]);
  c.scale = PyFloat_AsDouble(a[7]);
  if (PyErr_Occurred()) return nullptr;
  dtype_of(raw, kExpertRouter);
  TORCH_CHECK(raw.dim() == 2, kExpertRouter, ": raw logits (B, E) expected, got ", raw.sizes());
  const int64_t E = raw.size(1);
  TORCH_CHECK(E >= 1 && E <= 256 && c.k >= 1 && c.k <= 16, kExpertRouter,
              ": 1 to 256 experts and top_k 1 to 16, got ", E, " and ", c.k);
  TORCH_CHECK(c.groups >= 1 && c.groups <= E && E % c.groups == 0 && c.top_groups >= 1 &&
                  c.top_groups <= c.groups,
              kExpertRouter, ": ", c.top_groups, " of ", c.groups, " groups of ", E, " experts");
  TORCH_CHECK(c.k <= c.top_groups * (E / c.groups), kExpertRouter, ": top_k ", c.k, " of the ",
              c.top_groups * (E / c.groups), " experts of the open groups");
  TORCH_CHECK((float)c.scale > 0 && std::isfinite((float)c.scale), kExpertRouter, ": scale ", c.scale);
  if (c.bias) {
    const at::Tensor& t = *c.bias;
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == E, kExpertRouter, ": bias (",
                E, ") of float32 expected, got ", t.sizes(), " of ", t.scalar_type());
    TORCH_CHECK(!t.requires_grad(), kExpertRouter, ": the bias gets no gradient: give it detached");
    TORCH_CHECK(t.device() == raw.device(), kExpertRouter, ": bias on ", t.device(), ", logits on ",
                raw.device());
    c.bias = t.contiguous();
  }
  if (a[8] != Py_None) {
    const at::Tensor& m = tensor(a[8]);
    TORCH_CHECK(m.scalar_type() == at::kBool && m.dim() == 1 && m.size(0) == raw.size(0), kExpertRouter,
                ": mask (", raw.size(0), ") of bool expected, got ", m.sizes(), " of ", m.scalar_type());
    TORCH_CHECK(m.device() == raw.device(), kExpertRouter, ": mask on ", m.device(), ", logits on ",
                raw.device());
    c.mask = m.contiguous();
  }
  if (tangents_live()) check_tangent(raw, kExpertRouter);
  check_hip(raw, kExpertRouter);
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
      check_capture({&leaf}, kExpertRouter);
      o = ExpertRouter::apply(raw, c);
    } else {
      o = expert_router_forward(c);
    }
  }
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(o[i]));
  return r;
  END_HANDLE_TH_ERRORS
}

}  // namespace
