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
  decltype(&tmoe_fp8_quantize) fp8_quantize;
  decltype(&tmoe_fp8_gemm_workspace_bytes) fp8_workspace_bytes;
  decltype(&tmoe_fp8_gemm) fp8_gemm;
  decltype(&tmoe_fp8_gemm_values) fp8_gemm_values;
  decltype(&tmoe_muon_workspace_bytes) muon_workspace_bytes;
  decltype(&tmoe_muon_step) muon_step;
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
    variable_list kept{raw.is_same(c.raw) ? raw : c.raw, o[0].detach(), o[1].detach()};
    if (c.mask) kept.push_back(*c.mask);
    ctx->save_for_backward(std::move(kept));
    // (one number: each entry of saved_data costs a string and a node)
    ctx->saved_data["form"] = (int64_t)(c.k << 34 | c.score << 33 | (int64_t)c.renormalize << 32 |
                                        (int64_t)c10::bit_cast<uint32_t>((float)c.scale));
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[1].defined()) return {at::Tensor(), at::Tensor()};
    const variable_list s = ctx->get_saved_variables();
    ExpertRouterCall c;
    c.raw = s[0];
    if (s.size() > 3) c.mask = s[3];
    const int64_t form = ctx->saved_data["form"].toInt();
    c.k = form >> 34;
    c.score = form >> 33 & 1;
    c.renormalize = form >> 32 & 1;
    c.scale = c10::bit_cast<float>((uint32_t)form);
    const c10::DeviceGuard guard(c.raw.device());
    const tmoe_expert_router r = c.args();
    const at::Tensor dw = g[1].contiguous();
    at::Tensor draw = at::empty({r.B, r.E}, c.raw.options());
    check_rc(g_step.expert_router_backward(&r, s[1].const_data_ptr<int64_t>(), s[2].const_data_ptr<float>(),
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

// ---- 8-bit block products ----------------------------------------------------------

constexpr int64_t kFp8Most = (int64_t)1 << 23;
int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// codes (rows, K padded to 128) and scales (rows, or 128 of them, blocks)
struct Fp8 {
  at::Tensor codes, scales;
  bool tiles = false;
  tmoe_fp8_operand args() const {
    tmoe_fp8_operand o{};
    o.codes = codes.data_ptr();
    o.scales = scales.data_ptr<float>();
    o.rows = codes.size(0);
    o.row_bytes = codes.size(0) > 1 ? codes.stride(0) : codes.size(1);
    o.scale_row = scales.stride(0);
    o.scale_block = scales.stride(1);
    o.tiles = tiles;
    return o;
  }
};
// The operand of `rows` rows of K; scales of single rows lie row by row within a block, so that
// the rows of a tile read them side by side.
Fp8 fp8_empty(const at::Tensor& like, int64_t rows, int64_t K, bool tiles) {
  const auto o = like.options().requires_grad(false);
  Fp8 q;
  q.tiles = tiles;
  q.codes = at::empty({rows, 128 * blocks_of(K)}, o.dtype(at::kFloat8_e4m3fn));
  q.scales = tiles ? at::empty({blocks_of(rows), blocks_of(K)}, o.dtype(at::kFloat))
                   : at::empty({blocks_of(K), rows}, o.dtype(at::kFloat)).t();
  return q;
}
int32_t code_of(at::ScalarType t) { return t == at::kBFloat16 ? TMOE_BF16 : TMOE_F32; }
// x (its rows (R, C) at one stride) along its rows, its columns, or both
void fp8_quantize_into(const Rows& x, int64_t R, int64_t C, const tmoe_fp8_operand* rows,
                       const tmoe_fp8_operand* cols) {
  check_rc(g_step.fp8_quantize(x.t.const_data_ptr(), R, C, x.stride, code_of(x.t.scalar_type()), rows, cols,
                               current_stream(x.t)));
}
// out (M, N) = a b^T, of codes, or of the rows of values x
void fp8_gemm_into(const tmoe_fp8_operand* a, const Rows* x, int64_t M, const tmoe_fp8_operand& b, int64_t K,
                   const at::Tensor& out, void* ws, size_t nws) {
  const int dt = code_of(out.scalar_type());
  if (a) check_rc(g_step.fp8_gemm(a, &b, K, dt, out.data_ptr(), ws, nws, current_stream(out)));
  else check_rc(g_step.fp8_gemm_values(x->t.const_data_ptr(), M, x->stride, code_of(x->t.scalar_type()), &b, K, dt,
                                       out.data_ptr(), ws, nws, current_stream(out)));
}
at::Tensor fp8_product(const Fp8* a, const Rows* x, int64_t M, const Fp8& b, int64_t K, at::ScalarType dt) {
  const int64_t N = b.codes.size(0);
  at::Tensor out = at::empty({M, N}, b.codes.options().dtype(dt));
  if (M == 0) return out;
  const size_t nws = g_step.fp8_workspace_bytes(M, N, K, code_of(dt), !a);
  at::Tensor ws;
  if (nws) ws = bytes_like(out, nws);
  const tmoe_fp8_operand l = a ? a->args() : tmoe_fp8_operand{};
  fp8_gemm_into(a ? &l : nullptr, x, M, b.args(), K, out, out_ptr(ws), nws);
  return out;
}

PyObject* fp8_pair(const Fp8& q) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(q.codes));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(q.scales));
  return t;
}

// fp8_quantize(x, transpose, tiles): (codes, scales)
PyObject* fp8_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr const char* kWho = "fp8_quantize";
  HANDLE_TH_ERRORS
  if (bad_args(n, 3, "fp8_quantize")) return nullptr;
  const at::Tensor& x = tensor(a[0]);
  const bool transpose = PyObject_IsTrue(a[1]), tiles = PyObject_IsTrue(a[2]);
  dtype_of(x, kWho);
  TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1, kWho, ": (R, C) expected, got ", x.sizes());
  TORCH_CHECK(x.size(0) <= kFp8Most && x.size(1) <= kFp8Most, kWho, ": at most 2^23 rows and columns, got ",
              x.sizes());
  TORCH_CHECK(!transpose || x.size(0) >= 1, kWho, ": no rows to lie along");
  if (tangents_live()) check_tangent(x, kWho);
  TORCH_CHECK(!(at::GradMode::is_enabled() && x.requires_grad()), kWho,
              " has no gradient: give it detached, or call fp8_matmul");
  check_hip(x, kWho);
  Fp8 q;
  {
    pybind11::gil_scoped_release nogil;
    const c10::DeviceGuard guard(x.device());
    const at::NoGradGuard no_grad;
    const int64_t R = x.size(0), C = x.size(1);
    q = transpose ? fp8_empty(x, C, R, tiles) : fp8_empty(x, R, C, tiles);
    if (R) {
      const tmoe_fp8_operand o = q.args();
      fp8_quantize_into(rows_of(x), R, C, transpose ? nullptr : &o, transpose ? &o : nullptr);
    }
  }
  return fp8_pair(q);
  END_HANDLE_TH_ERRORS
}

Fp8 fp8_operand(PyObject* codes, PyObject* scales, int64_t K, const char* who) {
  Fp8 q;
  q.codes = tensor(codes);
  q.scales = tensor(scales);
  const at::Tensor &c = q.codes, &s = q.scales;
  TORCH_CHECK((c.scalar_type() == at::kFloat8_e4m3fn || c.scalar_type() == at::kByte) && c.dim() == 2 &&
                  K >= 1 && c.size(1) == 128 * blocks_of(K),
              who, ": codes (rows, ", K, " padded to a multiple of 128) of float8_e4m3fn (or uint8) expected, got ",
              c.sizes(), " of ", c.scalar_type());
  const int64_t rows = c.size(0);
  TORCH_CHECK(rows <= kFp8Most && K <= kFp8Most, who, ": at most 2^23 rows and columns, got ", c.sizes());
  TORCH_CHECK(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(1) == blocks_of(K) &&
                  (s.size(0) == rows || s.size(0) == blocks_of(rows)),
              who, ": scales of float32 for each row or each 128 of ", rows, " and each of ", blocks_of(K),
              " blocks expected, got ", s.sizes(), " of ", s.scalar_type());
  TORCH_CHECK(c.device() == s.device(), who, ": codes on ", c.device(), ", scales on ", s.device());
  TORCH_CHECK(!s.requires_grad(), who, ": scales get no gradient: give them detached");
  q.tiles = s.size(0) != rows;
  return q;
}
void fp8_align(Fp8& q) {     // rows that direct loads of 16 bytes can read
  const at::Tensor& c = q.codes;
  if (c.size(0) == 0) return;
  const bool ok = c.stride(1) == 1 && reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0 &&
                  (c.size(0) == 1 || (c.stride(0) % 16 == 0 && c.stride(0) >= c.size(1) &&
                                      c.stride(0) <= 2 * kFp8Most));
  if (!ok) q.codes = c.clone(at::MemoryFormat::Contiguous);
}

// fp8_block_matmul(a codes or values, a scales or None, K, b codes, b scales, out dtype is bf16):
// out (..., N)
PyObject* fp8_block_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr const char* kWho = "fp8_block_matmul";
  HANDLE_TH_ERRORS
  if (bad_args(n, 6, "fp8_block_matmul")) return nullptr;
  const int64_t K = integer(a[2]);
  const at::ScalarType dt = PyObject_IsTrue(a[5]) ? at::kBFloat16 : at::kFloat;
  Fp8 b = fp8_operand(a[3], a[4], K, kWho);
  TORCH_CHECK(b.codes.size(0) >= 1, kWho, ": b of no rows");
  const at::Tensor& x = tensor(a[0]);
  TORCH_CHECK(x.device() == b.codes.device(), kWho, ": operands on ", x.device(), " and ", b.codes.device());
  at::Tensor out;
  if (a[1] != Py_None) {
    Fp8 q = fp8_operand(a[0], a[1], K, kWho);
    check_hip(x, kWho);
    pybind11::gil_scoped_release nogil;
    const c10::DeviceGuard guard(x.device());
    fp8_align(q);
    fp8_align(b);
    out = fp8_product(&q, nullptr, q.codes.size(0), b, K, dt);
  } else {
    dtype_of(x, kWho);
    TORCH_CHECK(x.dim() >= 1 && x.size(x.dim() - 1) == K, kWho, ": rows of ", K, " expected, got ", x.sizes());
    const int64_t M = x.numel() / K;
    TORCH_CHECK(M <= kFp8Most, kWho, ": at most 2^23 rows, got ", M);
    if (tangents_live()) check_tangent(x, kWho);
    TORCH_CHECK(!(at::GradMode::is_enabled() && x.requires_grad()), kWho,
                " has no gradient: give it detached, or call fp8_matmul");
    check_hip(x, kWho);
    pybind11::gil_scoped_release nogil;
    const c10::DeviceGuard guard(x.device());
    const at::NoGradGuard no_grad;
    fp8_align(b);
    const Rows rows = rows_of(x);
    out = fp8_product(nullptr, &rows, M, b, K, dt);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = b.codes.size(0);
    out = out.view(shape);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

constexpr const char* kFp8Matmul = "fp8_matmul";

// Operands that no caller sees lie in one byte tensor, codes and then scales: an allocation each,
// with views, took a fifth of a small layer's step on the host.
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
struct Fp8Place {
  int64_t rows = 0, K = 0, at = 0, scales_at = 0;
  bool tiles = false;
  // behind the `end` bytes that are taken
  Fp8Place(int64_t rows, int64_t K, bool tiles, int64_t& end) : rows(rows), K(K), at(end), tiles(tiles) {
    scales_at = at + up256(rows * 128 * blocks_of(K));
    end = scales_at + up256((tiles ? blocks_of(rows) : rows) * blocks_of(K) * 4);
  }
  tmoe_fp8_operand in(const at::Tensor& buf) const {
    char* p = static_cast<char*>(buf.data_ptr());
    tmoe_fp8_operand o{};
    o.codes = p + at;
    o.scales = reinterpret_cast<float*>(p + scales_at);
    o.rows = rows;
    o.row_bytes = 128 * blocks_of(K);
    o.scale_row = tiles ? blocks_of(K) : 1;
    o.scale_block = tiles ? 1 : rows;
    o.tiles = tiles;
    return o;
  }
};
struct Fp8Call {
  at::Tensor x, w;
  bool want_x = false, want_w = false;
};
// What the backward keeps: x^T (K, M) by rows for dw, w (K, N) by tiles for dx
struct Fp8Kept {
  int64_t end = 0;
  Fp8Place x, w;
  Fp8Kept(int64_t M, int64_t K, int64_t N, bool want_x, bool want_w)
      : x(want_w ? K : 0, M, false, end), w(want_x ? K : 0, N, true, end) {}
};
at::Tensor fp8_matmul_forward(const Fp8Call& c, at::Tensor* kept) {
  const c10::DeviceGuard guard(c.x.device());
  const int64_t K = c.w.size(0), N = c.w.size(1), M = c.x.numel() / K;
  const Rows x = rows_of(c.x);
  std::vector<int64_t> shape = c.x.sizes().vec();
  shape.back() = N;
  at::Tensor out = at::empty(shape, c.x.options().requires_grad(false));
  const Fp8Kept k(M, K, N, c.want_x, c.want_w);
  if (k.end) *kept = bytes_like(out, (size_t)k.end);
  const bool both = c.want_w && M > 0;            // x is quantised along both axes at once
  int64_t end = 0;
  const Fp8Place wt(N, K, true, end), xr(both ? M : 0, K, false, end);
  const size_t nws = M ? g_step.fp8_workspace_bytes(M, N, K, code_of(out.scalar_type()), !both) : 0;
  const at::Tensor tmp = bytes_like(out, (size_t)end + nws);
  tmoe_fp8_operand b = wt.in(tmp), w{};
  if (c.want_x) {
    w = k.w.in(*kept);
    b.scales = w.scales;
    b.scale_row = w.scale_block;
    b.scale_block = w.scale_row;
  }
  if (c.want_x || M > 0) fp8_quantize_into(rows_of(c.w), K, N, c.want_x ? &w : nullptr, &b);
  if (M == 0) return out;
  void* ws = nws ? static_cast<char*>(tmp.data_ptr()) + end : nullptr;
  if (both) {
    const tmoe_fp8_operand r = xr.in(tmp), t = k.x.in(*kept);
    fp8_quantize_into(x, M, K, &r, &t);
    fp8_gemm_into(&r, nullptr, M, b, K, out, ws, nws);
  } else {
    fp8_gemm_into(nullptr, &x, M, b, K, out, ws, nws);
  }
  return out;
}

struct Fp8Matmul : torch::autograd::Function<Fp8Matmul> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, Fp8Call c) {
    c.want_x = x.requires_grad();
    c.want_w = w.requires_grad();
    at::Tensor kept;
    const at::Tensor out = fp8_matmul_forward(c, &kept);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({kept});
    // (K and what was kept, in one number)
    ctx->saved_data["kept"] = w.size(0) * 4 + (c.want_x ? 2 : 0) + (c.want_w ? 1 : 0);
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    const variable_list s = ctx->get_saved_variables();
    const int64_t kept = ctx->saved_data["kept"].toInt(), K = kept >> 2;
    const at::Tensor& dy = g[0];
    const int64_t N = dy.size(-1), M = dy.numel() / N;
    const Fp8Kept k(M, K, N, kept & 2, kept & 1);
    const c10::DeviceGuard guard(dy.device());
    const Rows d = rows_of(dy);
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), both = want_w && M > 0;
    const int dt = code_of(dy.scalar_type());
    at::Tensor dx, dw;
    if (want_x) {
      std::vector<int64_t> shape = dy.sizes().vec();
      shape.back() = K;
      dx = at::empty(shape, dy.options());
    }
    if (want_w) dw = M ? at::empty({K, N}, dy.options()) : at::zeros({K, N}, dy.options());
    if (M > 0) {
      int64_t end = 0;
      const Fp8Place dr(both && want_x ? M : 0, N, false, end), dc(both ? N : 0, M, false, end);
      const size_t nx = want_x ? g_step.fp8_workspace_bytes(M, K, N, dt, !both) : 0;
      const size_t nw = want_w ? g_step.fp8_workspace_bytes(K, N, M, dt, 0) : 0;
      const int64_t room = end + (int64_t)std::max(nx, nw);
      at::Tensor tmp;
      if (room) tmp = bytes_like(dy, (size_t)room);
      void* ws = room > end ? static_cast<char*>(tmp.data_ptr()) + end : nullptr;
      tmoe_fp8_operand r{}, c{};
      if (both) {
        c = dc.in(tmp);
        if (want_x) r = dr.in(tmp);
        fp8_quantize_into(d, M, N, want_x ? &r : nullptr, &c);
        const tmoe_fp8_operand x = k.x.in(s[0]);
        fp8_gemm_into(&x, nullptr, K, c, M, dw, ws, nw);
      }
      if (want_x) fp8_gemm_into(both ? &r : nullptr, &d, M, k.w.in(s[0]), N, dx, ws, nx);
    }
    return once({dx, dw, at::Tensor()}, kFp8Matmul);
  }
};

// fp8_matmul(x, w): x w in 8-bit block products, with their gradients
PyObject* fp8_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (bad_args(n, 2, "fp8_matmul")) return nullptr;
  const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]);
  dtype_of(x, kFp8Matmul);
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), kFp8Matmul, ": dtypes ", x.scalar_type(), " and ",
              w.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && w.size(0) >= 1 && w.size(1) >= 1 &&
                  x.size(x.dim() - 1) == w.size(0),
              kFp8Matmul, ": (..., K) and (K, N) expected, got ", x.sizes(), " and ", w.sizes());
  TORCH_CHECK(x.numel() / w.size(0) <= kFp8Most && w.size(0) <= kFp8Most && w.size(1) <= kFp8Most, kFp8Matmul,
              ": at most 2^23 of each, got ", x.sizes(), " and ", w.sizes());
  TORCH_CHECK(x.device() == w.device(), kFp8Matmul, ": tensors on ", x.device(), " and ", w.device());
  if (tangents_live()) {
    check_tangent(x, kFp8Matmul);
    check_tangent(w, kFp8Matmul);
  }
  check_hip(x, kFp8Matmul);
  at::Tensor out;
  {
    pybind11::gil_scoped_release nogil;
    Fp8Call c{x, w};
    const OptTensor xo = x, wo = w;
    if (wants_grad({&xo, &wo})) {
      const c10::DeviceGuard guard(x.device());
      check_capture({&xo, &wo}, kFp8Matmul);
      out = Fp8Matmul::apply(x, w, c)[0];
    } else {
      const at::NoGradGuard no_grad;
      out = fp8_matmul_forward(c, nullptr);
    }
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- Muon ----------------------------------------------------------------------

// muon(params, grads, momenta or None, lr, momentum, weight_decay, update_rms, eps, coefficients (a,
// b, c), steps, nesterov, write only, check only): params None: a list of new tensors like grads. Check
// only: refuses what the call would refuse, and does nothing
PyObject* muon(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (bad_args(nargs, 13, "muon")) return nullptr;
  const bool write_only = a[0] == Py_None;
  const char* const who = write_only ? "orthogonalize" : "muon_step";
  auto list = [&](PyObject* o, const char* what, size_t want) {
    if (!PyList_Check(o) && !PyTuple_Check(o))
      throw torch::TypeError(std::string(who) + ": a list of tensors expected for " + what);
    const Py_ssize_t k = PySequence_Fast_GET_SIZE(o);
    TORCH_CHECK(want == (size_t)-1 || (size_t)k == want, who, ": ", k, " ", what, " for ", want, " gradients");
    std::vector<at::Tensor> v;
    v.reserve(k);
    for (Py_ssize_t i = 0; i < k; ++i) v.push_back(tensor(PySequence_Fast_GET_ITEM(o, i)));
    return v;
  };
  std::vector<at::Tensor> g = list(a[1], "gradients", (size_t)-1);
  const size_t n = g.size();
  std::vector<at::Tensor> p, m;
  if (!write_only) {
    p = list(a[0], "parameters", n);
    m = list(a[2], "momenta", n);
  }
  tmoe_muon_step_args s{};
  double num[5];
  for (int i = 0; i < 5; ++i) num[i] = PyFloat_AsDouble(a[3 + i]);
  if (PyErr_Occurred()) return nullptr;
  s.lr = num[0]; s.momentum = num[1]; s.weight_decay = num[2]; s.update_rms = num[3]; s.eps = num[4];
  if (!PyTuple_Check(a[8]) || PyTuple_GET_SIZE(a[8]) != 3)
    throw torch::TypeError(std::string(who) + ": three coefficients expected");
  for (int i = 0; i < 3; ++i) s.coefficients[i] = PyFloat_AsDouble(PyTuple_GET_ITEM(a[8], i));
  if (PyErr_Occurred()) return nullptr;
  const int64_t steps = integer(a[9]);
  TORCH_CHECK(steps >= 1 && steps <= 16, who, ": steps ", steps, " (1 to 16)");
  s.steps = (int32_t)steps;
  s.nesterov = PyObject_IsTrue(a[10]);
  s.write_only = write_only;
  const bool check_only = PyObject_IsTrue(a[12]);
  s.dtype = TMOE_F32;
  if (n == 0 || check_only) check_rc(g_step.muon_step(nullptr, 0, &s, nullptr, 0, nullptr));   // the numbers alone
  if (n == 0) return PyList_New(0);
  const at::Device dev = g[0].device();
  const auto dt = g[0].scalar_type();
  s.dtype = dtype_of(g[0], who);
  struct Span { uintptr_t at, end; };
  std::vector<Span> written, read;
  auto span = [](const at::Tensor& t, std::vector<Span>& to) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    if (t.numel()) to.push_back({at, at + (uintptr_t)t.numel() * t.element_size()});
  };
  const bool tangents = tangents_live();
  std::vector<tmoe_muon_tensor> t(n);
  for (size_t i = 0; i < n; ++i) {
    TORCH_CHECK(g[i].layout() == at::kStrided, who, ": tensor ", i, ": sparse gradients are refused");
    TORCH_CHECK(g[i].scalar_type() == dt, who, ": tensor ", i, " of ", g[i].scalar_type(), ", the first of ", dt);
    TORCH_CHECK(g[i].dim() >= 2, who, ": tensor ", i, ": matrices (..., rows, cols) expected, got ", g[i].sizes());
    TORCH_CHECK(g[i].device() == dev, who, ": tensor ", i, ": not all on ", dev);
    const int64_t rows = g[i].size(-2), cols = g[i].size(-1);
    TORCH_CHECK(std::max(rows, cols) <= (int64_t)1 << 22 && std::min(rows, cols) <= 65536, who, ": tensor ", i,
                ": matrices of ", rows, " x ", cols, " (at most 2^22, the smaller side 65536)");
    t[i].rows = rows;
    t[i].cols = cols;
    t[i].batch = rows && cols ? g[i].numel() / (rows * cols) : 0;
    if (tangents) check_tangent(g[i], who);
    if (write_only) continue;
    const at::Tensor& q = p[i];
    TORCH_CHECK(q.scalar_type() == dt && q.sizes() == g[i].sizes(), who, ": tensor ", i, ": parameter ", q.sizes(),
                " of ", q.scalar_type(), ", gradient ", g[i].sizes(), " of ", dt);
    TORCH_CHECK(m[i].scalar_type() == at::kFloat && m[i].sizes() == q.sizes(), who, ": tensor ", i,
                ": momentum of float32 in the parameter's shape expected, got ", m[i].sizes(), " of ",
                m[i].scalar_type());
    TORCH_CHECK(q.is_contiguous() && m[i].is_contiguous(), who, ": tensor ", i,
                ": contiguous parameters and momenta expected");
    TORCH_CHECK(q.device() == dev && m[i].device() == dev, who, ": tensor ", i, ": not all on ", dev);
    if (tangents) {
      check_tangent(q, who);
      check_tangent(m[i], who);
    }
    span(q, written);
    span(m[i], written);
    if (g[i].is_contiguous()) span(g[i], read);
  }
  std::sort(written.begin(), written.end(), [](Span x, Span y) { return x.at < y.at; });
  for (size_t i = 1; i < written.size(); ++i)
    TORCH_CHECK(written[i - 1].end <= written[i].at, who, ": two of the parameters and momenta share memory");
  for (const Span& r : read) {      // the last written one that begins before r ends
    const auto w = std::lower_bound(written.begin(), written.end(), r.end,
                                    [](const Span& x, uintptr_t end) { return x.at < end; });
    TORCH_CHECK(w == written.begin() || (w - 1)->end <= r.at, who,
                ": a gradient shares memory with a parameter or momentum");
  }
  TORCH_CHECK(!(write_only && at::GradMode::is_enabled() &&
                std::any_of(g.begin(), g.end(), [](const at::Tensor& x) { return x.requires_grad(); })),
              who, " has no gradient: give the matrices detached");
  check_hip(g[0], who);
  if (check_only) return none();
  {
    pybind11::gil_scoped_release nogil;
    const c10::DeviceGuard guard(dev);
    const at::AutoDispatchBelowADInplaceOrView below;
    for (size_t i = 0; i < n; ++i) {
      g[i] = g[i].contiguous();
      if (write_only) p.push_back(at::empty(g[i].sizes(), g[i].options().requires_grad(false)));
      t[i].p = p[i].data_ptr();
      t[i].g = g[i].const_data_ptr();
      t[i].m = write_only ? nullptr : m[i].data_ptr<float>();
    }
    const size_t nws = g_step.muon_workspace_bytes(t.data(), (int64_t)n);
    at::Tensor ws;
    if (nws) ws = bytes_like(g[0], nws);
    check_rc(g_step.muon_step(t.data(), (int64_t)n, &s, out_ptr(ws), nws, current_stream(g[0])));
    // what a graph saved of a parameter before this step is not its value any more
    if (!write_only)
      for (const auto* each : {&p, &m})
        for (const at::Tensor& q : *each)
          if (!q.is_inference()) q.unsafeGetTensorImpl()->bump_version();
  }
  if (!write_only) return none();
  PyObject* out = PyList_New((Py_ssize_t)n);
  if (!out) return nullptr;
  for (size_t i = 0; i < n; ++i) PyList_SET_ITEM(out, (Py_ssize_t)i, THPVariable_Wrap(p[i]));
  return out;
  END_HANDLE_TH_ERRORS
}

}  // namespace
