// The C ABI's entry points of the training layer's wider operators (include/tmoe.h:
// tmoe_expert_router_*, tmoe_fp8_*, tmoe_muon_*): argument checks on the host before the first
// HIP call, then the launchers of tmoe_step.h.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "tmoe.h"
#include "tmoe_step.h"
#include "tmoe_train.h"

namespace {

int fail(int code, const char* fmt, ...) {
  char text[384];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  return tmoe::fail_text(code, text);
}
int done(hipError_t e, const char* who) {
  return e == hipSuccess ? TMOE_OK : fail(TMOE_EHIP, "%s: %s", who, hipGetErrorString(e));
}
bool on(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool dtype_ok(int dtype) { return dtype == TMOE_BF16 || dtype == TMOE_F32; }
size_t size_of(int dtype) { return dtype == TMOE_BF16 ? 2 : 4; }

constexpr int64_t kMaxRows = (int64_t)1 << 30;

int er_check(const char* who, const tmoe_expert_router* r) {
  if (!r) return fail(TMOE_EINVAL, "%s: null router", who);
  if (!dtype_ok(r->dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d is not TMOE_BF16 or TMOE_F32", who, (int)r->dtype);
  if (r->score != TMOE_SCORE_SOFTMAX && r->score != TMOE_SCORE_SIGMOID)
    return fail(TMOE_EINVAL, "%s: score %d", who, (int)r->score);
  if (r->B < 0 || r->E < 1 || r->k < 1)
    return fail(TMOE_EINVAL, "%s: B=%lld E=%lld k=%lld", who, (long long)r->B, (long long)r->E,
                (long long)r->k);
  if (r->E > tmoe::kRouterMaxE || r->k > tmoe::kRouterMaxK || r->B > kMaxRows)
    return fail(TMOE_EUNSUPPORTED, "%s: B=%lld E=%lld k=%lld (at most 2^30, 256, 16)", who,
                (long long)r->B, (long long)r->E, (long long)r->k);
  if (r->groups < 1 || r->groups > r->E || r->E % r->groups || r->top_groups < 1 ||
      r->top_groups > r->groups)
    return fail(TMOE_EINVAL, "%s: %lld of %lld groups of %lld experts", who, (long long)r->top_groups,
                (long long)r->groups, (long long)r->E);
  if (r->k > r->top_groups * (r->E / r->groups))
    return fail(TMOE_EINVAL, "%s: k=%lld of the %lld experts of the open groups", who, (long long)r->k,
                (long long)(r->top_groups * (r->E / r->groups)));
  if (!(r->scale > 0.f) || !isfinite(r->scale))
    return fail(TMOE_EINVAL, "%s: scale must be positive and finite", who);
  if (r->B > 0 && !r->raw) return fail(TMOE_EINVAL, "%s: null raw", who);
  if (r->row_stride < (r->B > 1 ? r->E : 0))
    return fail(TMOE_EINVAL, "%s: row_stride %lld", who, (long long)r->row_stride);
  if (!on(r->raw, size_of(r->dtype)) || !on(r->bias, 4))
    return fail(TMOE_EINVAL, "%s: misaligned raw or bias", who);
  return TMOE_OK;
}
tmoe::ExpertRouterArgs er_args(const tmoe_expert_router* r) {
  tmoe::ExpertRouterArgs a{};
  a.raw = r->raw; a.row_stride = r->row_stride; a.B = r->B;
  a.E = (int)r->E; a.k = (int)r->k; a.groups = (int)r->groups; a.top_groups = (int)r->top_groups;
  a.dtype = r->dtype; a.score = r->score; a.renormalize = r->renormalize != 0; a.scale = r->scale;
  a.bias = r->bias; a.mask = r->mask;
  return a;
}

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// an operand of `rows` rows of K elements
int fp8_check(const char* who, const char* what, const tmoe_fp8_operand* o, int64_t rows, int64_t K) {
  if (!o) return fail(TMOE_EINVAL, "%s: null %s", who, what);
  if (rows < 0 || o->rows != rows || K < 1)
    return fail(TMOE_EINVAL, "%s: %s of %lld rows of %lld", who, what, (long long)o->rows, (long long)K);
  if (rows > tmoe::kFp8MaxDim || K > tmoe::kFp8MaxDim)
    return fail(TMOE_EUNSUPPORTED, "%s: %s of %lld rows of %lld (at most 2^23)", who, what,
                (long long)rows, (long long)K);
  if (rows == 0) return TMOE_OK;
  if (!o->codes || !o->scales) return fail(TMOE_EINVAL, "%s: null pointer in %s", who, what);
  if (!on(o->codes, 16) || !on(o->scales, 4))
    return fail(TMOE_EINVAL, "%s: misaligned pointer in %s", who, what);
  if (o->row_bytes % 16 || o->row_bytes < blocks_of(K) * 128 || o->row_bytes > 2 * tmoe::kFp8MaxDim)
    return fail(TMOE_EINVAL, "%s: %s of rows %lld bytes apart", who, what, (long long)o->row_bytes);
  if (o->scale_row < 0 || o->scale_block < 0)
    return fail(TMOE_EINVAL, "%s: negative steps of scales in %s", who, what);
  return TMOE_OK;
}
struct Fp8Workspace {
  size_t planes, codes, scales, total;
};
Fp8Workspace fp8_workspace(int64_t M, int64_t N, int64_t K, bool values, int dtype) {
  Fp8Workspace w{};
  w.planes = (size_t)up16((int64_t)tmoe::fp8_gemm_workspace_bytes(M, N, blocks_of(K), dtype));
  if (values && !tmoe::fp8_gemm_takes_values(M, blocks_of(K))) {
    w.codes = (size_t)(M * blocks_of(K) * 128);
    w.scales = (size_t)up16(M * blocks_of(K) * 4);
  }
  w.total = w.planes + w.codes + w.scales;
  return w;
}
bool fp8_sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && N >= 1 && K >= 1 && M <= tmoe::kFp8MaxDim && N <= tmoe::kFp8MaxDim &&
         K <= tmoe::kFp8MaxDim;
}
int fp8_gemm_check(const char* who, int64_t M, const tmoe_fp8_operand* b, int64_t K, int dtype,
                   const void* out, const void* ws, size_t bytes, size_t need) {
  if (!dtype_ok(dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d is not TMOE_BF16 or TMOE_F32", who, dtype);
  if (b->rows < 1) return fail(TMOE_EINVAL, "%s: b of no rows", who);
  if (M > 0 && !out) return fail(TMOE_EINVAL, "%s: null out", who);
  if (!on(out, 16) || !on(ws, 16)) return fail(TMOE_EINVAL, "%s: misaligned out or workspace", who);
  if (need && (!ws || bytes < need))
    return fail(TMOE_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, bytes, need);
  return TMOE_OK;
}
void fp8_b(tmoe::Fp8GemmArgs& g, const tmoe_fp8_operand* b, int64_t K, int dtype, void* out) {
  g.b = b->codes; g.b_bytes = b->row_bytes; g.sb = b->scales;
  g.sb_rs = b->scale_row; g.sb_ks = b->scale_block; g.b_tiles = b->tiles != 0;
  g.N = b->rows; g.K = K; g.blocks = (int)blocks_of(K); g.dtype = dtype; g.out = out;
}

bool muon_size_ok(const tmoe_muon_tensor& t) {
  if (t.batch < 0 || t.rows < 0 || t.cols < 0 || t.rows > tmoe::kMuonMaxSide || t.cols > tmoe::kMuonMaxSide)
    return false;
  const int64_t lo = t.rows < t.cols ? t.rows : t.cols;
  if (lo > tmoe::kMuonMaxShort) return false;
  const int64_t n = t.rows * t.cols;
  return n == 0 || t.batch <= ((int64_t)1 << 36) / n;
}
// Whether the polynomial keeps what the kernels store within its range, from [0, 1] on
bool muon_stays(const double k[3], int steps) {
  double most = 1.0;
  for (int i = 0; i < steps; ++i) {
    double next = 0.0;
    constexpr int n = 512;       // (the polynomial moves little between two of so many places)
    for (int j = 0; j <= n; ++j) {
      const double x = most * j / n, s = x * x;
      const double q = s * (k[1] + k[2] * s), y = fabs(x * (k[0] + q));
      if (!(y <= 2.0) || !(fabs(q) <= 16.0) || !(fabs(k[1]) * s + fabs(k[2]) * s * s <= 64.0)) return false;
      if (y > next) next = y;
    }
    most = next;
  }
  return true;
}

}  // namespace

extern "C" {

size_t tmoe_expert_router_workspace_bytes(int64_t B, int64_t E) {
  if (B < 0 || E < 1 || E > tmoe::kRouterMaxE || B > kMaxRows) return 0;
  return tmoe::expert_router_workspace_bytes(B, E);
}

int tmoe_expert_router_forward(const tmoe_expert_router* r, int64_t* idx, float* w, int64_t* counts,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "tmoe_expert_router_forward";
  tmoe::clear_error();
  if (int rc = er_check(who, r)) return rc;
  if ((r->B > 0 && (!idx || !w)) || !counts || !workspace)
    return fail(TMOE_EINVAL, "%s: null pointer", who);
  if (!on(idx, 8) || !on(w, 4) || !on(counts, 8) || !on(workspace, 4))
    return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  const size_t need = tmoe::expert_router_workspace_bytes(r->B, r->E);
  if (workspace_bytes < need)
    return fail(TMOE_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  tmoe::ExpertRouterArgs a = er_args(r);
  a.idx = idx; a.w = w; a.counts = counts; a.part = static_cast<uint32_t*>(workspace);
  return done(tmoe::expert_router_forward(a, static_cast<hipStream_t>(stream)), who);
}

int tmoe_expert_router_backward(const tmoe_expert_router* r, const int64_t* idx, const float* w,
                                const float* dw, void* draw, void* stream) {
  const char* who = "tmoe_expert_router_backward";
  tmoe::clear_error();
  if (int rc = er_check(who, r)) return rc;
  if (r->B == 0) return TMOE_OK;
  if (!idx || !w || !dw || !draw) return fail(TMOE_EINVAL, "%s: null pointer", who);
  if (!on(idx, 8) || !on(w, 4) || !on(dw, 4) || !on(draw, size_of(r->dtype)))
    return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  tmoe::ExpertRouterArgs a = er_args(r);
  a.idx = const_cast<int64_t*>(idx); a.w = const_cast<float*>(w); a.dw = dw; a.draw = draw;
  return done(tmoe::expert_router_backward(a, static_cast<hipStream_t>(stream)), who);
}

int tmoe_fp8_quantize(const void* x, int64_t R, int64_t C, int64_t row_stride, int dtype,
                      const tmoe_fp8_operand* rows, const tmoe_fp8_operand* cols, void* stream) {
  const char* who = "tmoe_fp8_quantize";
  tmoe::clear_error();
  if (!dtype_ok(dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d is not TMOE_BF16 or TMOE_F32", who, dtype);
  if (!rows && !cols) return fail(TMOE_EINVAL, "%s: nothing is wanted", who);
  if (R < 0 || C < 1) return fail(TMOE_EINVAL, "%s: R=%lld C=%lld", who, (long long)R, (long long)C);
  if (R == 0) return TMOE_OK;
  if (rows)
    if (int rc = fp8_check(who, "rows", rows, R, C)) return rc;
  if (cols)
    if (int rc = fp8_check(who, "cols", cols, C, R)) return rc;
  if (blocks_of(R) * blocks_of(C) >= (int64_t)1 << 31)
    return fail(TMOE_EUNSUPPORTED, "%s: R=%lld C=%lld", who, (long long)R, (long long)C);
  const bool tiles = (rows ? rows : cols)->tiles != 0;
  if (rows && cols) {
    if ((cols->tiles != 0) != tiles)
      return fail(TMOE_EINVAL, "%s: tiles in one of rows and cols", who);
    if (tiles && (rows->scales != cols->scales || rows->scale_row != cols->scale_block ||
                  rows->scale_block != cols->scale_row))
      return fail(TMOE_EINVAL, "%s: tiles have one set of scales", who);
  }
  if (!x) return fail(TMOE_EINVAL, "%s: null x", who);
  if (!on(x, size_of(dtype))) return fail(TMOE_EINVAL, "%s: misaligned x", who);
  if (row_stride < (R > 1 ? C : 0)) return fail(TMOE_EINVAL, "%s: rows that overlap", who);
  tmoe::Fp8QuantizeArgs a{};
  a.x = x; a.R = R; a.C = C; a.row_stride = row_stride; a.dtype = dtype; a.tiles = tiles;
  if (rows) {
    a.row_codes = rows->codes; a.row_scales = rows->scales; a.row_bytes = rows->row_bytes;
    a.row_rs = rows->scale_row; a.row_ks = rows->scale_block;
  }
  if (cols) {
    a.col_codes = cols->codes; a.col_scales = cols->scales; a.col_bytes = cols->row_bytes;
    a.col_rs = cols->scale_row; a.col_ks = cols->scale_block;
    if (!rows && tiles) {      // the kernel writes a tile's scale by its place in x
      a.row_scales = cols->scales; a.row_rs = cols->scale_block; a.row_ks = cols->scale_row;
    }
  }
  return done(tmoe::fp8_quantize(a, static_cast<hipStream_t>(stream)), who);
}

size_t tmoe_fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int values) {
  if (!fp8_sizes_ok(M, N, K) || !dtype_ok(dtype)) return 0;
  return fp8_workspace(M, N, K, values != 0, dtype).total;
}

int tmoe_fp8_gemm(const tmoe_fp8_operand* a, const tmoe_fp8_operand* b, int64_t K, int dtype, void* out,
                  void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "tmoe_fp8_gemm";
  tmoe::clear_error();
  if (int rc = fp8_check(who, "a", a, a ? a->rows : 0, K)) return rc;
  if (int rc = fp8_check(who, "b", b, b ? b->rows : 0, K)) return rc;
  const int64_t M = a->rows;
  const size_t need = tmoe_fp8_gemm_workspace_bytes(M, b->rows, K, dtype, 0);
  if (int rc = fp8_gemm_check(who, M, b, K, dtype, out, workspace, workspace_bytes, need)) return rc;
  tmoe::Fp8GemmArgs g{};
  fp8_b(g, b, K, dtype, out);
  g.a = a->codes; g.a_bytes = a->row_bytes; g.sa = a->scales; g.sa_rs = a->scale_row;
  g.sa_ks = a->scale_block; g.a_tiles = a->tiles != 0; g.a_dtype = -1; g.M = M;
  g.planes = static_cast<float*>(workspace);
  return done(tmoe::fp8_gemm(g, static_cast<hipStream_t>(stream)), who);
}

int tmoe_fp8_gemm_values(const void* x, int64_t M, int64_t row_stride, int x_dtype,
                         const tmoe_fp8_operand* b, int64_t K, int dtype, void* out, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const char* who = "tmoe_fp8_gemm_values";
  tmoe::clear_error();
  if (!dtype_ok(x_dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d of x is not TMOE_BF16 or TMOE_F32", who, x_dtype);
  if (int rc = fp8_check(who, "b", b, b ? b->rows : 0, K)) return rc;
  if (M < 0) return fail(TMOE_EINVAL, "%s: M=%lld", who, (long long)M);
  if (M > tmoe::kFp8MaxDim)
    return fail(TMOE_EUNSUPPORTED, "%s: M=%lld (at most 2^23)", who, (long long)M);
  const Fp8Workspace w = fp8_workspace(M, b->rows < 1 ? 1 : b->rows, K, true, dtype);
  if (int rc = fp8_gemm_check(who, M, b, K, dtype, out, workspace, workspace_bytes, w.total)) return rc;
  if (M == 0) return TMOE_OK;
  if (!x) return fail(TMOE_EINVAL, "%s: null x", who);
  if (!on(x, size_of(x_dtype))) return fail(TMOE_EINVAL, "%s: misaligned x", who);
  if (row_stride < (M > 1 ? K : 0)) return fail(TMOE_EINVAL, "%s: rows that overlap", who);
  tmoe::Fp8GemmArgs g{};
  fp8_b(g, b, K, dtype, out);
  g.M = M;
  g.planes = static_cast<float*>(workspace);
  if (!w.codes) {
    g.a = x; g.a_bytes = row_stride; g.a_dtype = x_dtype;
    return done(tmoe::fp8_gemm(g, static_cast<hipStream_t>(stream)), who);
  }
  const int64_t kb = blocks_of(K);
  tmoe::Fp8QuantizeArgs q{};
  q.x = x; q.R = M; q.C = K; q.row_stride = row_stride; q.dtype = x_dtype;
  q.row_codes = static_cast<char*>(workspace) + w.planes;
  q.row_scales = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.planes + w.codes);
  q.row_bytes = kb * 128; q.row_rs = 1; q.row_ks = M;
  if (hipError_t e = tmoe::fp8_quantize(q, static_cast<hipStream_t>(stream)); e != hipSuccess)
    return done(e, who);
  g.a = q.row_codes; g.a_bytes = q.row_bytes; g.sa = q.row_scales; g.sa_rs = 1; g.sa_ks = M;
  g.a_dtype = -1;
  return done(tmoe::fp8_gemm(g, static_cast<hipStream_t>(stream)), who);
}

size_t tmoe_muon_workspace_bytes(const tmoe_muon_tensor* t, int64_t count) {
  if (count <= 0 || !t) return 0;
  for (int64_t i = 0; i < count; ++i)
    if (!muon_size_ok(t[i])) return 0;
  return tmoe::muon_workspace_bytes(t, count);
}

int tmoe_muon_step(const tmoe_muon_tensor* t, int64_t count, const tmoe_muon_step_args* a, void* workspace,
                   size_t workspace_bytes, void* stream) {
  const char* who = "tmoe_muon_step";
  tmoe::clear_error();
  if (!a || count < 0 || (count > 0 && !t)) return fail(TMOE_EINVAL, "%s: null or count", who);
  if (!dtype_ok(a->dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d is not TMOE_BF16 or TMOE_F32", who, (int)a->dtype);
  if (a->steps < 1 || a->steps > 16) return fail(TMOE_EINVAL, "%s: steps %d (1 to 16)", who, (int)a->steps);
  if (!(a->momentum >= 0.0 && a->momentum < 1.0))
    return fail(TMOE_EINVAL, "%s: momentum must be in [0, 1)", who);
  for (double v : {a->lr, a->weight_decay, a->update_rms})
    if (!(v >= 0.0) || !isfinite((float)v))
      return fail(TMOE_EINVAL, "%s: lr, weight_decay and update_rms must be finite and >= 0", who);
  if (!((float)a->eps > 0.f) || !isfinite((float)a->eps))
    return fail(TMOE_EINVAL, "%s: eps must be positive and finite", who);
  if (!muon_stays(a->coefficients, a->steps))
    return fail(TMOE_EINVAL, "%s: coefficients %g, %g, %g do not stay in range", who, a->coefficients[0],
                a->coefficients[1], a->coefficients[2]);
  const size_t es = size_of(a->dtype);
  for (int64_t i = 0; i < count; ++i) {
    const tmoe_muon_tensor& q = t[i];
    if (q.batch < 0 || q.rows < 0 || q.cols < 0)
      return fail(TMOE_EINVAL, "%s: tensor %lld: %lld of (%lld, %lld)", who, (long long)i,
                  (long long)q.batch, (long long)q.rows, (long long)q.cols);
    if (!muon_size_ok(q))
      return fail(TMOE_EUNSUPPORTED, "%s: tensor %lld: %lld of (%lld, %lld)", who, (long long)i,
                  (long long)q.batch, (long long)q.rows, (long long)q.cols);
    if (q.batch == 0 || q.rows == 0 || q.cols == 0) continue;
    if (!q.p || !q.g) return fail(TMOE_EINVAL, "%s: tensor %lld: null pointer", who, (long long)i);
    if (!on(q.p, es) || !on(q.g, es) || !on(q.m, 4))
      return fail(TMOE_EINVAL, "%s: tensor %lld: misaligned pointer", who, (long long)i);
  }
  const size_t need = tmoe_muon_workspace_bytes(t, count);
  if (need && (!workspace || workspace_bytes < need))
    return fail(TMOE_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  if (!on(workspace, 256)) return fail(TMOE_EINVAL, "%s: misaligned workspace", who);
  return done(tmoe::muon(t, count, *a, workspace, static_cast<hipStream_t>(stream)), who);
}

}  // extern "C"
