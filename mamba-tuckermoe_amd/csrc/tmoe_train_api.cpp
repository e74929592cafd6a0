// The C ABI's entry points of the training operators around the expert contraction
// (include/tmoe.h: tmoe_router_*, tmoe_block_norm_*, tmoe_adamw_step): argument checks on
// the host before the first HIP call, then the launchers of tmoe_train.hip.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "tmoe.h"
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

int router_check(const char* who, const tmoe_router* r) {
  if (!r) return fail(TMOE_EINVAL, "%s: null router", who);
  if (!dtype_ok(r->dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d is not TMOE_BF16 or TMOE_F32", who, (int)r->dtype);
  if (r->B < 0 || r->E < 1 || r->k < 1 || r->k > r->E)
    return fail(TMOE_EINVAL, "%s: B=%lld E=%lld k=%lld", who, (long long)r->B, (long long)r->E,
                (long long)r->k);
  if (r->E > tmoe::kRouterMaxE || r->k > tmoe::kRouterMaxK || r->B > kMaxRows)
    return fail(TMOE_EUNSUPPORTED, "%s: B=%lld E=%lld k=%lld (at most 2^30, 256, 16)", who,
                (long long)r->B, (long long)r->E, (long long)r->k);
  if (!(r->cap > 0.f) || !isfinite(r->cap))
    return fail(TMOE_EINVAL, "%s: cap must be positive and finite", who);
  if (!r->temperature_dev && (!(r->temperature > 0.f) || !isfinite(r->temperature)))
    return fail(TMOE_EINVAL, "%s: temperature must be positive and finite", who);
  if (r->B > 0 && !r->raw) return fail(TMOE_EINVAL, "%s: null raw", who);
  if (r->row_stride < (r->B > 1 ? r->E : 0))
    return fail(TMOE_EINVAL, "%s: row_stride %lld", who, (long long)r->row_stride);
  if (!on(r->raw, size_of(r->dtype)) || !on(r->temperature_dev, 4))
    return fail(TMOE_EINVAL, "%s: misaligned raw or temperature_dev", who);
  return TMOE_OK;
}
tmoe::RouterArgs router_args(const tmoe_router* r) {
  tmoe::RouterArgs a{};
  a.raw = r->raw; a.row_stride = r->row_stride; a.B = r->B;
  a.E = (int)r->E; a.k = (int)r->k; a.dtype = r->dtype;
  a.cap = r->cap; a.tau = r->temperature; a.tau_dev = r->temperature_dev; a.mask = r->mask;
  return a;
}

int norm_check(const char* who, const tmoe_block_norm* n) {
  if (!n) return fail(TMOE_EINVAL, "%s: null norm", who);
  if (!dtype_ok(n->dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d is not TMOE_BF16 or TMOE_F32", who, (int)n->dtype);
  if (n->T < 0 || n->d < 1)
    return fail(TMOE_EINVAL, "%s: T=%lld d=%lld", who, (long long)n->T, (long long)n->d);
  if (n->T > kMaxRows || n->d > tmoe::kBlockNormMaxD)
    return fail(TMOE_EUNSUPPORTED, "%s: T=%lld d=%lld (at most 2^30, 16384)", who,
                (long long)n->T, (long long)n->d);
  if (!(n->eps >= 0.f)) return fail(TMOE_EINVAL, "%s: eps must be >= 0", who);
  if (n->T > 0 && !n->y) return fail(TMOE_EINVAL, "%s: null y", who);
  const int64_t least = n->T > 1 ? n->d : 0;
  if ((n->x && n->x_stride < least) || n->y_stride < least || (n->gate && n->gate_stride < least))
    return fail(TMOE_EINVAL, "%s: rows that overlap", who);
  const size_t es = size_of(n->dtype);
  for (const void* p : {n->x, n->y, n->gate, n->post_weight, n->gamma, n->next_weight})
    if (!on(p, es)) return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  return TMOE_OK;
}
tmoe::BlockNormArgs norm_args(const tmoe_block_norm* n) {
  tmoe::BlockNormArgs a{};
  a.x = n->x; a.y = n->y; a.gate = n->gate;
  a.x_rs = n->x_stride; a.y_rs = n->y_stride; a.gate_rs = n->gate_stride;
  a.post_w = n->post_weight; a.gamma = n->gamma; a.next_w = n->next_weight;
  a.T = n->T; a.d = n->d; a.dtype = n->dtype; a.eps = n->eps;
  return a;
}

}  // namespace

extern "C" {

size_t tmoe_router_workspace_bytes(int64_t B, int64_t E) {
  if (B < 0 || E < 1 || E > tmoe::kRouterMaxE || B > kMaxRows) return 0;
  return tmoe::router_workspace_bytes(B, E);
}

int tmoe_router_forward(const tmoe_router* r, int64_t* idx, float* w, float* lb, float* z,
                        float* tokens, int64_t* counts, void* workspace, size_t workspace_bytes,
                        void* stream) {
  const char* who = "tmoe_router_forward";
  tmoe::clear_error();
  if (int rc = router_check(who, r)) return rc;
  if ((r->B > 0 && (!idx || !w)) || !lb || !z || !tokens || !counts || !workspace)
    return fail(TMOE_EINVAL, "%s: null pointer", who);
  if (!on(idx, 8) || !on(w, 4) || !on(lb, 4) || !on(z, 4) || !on(tokens, 4) || !on(counts, 8) ||
      !on(workspace, 8))
    return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  const size_t need = tmoe::router_workspace_bytes(r->B, r->E);
  if (workspace_bytes < need)
    return fail(TMOE_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
  tmoe::RouterArgs a = router_args(r);
  a.idx = idx; a.w = w; a.lb = lb; a.z = z; a.tokens = tokens; a.counts = counts;
  a.part = static_cast<float*>(workspace);
  return done(tmoe::router_forward(a, static_cast<hipStream_t>(stream)), who);
}

int tmoe_router_backward(const tmoe_router* r, const int64_t* idx, const float* tokens,
                         const int64_t* counts, const float* dw, const float* dlb,
                         const float* dz, void* draw, void* stream) {
  const char* who = "tmoe_router_backward";
  tmoe::clear_error();
  if (int rc = router_check(who, r)) return rc;
  if (r->B == 0) return TMOE_OK;
  if (!idx || !tokens || !counts || !draw) return fail(TMOE_EINVAL, "%s: null pointer", who);
  if (!on(idx, 8) || !on(tokens, 4) || !on(counts, 8) || !on(dw, 4) || !on(dlb, 4) ||
      !on(dz, 4) || !on(draw, size_of(r->dtype)))
    return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  tmoe::RouterArgs a = router_args(r);
  a.idx = const_cast<int64_t*>(idx); a.tokens = const_cast<float*>(tokens);
  a.counts = const_cast<int64_t*>(counts);
  a.dw = dw; a.dlb = dlb; a.dz = dz; a.draw = draw;
  return done(tmoe::router_backward(a, static_cast<hipStream_t>(stream)), who);
}

size_t tmoe_block_norm_workspace_bytes(int64_t T, int64_t d, int dtype) {
  if (T < 0 || T > kMaxRows || d < 1 || d > tmoe::kBlockNormMaxD || !dtype_ok(dtype)) return 0;
  return tmoe::block_norm_workspace_bytes(T, d, dtype);
}

int tmoe_block_norm_forward(const tmoe_block_norm* n, void* r, void* h, float* inv,
                            void* stream) {
  const char* who = "tmoe_block_norm_forward";
  tmoe::clear_error();
  if (int rc = norm_check(who, n)) return rc;
  if (n->T == 0) return TMOE_OK;
  if ((n->next_weight != nullptr) != (h != nullptr) || (!r && !h))
    return fail(TMOE_EINVAL, "%s: h goes with next_weight, and r or h is wanted", who);
  const size_t es = size_of(n->dtype);
  if (!on(r, es) || !on(h, es) || !on(inv, 4))
    return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  tmoe::BlockNormArgs a = norm_args(n);
  a.r = r; a.h = h; a.inv = inv;
  return done(tmoe::block_norm_forward(a, static_cast<hipStream_t>(stream)), who);
}

int tmoe_block_norm_backward(const tmoe_block_norm* n, const float* inv, const void* dr,
                             int64_t dr_stride, const void* dh, int64_t dh_stride, void* dx,
                             void* dy, void* dgate, void* dpost_weight, void* dgamma,
                             void* dnext_weight, void* workspace, size_t workspace_bytes,
                             void* stream) {
  const char* who = "tmoe_block_norm_backward";
  tmoe::clear_error();
  if (int rc = norm_check(who, n)) return rc;
  if ((dx && !n->x) || (dgate && !n->gate) || (dpost_weight && !n->post_weight) ||
      (dgamma && !n->gamma) || ((dnext_weight || dh) && !n->next_weight))
    return fail(TMOE_EINVAL, "%s: a gradient of an operand that is not there", who);
  if (n->T > 0 && !inv && (n->post_weight || n->next_weight))
    return fail(TMOE_EINVAL, "%s: null inv", who);
  const int64_t least = n->T > 1 ? n->d : 0;
  if ((dr && dr_stride < least) || (dh && dh_stride < least))
    return fail(TMOE_EINVAL, "%s: rows that overlap", who);
  const size_t es = size_of(n->dtype);
  for (const void* p : {dr, dh, (const void*)dx, (const void*)dy, (const void*)dgate,
                        (const void*)dpost_weight, (const void*)dgamma, (const void*)dnext_weight})
    if (!on(p, es)) return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  if (!on(inv, 4) || !on(workspace, 4)) return fail(TMOE_EINVAL, "%s: misaligned pointer", who);
  tmoe::BlockNormArgs a = norm_args(n);
  a.inv = const_cast<float*>(inv);
  a.dr = dr; a.dr_rs = dr_stride; a.dh = dh; a.dh_rs = dh_stride;
  a.dx = dx; a.dy = dy; a.dgate = dgate;
  a.dpost_w = dpost_weight; a.dgamma = dgamma; a.dnext_w = dnext_weight;
  if (dpost_weight || dgamma || dnext_weight) {
    const size_t need = tmoe::block_norm_workspace_bytes(n->T, n->d, n->dtype);
    if (need && (!workspace || workspace_bytes < need))
      return fail(TMOE_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
    a.part = static_cast<float*>(workspace);
  }
  return done(tmoe::block_norm_backward(a, static_cast<hipStream_t>(stream)), who);
}

int tmoe_adamw_step(const tmoe_adamw_tensor* t, int64_t count, const tmoe_adamw_step_args* a,
                    void* stream) {
  const char* who = "tmoe_adamw_step";
  tmoe::clear_error();
  if (!a || count < 0 || (count > 0 && !t)) return fail(TMOE_EINVAL, "%s: null or count", who);
  if (!dtype_ok(a->dtype))
    return fail(TMOE_EINVAL, "%s: dtype %d is not TMOE_BF16 or TMOE_F32", who, (int)a->dtype);
  if (a->state_bits != 32 && a->state_bits != 8)
    return fail(TMOE_EINVAL, "%s: state_bits %d is not 32 or 8", who, (int)a->state_bits);
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0) || !(a->beta2 >= 0.0 && a->beta2 < 1.0))
    return fail(TMOE_EINVAL, "%s: betas must be in [0, 1)", who);
  if (!(a->eps >= 0.0) || !(a->lr >= 0.0) || !(a->weight_decay >= 0.0) || !isfinite(a->lr) ||
      !isfinite(a->eps) || !isfinite(a->weight_decay))
    return fail(TMOE_EINVAL, "%s: lr, eps and weight_decay must be finite and >= 0", who);
  if (!a->step_dev && a->step < 1) return fail(TMOE_EINVAL, "%s: step %lld", who, (long long)a->step);
  if (!on(a->step_dev, 8)) return fail(TMOE_EINVAL, "%s: misaligned step_dev", who);
  const size_t es = size_of(a->dtype), ms = a->state_bits == 32 ? 4 : 1;
  for (int64_t i = 0; i < count; ++i) {
    const tmoe_adamw_tensor& q = t[i];
    if (q.n < 0) return fail(TMOE_EINVAL, "%s: tensor %lld: n=%lld", who, (long long)i, (long long)q.n);
    if (q.n == 0) continue;
    if (q.n > tmoe::kAdamwMaxN)
      return fail(TMOE_EUNSUPPORTED, "%s: tensor %lld: n=%lld", who, (long long)i, (long long)q.n);
    if (!q.p || !q.g || !q.m || !q.v || (a->state_bits == 8 && (!q.m_scale || !q.v_scale)))
      return fail(TMOE_EINVAL, "%s: tensor %lld: null pointer", who, (long long)i);
    if (!on(q.p, es) || !on(q.g, es) || !on(q.m, ms) || !on(q.v, ms) || !on(q.m_scale, 4) ||
        !on(q.v_scale, 4))
      return fail(TMOE_EINVAL, "%s: tensor %lld: misaligned pointer", who, (long long)i);
  }
  return done(tmoe::adamw(t, count, *a, static_cast<hipStream_t>(stream)), who);
}

}  // extern "C"
