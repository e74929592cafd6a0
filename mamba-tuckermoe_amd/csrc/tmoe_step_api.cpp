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

}  // extern "C"
