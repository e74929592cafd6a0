// Launchers of the training operators around the expert contraction: the router with its
// losses (tmoe_router.hpp), the block norms (tmoe_block_norm.hpp) and the AdamW step
// (tmoe_adamw.hpp).
#include <math.h>

#include "tmoe_adamw.hpp"
#include "tmoe_block_norm.hpp"
#include "tmoe_router.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace {

constexpr int kDtypeBF16 = TMOE_BF16;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int64_t kAdamwGroups = (1 << 24) - 1;   // a launch's threads are counted in 32 bits

// ---- router ----
int router_lanes(int64_t E) {
  int l = 1;
  while (4 * l < E) l <<= 1;
  return l;
}
constexpr int64_t kRouterBlocks = 512;   // planes that the second launch adds
int64_t router_blocks(int64_t B, int64_t E) {
  const int64_t n = ceil_div(B, dev::kRouterThreads / router_lanes(E));
  return n < 1 ? 1 : n < kRouterBlocks ? n : kRouterBlocks;
}

template <class T>
void router_launch(const RouterArgs& a, bool backward, int64_t blocks, hipStream_t st) {
  const dim3 grid((unsigned)blocks), block(dev::kRouterThreads);
#define TMOE_ROUTER(L)                                                            \
  case L:                                                                         \
    if (backward) hipLaunchKernelGGL((dev::k_router_bwd<T, L>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((dev::k_router_fwd<T, L>), grid, block, 0, st, a);    \
    break;
  switch (router_lanes(a.E)) {
    TMOE_ROUTER(1) TMOE_ROUTER(2) TMOE_ROUTER(4) TMOE_ROUTER(8)
    TMOE_ROUTER(16) TMOE_ROUTER(32) TMOE_ROUTER(64)
  }
#undef TMOE_ROUTER
}

// ---- block norm ----
struct NormPlan {
  bool wave;            // a wave to a row
  int chunks;           // chunks of 16 bytes a thread
  unsigned threads;
  int teams;            // rows at a time in a work-group
};
NormPlan norm_plan(int64_t d, int es) {
  const int64_t nch = ceil_div(d * es, 16);
  if (nch <= 128) return {true, nch <= 64 ? 1 : 2, dev::kNormThreads, dev::kNormThreads / 64};
  const int c = nch <= 1024 ? 1 : nch <= 2048 ? 2 : 4;
  return {false, c, (unsigned)(ceil_div(nch, 64 * c) * 64), 1};
}
constexpr int64_t kNormBlocks = 1024;     // of the backward
int64_t norm_bwd_blocks(int64_t T, const NormPlan& p) {
  const int64_t n = ceil_div(T, p.teams), most = p.wave ? kNormBlocks / 2 : kNormBlocks;
  return n < most ? n : most;
}

template <class T, bool kVec>
void norm_launch(const BlockNormArgs& a, bool backward, const NormPlan& p, int64_t blocks,
                 hipStream_t st) {
  const dim3 grid((unsigned)blocks), block(p.threads);
#define TMOE_NORM(C, W)                                                                        \
  if (p.chunks == C && p.wave == W) {                                                          \
    if (backward) hipLaunchKernelGGL((dev::k_block_norm_bwd<T, C, W, kVec>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((dev::k_block_norm_fwd<T, C, W, kVec>), grid, block, 0, st, a);    \
  }
  TMOE_NORM(1, true) TMOE_NORM(2, true)
  TMOE_NORM(1, false) TMOE_NORM(2, false) TMOE_NORM(4, false)
#undef TMOE_NORM
}
void norm_dispatch(const BlockNormArgs& a, bool backward, const NormPlan& p, int64_t blocks,
                   hipStream_t st) {
  const int epc = a.dtype == kDtypeBF16 ? 8 : 4;
  const void* ptrs[] = {a.x, a.y, a.gate, a.post_w, a.gamma, a.next_w, a.r, a.h,
                        a.dr, a.dh, a.dx, a.dy, a.dgate};
  bool vec = a.d % epc == 0;
  for (const void* q : ptrs) vec = vec && aligned(q);
  const int64_t strides[] = {a.x ? a.x_rs : 0, a.y_rs, a.gate ? a.gate_rs : 0, a.dr ? a.dr_rs : 0,
                             a.dh ? a.dh_rs : 0};
  for (int64_t s : strides) vec = vec && s % epc == 0;
  if (a.dtype == kDtypeBF16) {
    if (vec) norm_launch<uint16_t, true>(a, backward, p, blocks, st);
    else norm_launch<uint16_t, false>(a, backward, p, blocks, st);
  } else {
    if (vec) norm_launch<float, true>(a, backward, p, blocks, st);
    else norm_launch<float, false>(a, backward, p, blocks, st);
  }
}
int es_of(int dtype) { return dtype == kDtypeBF16 ? 2 : 4; }

}  // namespace

size_t router_workspace_bytes(int64_t B, int64_t E) {
  return (size_t)router_blocks(B, E) * (2 * E + 2) * sizeof(float);
}
hipError_t router_forward(RouterArgs a, hipStream_t st) {
  a.blocks = (int)router_blocks(a.B, a.E);
  if (a.dtype == kDtypeBF16) router_launch<uint16_t>(a, false, a.blocks, st);
  else router_launch<float>(a, false, a.blocks, st);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  hipLaunchKernelGGL(dev::k_router_finish, dim3(1), dim3(1024), 0, st, a);
  return hipGetLastError();
}
hipError_t router_backward(const RouterArgs& a, hipStream_t st) {
  if (a.B == 0) return hipSuccess;
  const int64_t n = ceil_div(a.B, dev::kRouterThreads / router_lanes(a.E));
  const int64_t blocks = n < 4096 ? n : 4096;
  if (a.dtype == kDtypeBF16) router_launch<uint16_t>(a, true, blocks, st);
  else router_launch<float>(a, true, blocks, st);
  return hipGetLastError();
}

size_t block_norm_workspace_bytes(int64_t T, int64_t d, int dtype) {
  const NormPlan p = norm_plan(d, es_of(dtype));
  return (size_t)(3 * norm_bwd_blocks(T, p) * p.teams * d) * sizeof(float);
}
hipError_t block_norm_forward(const BlockNormArgs& a, hipStream_t st) {
  if (a.T == 0) return hipSuccess;
  const NormPlan p = norm_plan(a.d, es_of(a.dtype));
  const int64_t n = ceil_div(a.T, p.teams);
  norm_dispatch(a, false, p, n < 8192 ? n : 8192, st);
  return hipGetLastError();
}
hipError_t block_norm_backward(const BlockNormArgs& a, hipStream_t st) {
  const NormPlan p = norm_plan(a.d, es_of(a.dtype));
  const int64_t blocks = norm_bwd_blocks(a.T, p);
  if (a.T > 0) {
    norm_dispatch(a, true, p, blocks, st);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (!a.dpost_w && !a.dgamma && !a.dnext_w) return hipSuccess;
  const dim3 grid((unsigned)ceil_div(a.d, 64), 3), block(1024);
  if (a.dtype == kDtypeBF16)
    hipLaunchKernelGGL(dev::k_block_norm_cols<uint16_t>, grid, block, 0, st, a, blocks * p.teams);
  else
    hipLaunchKernelGGL(dev::k_block_norm_cols<float>, grid, block, 0, st, a, blocks * p.teams);
  return hipGetLastError();
}

hipError_t adamw(const tmoe_adamw_tensor* t, int64_t count, const tmoe_adamw_step_args& a,
                 hipStream_t st) {
  static_assert(sizeof(dev::AdamwTable) <= 4096, "a launch's arguments");
  // a work-group's elements: enough work-groups for the chip where the tensors are small
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += t[i].n;
  int64_t chunk = 8192;
  while (chunk > 1024 && total / chunk < 2048) chunk >>= 1;
  dev::AdamwTable b;
  b.step_dev = a.step_dev;
  b.beta1 = a.beta1; b.beta2 = a.beta2; b.lr = a.lr;
  b.b1 = (float)a.beta1; b.ob1 = (float)(1.0 - a.beta1);
  b.b2 = (float)a.beta2; b.ob2 = (float)(1.0 - a.beta2);
  b.eps = (float)a.eps; b.keep = (float)(1.0 - a.lr * a.weight_decay);
  b.rate = (float)(a.lr / (1.0 - pow(a.beta1, (double)a.step)));
  b.inv_c2 = 1.f / (float)sqrt(1.0 - pow(a.beta2, (double)a.step));
  b.seed = a.step_dev ? a.seed : dev::mix32(a.seed + (uint32_t)a.step * 0x9E3779B1u);
  int64_t i = 0;
  while (i < count) {
    b.count = 0;
    b.first = (uint32_t)i;
    b.chunk = chunk;
    uint32_t groups = 0;
    for (; i < count && b.count < dev::kAdamwTensors; ++i) {
      const tmoe_adamw_tensor& q = t[i];
      const int64_t need = ceil_div(q.n, chunk);
      if (groups + need > kAdamwGroups) break;
      groups += (uint32_t)need;
      const int c = b.count++;
      b.p[c] = q.p; b.g[c] = q.g; b.m[c] = q.m; b.v[c] = q.v;
      b.ms[c] = q.m_scale; b.vs[c] = q.v_scale; b.n[c] = q.n; b.end[c] = groups;
    }
    if (b.count == 0) return hipErrorInvalidValue;
    if (groups == 0) continue;
    const dim3 grid(groups), block(dev::kAdamwThreads);
    if (a.state_bits == 32) {
      if (a.dtype == kDtypeBF16) hipLaunchKernelGGL(dev::k_adamw32<uint16_t>, grid, block, 0, st, b);
      else hipLaunchKernelGGL(dev::k_adamw32<float>, grid, block, 0, st, b);
    } else {
      if (a.dtype == kDtypeBF16) hipLaunchKernelGGL(dev::k_adamw8<uint16_t>, grid, block, 0, st, b);
      else hipLaunchKernelGGL(dev::k_adamw8<float>, grid, block, 0, st, b);
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tmoe
