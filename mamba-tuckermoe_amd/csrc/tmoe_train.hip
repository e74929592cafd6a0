// Launchers of the training operators around the expert contraction: the router with its
// losses (tmoe_router.hpp) and the AdamW step (tmoe_adamw.hpp); the block norms' are in
// tmoe_norm_launch.hpp.
#include <math.h>

#include "tmoe_adamw.hpp"
#include "tmoe_router.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace {

constexpr int kDtypeBF16 = TMOE_BF16;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kAdamwGroups = (1 << 24) - 1;   // a launch's threads are counted in 32 bits

// ---- router ----
// Lanes of a token: eight experts to a lane, four where that is all of them.
int router_lanes(int64_t E) {
  int l = 1;
  while (8 * l < E) l <<= 1;
  return l;
}
// Work-groups of the forward, a plane each for the second launch to add: at E = 64, B = 131072
// the two take 23.0 + 4.8 us with 768, 25.7 + 4.5 with 512, 22.8 + 5.3 with 1024, 22.6 + 5.9
// with 1280. The backward's, which sets up more than it gains by more waves (when that was
// measured; 21.9 us now): 21.6 us with 768, 22.7 with 1024, 23.2 with 1536, 25.0 with 2048; the next token's inputs read ahead,
// as in the forward, 22.0.
constexpr int64_t kRouterBlocks = 768, kRouterBwdBlocks = 768;
int64_t router_blocks(int64_t B, int64_t E) {
  const int64_t n = ceil_div(B, dev::kRouterThreads / router_lanes(E));
  return n < 1 ? 1 : n < kRouterBlocks ? n : kRouterBlocks;
}
int64_t router_finish_blocks(int64_t E) { return ceil_div(E, dev::kFinishCols); }

template <class T>
void router_launch(const RouterArgs& a, bool backward, int64_t blocks, hipStream_t st) {
  const dim3 grid((unsigned)blocks), block(dev::kRouterThreads);
#define TMOE_ROUTER(L, V)                                                                  \
  if (backward) hipLaunchKernelGGL((dev::k_router_bwd<T, L, V>), grid, block, 0, st, a);   \
  else hipLaunchKernelGGL((dev::k_router_fwd<T, L, V>), grid, block, 0, st, a);
  if (a.E <= 4) { TMOE_ROUTER(1, 4) return; }
  switch (router_lanes(a.E)) {
    case 1: TMOE_ROUTER(1, 8) break;
    case 2: TMOE_ROUTER(2, 8) break;
    case 4: TMOE_ROUTER(4, 8) break;
    case 8: TMOE_ROUTER(8, 8) break;
    case 16: TMOE_ROUTER(16, 8) break;
    case 32: TMOE_ROUTER(32, 8) break;
  }
#undef TMOE_ROUTER
}

}  // namespace

size_t router_workspace_bytes(int64_t B, int64_t E) {
  // the planes, then k_router_finish's count of its work-groups and their parts of lb
  return (size_t)(2 * router_blocks(B, E) * (E + 1) + 1 + router_finish_blocks(E)) * sizeof(float);
}
hipError_t router_forward(RouterArgs a, hipStream_t st) {
  a.blocks = (int)router_blocks(a.B, a.E);
  if (a.dtype == kDtypeBF16) router_launch<uint16_t>(a, false, a.blocks, st);
  else router_launch<float>(a, false, a.blocks, st);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (a.blocks == 1) return hipSuccess;   // one work-group has the sums whole
  hipLaunchKernelGGL(dev::k_router_finish, dim3((unsigned)router_finish_blocks(a.E)), dim3(1024), 0,
                     st, a);
  return hipGetLastError();
}
hipError_t router_backward(const RouterArgs& a, hipStream_t st) {
  if (a.B == 0) return hipSuccess;
  const int64_t n = ceil_div(a.B, dev::kRouterThreads / router_lanes(a.E));
  const int64_t blocks = n < kRouterBwdBlocks ? n : kRouterBwdBlocks;
  if (a.dtype == kDtypeBF16) router_launch<uint16_t>(a, true, blocks, st);
  else router_launch<float>(a, true, blocks, st);
  return hipGetLastError();
}

// of tmoe_norm_bf16.hip and tmoe_norm_f32.hip
template <class T>
size_t block_norm_workspace(int64_t rows, int64_t d);
template <class T>
hipError_t block_norm_fwd(const BlockNormArgs& a, hipStream_t st);
template <class T>
hipError_t block_norm_bwd(const BlockNormArgs& a, hipStream_t st);

size_t block_norm_workspace_bytes(int64_t T, int64_t d, int dtype) {
  return dtype == kDtypeBF16 ? block_norm_workspace<uint16_t>(T, d) : block_norm_workspace<float>(T, d);
}
hipError_t block_norm_forward(const BlockNormArgs& a, hipStream_t st) {
  return a.dtype == kDtypeBF16 ? block_norm_fwd<uint16_t>(a, st) : block_norm_fwd<float>(a, st);
}
hipError_t block_norm_backward(const BlockNormArgs& a, hipStream_t st) {
  return a.dtype == kDtypeBF16 ? block_norm_bwd<uint16_t>(a, st) : block_norm_bwd<float>(a, st);
}

hipError_t adamw(const tmoe_adamw_tensor* t, int64_t count, const tmoe_adamw_step_args& a,
                 hipStream_t st) {
  static_assert(sizeof(dev::AdamwTable) <= 4096, "a launch's arguments");
  // a work-group's elements: enough work-groups for the chip where the tensors are small, but
  // each thread four of 32 bits or eight of 8
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += t[i].n;
  int64_t chunk = 8192;
  const int64_t least = a.state_bits == 8 ? 2048 : 1024;
  while (chunk > least && total / chunk < 2048) chunk >>= 1;
  // a tensor of the largest size is less than a launch
  static_assert(kAdamwMaxN / 8192 <= kAdamwGroups, "");
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
