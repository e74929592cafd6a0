// Launchers of the expert router (tmoe_expert_router.hpp).
#include "tmoe_expert_router.hpp"

namespace tmoe {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int er_lanes(int64_t E) {
  int l = 1;
  while (dev::kErV * l < E) l <<= 1;
  return l;
}
constexpr int64_t kErBlocks = 768;      // three to a compute unit, which their registers allow
int64_t er_blocks(int64_t B, int64_t E) {
  const int64_t n = ceil_div(B, dev::kErThreads / er_lanes(E));
  return n < 1 ? 1 : n < kErBlocks ? n : kErBlocks;
}

template <class T>
void er_launch(const ExpertRouterArgs& a, bool backward, int64_t blocks, hipStream_t st) {
  const dim3 grid((unsigned)blocks), block(dev::kErThreads);
#define TMOE_ER(L)                                                                                \
  case L:                                                                                         \
    if (backward) hipLaunchKernelGGL((dev::k_expert_router_bwd<T, L>), grid, block, 0, st, a);    \
    else hipLaunchKernelGGL((dev::k_expert_router_fwd<T, L>), grid, block, 0, st, a);             \
    break;
  switch (er_lanes(a.E)) {
    TMOE_ER(1) TMOE_ER(2) TMOE_ER(4) TMOE_ER(8) TMOE_ER(16) TMOE_ER(32)
  }
#undef TMOE_ER
}

}  // namespace

size_t expert_router_workspace_bytes(int64_t B, int64_t E) {
  return (size_t)(er_blocks(B, E) * E) * sizeof(uint32_t);
}
hipError_t expert_router_forward(ExpertRouterArgs a, hipStream_t st) {
  a.blocks = (int)er_blocks(a.B, a.E);
  if (a.dtype == TMOE_BF16) er_launch<uint16_t>(a, false, a.blocks, st);
  else er_launch<float>(a, false, a.blocks, st);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (a.blocks == 1) return hipSuccess;   // one work-group has the counts whole
  hipLaunchKernelGGL(dev::k_expert_router_counts, dim3((unsigned)ceil_div(a.E, 16)), dim3(1024), 0, st, a);
  return hipGetLastError();
}
hipError_t expert_router_backward(const ExpertRouterArgs& a, hipStream_t st) {
  if (a.B == 0) return hipSuccess;
  const int64_t blocks = er_blocks(a.B, a.E);
  if (a.dtype == TMOE_BF16) er_launch<uint16_t>(a, true, blocks, st);
  else er_launch<float>(a, true, blocks, st);
  return hipGetLastError();
}

}  // namespace tmoe
