// Launchers of the training layer's wider operators: routing to experts by scores, bias and
// groups (tmoe_expert_router.hip), products in 8-bit floating point with a scale for each block
// of 128 (tmoe_fp8_block.hip) and the Muon step (tmoe_muon.hip), called by the C ABI's entry
// points in tmoe_step_api.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "tmoe.h"

namespace tmoe {

struct ExpertRouterArgs {
  const void* raw;
  int64_t row_stride, B;
  int E, k, groups, top_groups, dtype, score, renormalize;
  float scale;
  const float* bias;
  const uint8_t* mask;
  int64_t* idx;
  float* w;
  int64_t* counts;
  uint32_t* part;          // workspace: (blocks, E) counts
  int blocks;              // of the forward
  const float* dw;
  void* draw;
};
size_t expert_router_workspace_bytes(int64_t B, int64_t E);
hipError_t expert_router_forward(ExpertRouterArgs a, hipStream_t st);
hipError_t expert_router_backward(const ExpertRouterArgs& a, hipStream_t st);

}  // namespace tmoe
