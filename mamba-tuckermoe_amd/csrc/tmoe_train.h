// Launchers of the training operators around the expert contraction (tmoe_train.hip),
// called by the C ABI's entry points in tmoe_train_api.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "tmoe.h"

namespace tmoe {

// tmoe_last_error()'s text for an entry point that returns `code`; `code`.
int fail_text(int code, const char* text);
void clear_error();

constexpr int64_t kRouterMaxE = 256, kRouterMaxK = 16;

struct RouterArgs {
  const void* raw;
  int64_t row_stride, B;
  int E, k, dtype;
  float cap, tau;
  const float* tau_dev;
  const uint8_t* mask;
  int64_t* idx;
  float* w;
  float *lb, *z, *tokens;  // the losses; how many tokens are not masked
  int64_t* counts;
  float* part;             // workspace
  int blocks;              // of the forward
  const float *dw, *dlb, *dz;
  void* draw;
};
size_t router_workspace_bytes(int64_t B, int64_t E);
hipError_t router_forward(RouterArgs a, hipStream_t st);
hipError_t router_backward(const RouterArgs& a, hipStream_t st);

constexpr int64_t kBlockNormMaxD = 16384;

struct BlockNormArgs {
  const void *x, *y, *gate;
  int64_t x_rs, y_rs, gate_rs;              // row strides in elements
  const void *post_w, *gamma, *next_w;
  int64_t T, d;
  int dtype;
  float eps;
  void *r, *h;
  float* inv;                               // (2, T): 1 / rms of u and of r
  // backward
  const void *dr, *dh;
  int64_t dr_rs, dh_rs;
  void *dx, *dy, *dgate, *dpost_w, *dgamma, *dnext_w;
  float* part;
};
size_t block_norm_workspace_bytes(int64_t T, int64_t d, int dtype);
hipError_t block_norm_forward(const BlockNormArgs& a, hipStream_t st);
hipError_t block_norm_backward(const BlockNormArgs& a, hipStream_t st);

constexpr int64_t kAdamwBlock = 256;        // elements that share a scale in 8-bit states
constexpr int64_t kAdamwMaxN = (int64_t)1 << 36;

hipError_t adamw(const tmoe_adamw_tensor* t, int64_t count, const tmoe_adamw_step_args& a,
                 hipStream_t st);

}  // namespace tmoe
