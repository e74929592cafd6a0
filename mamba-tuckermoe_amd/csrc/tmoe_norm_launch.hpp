// Launchers of the block norms (tmoe_block_norm.hpp) for one element type; a source file of
// its own for each (tmoe_norm_bf16.hip, tmoe_norm_f32.hip), compiled side by side.
#pragma once

#include "tmoe_block_norm.hpp"

namespace tmoe {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct NormPlan {
  int lanes;            // of a row in a wave, or 0: a row takes a work-group
  int steps;            // of 4 elements a lane, or of 16 bytes a thread
  unsigned threads;
  int teams;            // rows at a time in a work-group
  bool wide;            // the backward that reads a row twice, 4 elements a thread and step
};
// Whether a backward reads its rows twice (k_block_norm_bwd_wide) rather than hold them: by
// the elements a thread would hold, of work-groups of up to 768 or 1024 threads. Measured,
// held against read twice: gate, residual and all norms d = 9216, bf16, T = 4096 808 and
// 177 us, d = 8192 249 and 155 (fp32 392 and 258); residual and next norm d = 16384,
// T = 2048 248 and 119 (fp32 360 and 206). Where they are held without spills: d = 6144,
// bf16, T = 4096 86 and 121, fp32 with a next norm d = 8192 159 and 191.
constexpr bool norm_wide_rows(int held, int threads, bool full) {
  return held >= 16 || (full && held >= 8 && threads > 768);
}
// full: the backward with a gate or a norm after the block, whose rows of over 512 elements
// would need more registers than one wave's lanes have.
NormPlan norm_plan(int64_t d, int es, bool full, bool backward) {
  if (d <= (full ? 512 : 1024)) {
    const int lanes = d <= 64 ? 16 : d <= 128 ? 32 : 64;
    return {lanes, (int)ceil_div(d, 4 * lanes), dev::kNormThreads, dev::kNormThreads / lanes, false};
  }
  const int64_t nch = ceil_div(d * es, 16);
  const int c = nch <= 1024 ? 1 : nch <= 2048 ? 2 : 4;
  const unsigned threads = (unsigned)(ceil_div(nch, 64 * c) * 64);
  if (backward && norm_wide_rows(c * 16 / es, threads > 768 ? 1024 : 768, full)) {
    const int s = d <= 8192 ? 2 : d <= 12288 ? 3 : 4;
    return {0, s, (unsigned)(ceil_div(d, 256 * s) * 64), 1, true};
  }
  return {0, c, threads, 1, false};
}
// Work-groups of a persistent walk over the rows: what the chip holds at once.
int64_t norm_blocks(int64_t T, const NormPlan& p) {
  const int64_t n = ceil_div(T, p.teams);
  const int64_t most = p.threads <= 256 ? 2048 : p.threads <= 512 ? 1024 : 512;
  return n < most ? n : most;
}
// The backward's, with a plane of each weight's gradient for each: two to a compute unit
// (measured against 256, 768 and 1024: 119 us of T = 16384, d = 2304 with all operands
// against 114, 123 and 127, 25.7 against 26.6, 26.2 and 26.8 of d = 768 with a residual
// and the next norm). One for so few rows that a second launch would cost more than their
// walk.
int64_t norm_bwd_blocks(int64_t T, const NormPlan& p) {
  const int64_t n = ceil_div(T, p.teams);
  const int64_t most = p.threads <= 512 ? 512 : 256;   // of 1024 threads a unit holds one
  return n <= 2 ? 1 : n < most ? n : most;
}

using NormKernel = void (*)(BlockNormArgs);

// The form (F) of a backward whose rows' gradients are all wanted, else -1.
int norm_form(const BlockNormArgs& a) {
  using namespace dev;
  const bool all = a.dr && a.dy && (a.dh || !a.next_w) && (a.dx || !a.x) && (a.dgate || !a.gate);
  return !all ? -1
              : (a.gate ? kGate : 0) | (a.x ? kRes : 0) | (a.next_w ? kNext : 0) | (a.post_w ? kPost : 0);
}
template <class T, int EPC, int NCH, int kLanes, dev::RowEnd kEnd, int kThreads, bool kFull>
NormKernel norm_bwd_form(int form) {
  using namespace dev;
#define TMOE_FORM(F) \
  case F: return k_block_norm_bwd<T, EPC, NCH, kLanes, kEnd, kThreads, kFull, (F)>;
#define TMOE_FORMS(F) TMOE_FORM(F) TMOE_FORM(F | kRes) TMOE_FORM(F | kNext) TMOE_FORM(F | kRes | kNext)
  if constexpr (kThreads <= 512 && kEnd != kTiny) {
    if constexpr (kFull) switch (form) {
      TMOE_FORMS(kGate) TMOE_FORMS(kPost) TMOE_FORMS(kGate | kPost)
    }
    else switch (form) {
      TMOE_FORMS(0)
    }
  }
#undef TMOE_FORMS
#undef TMOE_FORM
  return k_block_norm_bwd<T, EPC, NCH, kLanes, kEnd, kThreads, kFull, -1>;
}
template <class T, dev::RowEnd kEnd, int NCH>
NormKernel norm_wide_form(int form) {
  using namespace dev;
  constexpr int kAll = kGate | kRes | kNext | kPost;
  if (form == (kRes | kNext)) return k_block_norm_bwd_wide<T, NCH, kEnd, kRes | kNext>;
  // four steps with every operand known spill as much as at run time, and take as long
  if constexpr (NCH < 4)
    if (form == kAll) return k_block_norm_bwd_wide<T, NCH, kEnd, kAll>;
  return k_block_norm_bwd_wide<T, NCH, kEnd, -1>;
}
template <class T, dev::RowEnd kEnd>
NormKernel norm_wide(int steps, int form) {
  switch (steps) {
    case 2: return norm_wide_form<T, kEnd, 2>(form);
    case 3: return norm_wide_form<T, kEnd, 3>(form);
    default: return norm_wide_form<T, kEnd, 4>(form);
  }
}
template <class T, dev::RowEnd kEnd>
NormKernel norm_kernel(const BlockNormArgs& a, bool backward, const NormPlan& p) {
  const bool full = a.gate || a.post_w;
  const int form = backward ? norm_form(a) : -1;
  if constexpr (kEnd != dev::kTiny)
    if (p.wide) return norm_wide<T, kEnd>(p.steps, form);
#define TMOE_NORM(EPC, C, LANES, THREADS)                                                     \
  if (p.lanes == LANES && p.steps == C && p.threads <= THREADS) {                             \
    if (!backward) return dev::k_block_norm_fwd<T, EPC, C, LANES, kEnd, THREADS>;            \
    if constexpr ((LANES == 0 || C <= 2) && !(LANES == 0 && norm_wide_rows(C * (EPC), THREADS, true))) \
      if (full) return norm_bwd_form<T, EPC, C, LANES, kEnd, THREADS, true>(form);           \
    if constexpr (!(LANES == 0 && norm_wide_rows(C * (EPC), THREADS, false)))                  \
      return norm_bwd_form<T, EPC, C, LANES, kEnd, THREADS, false>(form);                     \
  }
  constexpr int E16 = 16 / (int)sizeof(T);
  TMOE_NORM(4, 1, 16, 256)
  if constexpr (kEnd != dev::kTiny) {
    TMOE_NORM(4, 1, 32, 256)
    TMOE_NORM(4, 1, 64, 256) TMOE_NORM(4, 2, 64, 256)
    TMOE_NORM(4, 3, 64, 256) TMOE_NORM(4, 4, 64, 256)
    TMOE_NORM(E16, 1, 0, 512) TMOE_NORM(E16, 1, 0, 768) TMOE_NORM(E16, 1, 0, 1024)
    TMOE_NORM(E16, 2, 0, 768) TMOE_NORM(E16, 2, 0, 1024)
    if constexpr (sizeof(T) == 4) { TMOE_NORM(E16, 4, 0, 1024) }
  }
#undef TMOE_NORM
  return nullptr;
}
template <class T>
hipError_t norm_launch(const BlockNormArgs& a, bool backward, const NormPlan& p, int64_t blocks,
                       hipStream_t st) {
  const int epc = p.lanes || p.wide ? 4 : 16 / (int)sizeof(T);
  const NormKernel k = a.d < epc    ? norm_kernel<T, dev::kTiny>(a, backward, p)
                       : a.d % epc ? norm_kernel<T, dev::kOverlap>(a, backward, p)
                                   : norm_kernel<T, dev::kWhole>(a, backward, p);
  hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(p.threads), 0, st, a);
  return hipGetLastError();
}

}  // namespace

template <class T>
size_t block_norm_workspace(int64_t T_, int64_t d) {
  int64_t blocks = 1;
  for (bool full : {false, true}) {
    const int64_t n = norm_bwd_blocks(T_, norm_plan(d, sizeof(T), full, true));
    blocks = n > blocks ? n : blocks;
  }
  return blocks > 1 ? (size_t)(3 * blocks * d) * sizeof(float) : 0;
}
template <class T>
hipError_t block_norm_fwd(const BlockNormArgs& a, hipStream_t st) {
  const NormPlan p = norm_plan(a.d, sizeof(T), false, false);
  return norm_launch<T>(a, false, p, norm_blocks(a.T, p), st);
}
template <class T>
hipError_t block_norm_bwd(const BlockNormArgs& a, hipStream_t st) {
  const NormPlan p = norm_plan(a.d, sizeof(T), a.gate || a.post_w, true);
  const int64_t blocks = norm_bwd_blocks(a.T, p);
  if (a.T > 0)
    if (hipError_t e = norm_launch<T>(a, true, p, blocks, st); e != hipSuccess) return e;
  if ((!a.dpost_w && !a.dgamma && !a.dnext_w) || (a.T > 0 && blocks == 1)) return hipSuccess;
  // without rows the sums of no planes: zeros
  hipLaunchKernelGGL(dev::k_block_norm_cols<T>, dim3((unsigned)ceil_div(a.d, 32), 3), dim3(1024), 0,
                     st, a, a.T > 0 ? blocks : 0);
  return hipGetLastError();
}

#define TMOE_NORM_TYPE(T)                                                 \
  template size_t block_norm_workspace<T>(int64_t, int64_t);              \
  template hipError_t block_norm_fwd<T>(const BlockNormArgs&, hipStream_t); \
  template hipError_t block_norm_bwd<T>(const BlockNormArgs&, hipStream_t);

}  // namespace tmoe
