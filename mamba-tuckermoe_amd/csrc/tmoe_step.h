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

constexpr int64_t kFp8MaxDim = (int64_t)1 << 23;   // rows' bytes within a tile are counted in 32 bits

// x (R, C) to codes in blocks of 1 x 128 along its rows (row_codes), along its columns
// (col_codes, transposed: C rows of R padded to 128), or of 128 x 128 (tiles: both the same codes)
struct Fp8QuantizeArgs {
  const void* x;
  int64_t R, C, row_stride;
  int dtype, tiles;
  void* row_codes;
  float* row_scales;
  int64_t row_bytes, row_rs, row_ks;   // codes' rows; the scales' steps for a row and a block
  void* col_codes;
  float* col_scales;
  int64_t col_bytes, col_rs, col_ks;
};
hipError_t fp8_quantize(const Fp8QuantizeArgs& a, hipStream_t st);

struct Fp8GemmArgs {
  const void *a, *b;       // codes; a: with a_dtype values of M rows of K elements, a_bytes apart
  int64_t a_bytes, b_bytes;
  const float *sa, *sb;
  int64_t sa_rs, sa_ks, sb_rs, sb_ks;
  int a_tiles, b_tiles;    // scales of 128 rows each
  int a_dtype;             // -1: codes
  int64_t M, N, K;
  int blocks, slice_blocks, slices;
  int dtype;
  void* out;
  float* planes;           // workspace: (slices, M, N), null for one slice
};
bool fp8_gemm_takes_values(int64_t M, int64_t blocks);   // whether a may be values
size_t fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t blocks, int dtype);
hipError_t fp8_gemm(Fp8GemmArgs a, hipStream_t st);

constexpr int64_t kMuonMaxSide = (int64_t)1 << 22, kMuonMaxShort = (int64_t)1 << 16;

// A tensor of matrices (rows, cols). planes: each matrix's X, X', A and B (MuonPlanes)
struct MuonDesc {
  void* p;
  const void* g;
  float* m;                // null: u = g
  uint16_t* planes;
  int rows, cols;
  uint32_t chunk0, chunks; // the first of its chunks among the group's, and those of a matrix
  uint32_t tile0, gram0, sum0, sym0, app0;   // the first of its work-groups of each kind
  int slices, slice_tiles; // the Gram product's of its summed axis
  float rate;
};
constexpr int kMuonTensors = 48;     // of a group
struct MuonArgs {
  MuonDesc* t;             // the group's tensors, in the workspace
  double* sums;            // of a chunk's squares
  int count, cur, nesterov, write_only;
  float mu, eps, a, b, c, keep;
};
struct MuonFirstArgs {     // the first launch's, which writes them there
  MuonArgs a;
  MuonDesc t[kMuonTensors];
};
size_t muon_workspace_bytes(const tmoe_muon_tensor* t, int64_t count);
hipError_t muon(const tmoe_muon_tensor* t, int64_t count, const tmoe_muon_step_args& a, void* ws,
                hipStream_t st);

}  // namespace tmoe
