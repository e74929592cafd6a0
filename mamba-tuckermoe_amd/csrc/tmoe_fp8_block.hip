// Launchers of the 8-bit block products (tmoe_fp8_block.hpp).
#include "tmoe_fp8_block.hpp"

namespace tmoe {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kSkinnyRows = 32, kSkinnyWaves = 8;
constexpr int64_t kMaxSlices = 16;

struct Fp8Form {
  int bm = 0, bn = 0, slices = 1;     // bm 0: skinny
};
Fp8Form fp8_form(int64_t M, int64_t N, int64_t blocks) {
  Fp8Form f;
  if (M <= kSkinnyRows) return f;
  if (ceil_div(M, 256) * ceil_div(N, 256) >= 200) {
    f.bm = f.bn = 256;
    return f;
  }
  f.bm = f.bn = 128;
  const int64_t tiles = ceil_div(M, 128) * ceil_div(N, 128);
  int64_t s = 512 / tiles;
  if (s > blocks / 2) s = blocks / 2;
  if (s > kMaxSlices) s = kMaxSlices;
  if (s < 1) s = 1;
  f.slices = (int)ceil_div(blocks, ceil_div(blocks, s));
  return f;
}

template <int BM, int BN, int WM, int WN>
void gemm_launch(const Fp8GemmArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(ceil_div(a.M, BM) * ceil_div(a.N, BN) * a.slices)), block(64 * WM * WN);
#define TMOE_FP8(ROWS, EXACT) hipLaunchKernelGGL((dev::k_fp8_gemm<BM, BN, WM, WN, ROWS, EXACT>), grid, block, 0, st, a)
  const bool exact = a.dtype == TMOE_F32;
  if (a.b_tiles) { if (exact) TMOE_FP8(false, true); else TMOE_FP8(false, false); }
  else { if (exact) TMOE_FP8(true, true); else TMOE_FP8(true, false); }
#undef TMOE_FP8
}
template <class T>
void skinny_launch(const Fp8GemmArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.N, 32)), block(64 * kSkinnyWaves);
  if (a.dtype == TMOE_F32) hipLaunchKernelGGL((dev::k_fp8_skinny<T, kSkinnyWaves, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((dev::k_fp8_skinny<T, kSkinnyWaves, false>), grid, block, 0, st, a);
}

}  // namespace

hipError_t fp8_quantize(const Fp8QuantizeArgs& a, hipStream_t st) {
  const int64_t n = ceil_div(a.R, 128) * ceil_div(a.C, 128);
  if (n == 0) return hipSuccess;
  const dim3 grid((unsigned)n), block(256);
  if (a.dtype == TMOE_BF16) {
    if (a.tiles) hipLaunchKernelGGL((dev::k_fp8_quantize<uint16_t, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((dev::k_fp8_quantize<uint16_t, false>), grid, block, 0, st, a);
  } else {
    if (a.tiles) hipLaunchKernelGGL((dev::k_fp8_quantize<float, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((dev::k_fp8_quantize<float, false>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}

int64_t fp8_gemm_skinny_rows() { return kSkinnyRows; }
size_t fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t blocks) {
  const Fp8Form f = fp8_form(M, N, blocks);
  return f.slices > 1 ? (size_t)f.slices * M * N * sizeof(float) : 0;
}

hipError_t fp8_gemm(Fp8GemmArgs a, hipStream_t st) {
  if (a.M == 0) return hipSuccess;
  const Fp8Form f = fp8_form(a.M, a.N, a.blocks);
  if (!f.bm) {
    if (a.a_dtype < 0) skinny_launch<uint8_t>(a, st);
    else if (a.a_dtype == TMOE_BF16) skinny_launch<uint16_t>(a, st);
    else skinny_launch<float>(a, st);
    return hipGetLastError();
  }
  a.slices = f.slices;
  a.slice_blocks = (int)ceil_div(a.blocks, f.slices);
  if (f.slices == 1) a.planes = nullptr;
  if (f.bm == 256) gemm_launch<256, 256, 2, 4>(a, st);
  else gemm_launch<128, 128, 2, 2>(a, st);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || f.slices == 1) return e;
  const int64_t count = a.M * a.N, groups = ceil_div(count, 1024);
  const dim3 grid((unsigned)(groups < 4096 ? groups : 4096)), block(256);
  if (a.dtype == TMOE_BF16)
    hipLaunchKernelGGL(dev::k_fp8_sum<uint16_t>, grid, block, 0, st, a.planes, f.slices, count, static_cast<uint16_t*>(a.out));
  else
    hipLaunchKernelGGL(dev::k_fp8_sum<float>, grid, block, 0, st, a.planes, f.slices, count, static_cast<float*>(a.out));
  return hipGetLastError();
}

}  // namespace tmoe
