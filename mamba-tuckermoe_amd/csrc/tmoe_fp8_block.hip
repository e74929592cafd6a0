// Launchers of the 8-bit block products (tmoe_fp8_block.hpp).
#include "tmoe_fp8_block.hpp"

namespace tmoe {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kSkinnyRows = 32, kSkinnyWaves = 12;
constexpr int64_t kMaxSlices = 16;

constexpr int64_t kUnits = 256;       // compute units

struct Fp8Form {
  int bm = 0, slices = 1;             // tiles of bm x bm; 0: skinny
};
// Tiles of 256 x 256 (one work-group to a unit) or 128 x 128 (two), the latter with the summed axis
// in slices, by the least time of measured lines, in microseconds for a round of work-groups:
//   256 x 256, one scale for B's rows, bf16 results   2.0 a K tile + 4.4
//   128 x 128, one work-group to a unit (two)         0.85 (1.25) a K tile + 2.2, B's scales by row
//                                                     1.0 (1.35), fp32 results 1.25 (2.1)
//   adding s planes                                   4 + their bytes at 5.2 TB/s
// Measured, 256 x 256 against 128 x 128: M = N = K = 4096 69 and 86; M = 16384, N = 2304, K = 1024 63 and
// 54; N = 768, K = 4608 77 and 84. Slices: M = 512, N = 2048, K = 4096 one 29, two 21, four 18; M = 768,
// N = 4608, K = 16384 by row one 128, two 103, four 115. Of the other kinds of operands 256 x 256
// tiles need more registers than there are, and take 3.4 a K tile and more.
Fp8Form fp8_form(int64_t M, int64_t N, int64_t blocks, bool b_tiles, int dtype) {
  Fp8Form f;
  if (M <= kSkinnyRows) return f;
  const bool exact = dtype == TMOE_F32;
  const double one = exact ? 1.25 : b_tiles ? 0.85 : 1.0, two = exact ? 2.1 : b_tiles ? 1.25 : 1.35;
  const int64_t tiles = ceil_div(M, 128) * ceil_div(N, 128);
  double best = 0;
  f.bm = 128;
  for (int64_t want = 1; want <= kMaxSlices && want <= blocks; ++want) {
    const int64_t each = ceil_div(blocks, want), s = ceil_div(blocks, each), jobs = tiles * s;
    const int64_t rest = jobs % (2 * kUnits);
    double t = (double)(jobs / (2 * kUnits)) * (two * (double)each + 2.2);
    if (rest) t += (rest <= kUnits ? one : two) * (double)each + 2.2;
    if (s > 1) t += 4.0 + (double)((8 * s + (exact ? 4 : 2)) * M * N) / 5.2e6;
    if (want == 1 || t < best) {
      best = t;
      f.slices = (int)s;
    }
  }
  if (!exact && b_tiles) {
    const int64_t rounds = ceil_div(ceil_div(M, 256) * ceil_div(N, 256), kUnits);
    if ((double)rounds * (2.0 * (double)blocks + 4.4) < best) {
      f.bm = 256;
      f.slices = 1;
    }
  }
  return f;
}

template <int BM, int WM, int WN, bool kBRows, bool kExact>
void gemm_launch(const Fp8GemmArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(ceil_div(a.M, BM) * ceil_div(a.N, BM) * a.slices)), block(64 * WM * WN);
  hipLaunchKernelGGL((dev::k_fp8_gemm<BM, BM, WM, WN, kBRows, kExact>), grid, block, 0, st, a);
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

// A few rows are quantised within the product's launch where LDS holds them at once: eight rows of
// K = 4608 (288 blocks) take 11.2 us so and 14.0 in two launches, 16 of them (576) 15.3 and 14.7.
bool fp8_gemm_takes_values(int64_t M, int64_t blocks) { return M <= kSkinnyRows && M * blocks <= dev::kFp8Held; }
size_t fp8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t blocks, int dtype) {
  const int rows = fp8_form(M, N, blocks, false, dtype).slices, tiles = fp8_form(M, N, blocks, true, dtype).slices;
  const int slices = rows > tiles ? rows : tiles;
  return slices > 1 ? (size_t)slices * M * N * sizeof(float) : 0;
}

hipError_t fp8_gemm(Fp8GemmArgs a, hipStream_t st) {
  if (a.M == 0) return hipSuccess;
  const Fp8Form f = fp8_form(a.M, a.N, a.blocks, a.b_tiles, a.dtype);
  if (!f.bm) {
    if (a.a_dtype < 0) skinny_launch<uint8_t>(a, st);
    else if (a.a_dtype == TMOE_BF16) skinny_launch<uint16_t>(a, st);
    else skinny_launch<float>(a, st);
    return hipGetLastError();
  }
  a.slices = f.slices;
  a.slice_blocks = (int)ceil_div(a.blocks, f.slices);
  if (f.slices == 1) a.planes = nullptr;
  if (f.bm == 256) gemm_launch<256, 2, 4, false, false>(a, st);
  else if (a.dtype == TMOE_F32 && a.b_tiles) gemm_launch<128, 2, 2, false, true>(a, st);
  else if (a.dtype == TMOE_F32) gemm_launch<128, 2, 2, true, true>(a, st);
  else if (a.b_tiles) gemm_launch<128, 2, 2, false, false>(a, st);
  else gemm_launch<128, 2, 2, true, false>(a, st);
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
