// Products in 8-bit floating point (OCP e4m3) with one fp32 scale for each block of 128 along
// the summed axis, and the quantisation that makes their operands.
//
// Quantisation: over a block of 1 x 128 or 128 x 128 elements, top = max |x|,
//   scale = top / 448;  inv = 448 / top;  code = e4m3(x inv), to nearest, even on ties
// in fp32, and zeros where top <= 2^-100 (inv would leave fp32's range). A block with a value
// that is not finite stands for values that are not. k_fp8_quantize reads a 128 x 128 tile once
// and writes its codes along the rows, along the columns (transposed), or both: a training
// step's forward product sums over the columns of x and its weight gradient over the rows.
//
// Product: out[m, n] = sum_b sa[m, b] sb[n, b] sum_{k in block b} a[m, k] b[n, k], blocks
// added in fp32, a block's products by the matrix instruction (mma_fp8).
// One K tile of the LDS stages (128 bytes of a row) is one scale block, so that a K tile is two
// v_mfma_f32_32x32x64_f8f6f4 from a zero accumulator for each 32 x 32 block, and its result is
// added to the sums with its scale by 16 (one scale a row; B's scale by a row too: 32) vector
// instructions of 4 cycles beside 128 of the matrix unit.
#pragma once

#include "tmoe_mma.hpp"
#include "tmoe_step.h"

namespace tmoe {
namespace dev {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kFp8Tiny = 0x0d800000u;       // 2^-100
constexpr int kFp8Block = 128;
constexpr int kFp8Held = 512;                    // blocks of a few rows' values that one launch quantises itself

__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
struct Fp8Scale {
  float scale, inv;
  // bits of the largest magnitude, those of NaN above all
  __device__ __forceinline__ explicit Fp8Scale(uint32_t top) {
    const float t = __uint_as_float(top);
    const bool some = top > kFp8Tiny;
    scale = some ? t / 448.f : 0.f;
    inv = some ? 448.f / t : 0.f;
  }
};

// 8 consecutive elements of a row from column c on (zeros past C), at any alignment
template <class T>
__device__ __forceinline__ void fp8_load8(const T* row, int64_t c, int64_t C, float (&v)[8]) {
  constexpr int W = 8 * (int)sizeof(T) / 4;
  typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  if (c + 8 <= C) {
    const vec q = *reinterpret_cast<const vec*>(row + c);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(q[j]);
      else v[j] = __uint_as_float(j & 1 ? q[j / 2] & 0xffff0000u : q[j / 2] << 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < C ? load_as_f32(row + c + j) : 0.f;
  }
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// One 128 x 128 tile: 256 threads, 16 of them to a row, eight columns each; a thread's rows are
// two runs of four, so that four codes of a column are one word of the transposed tile. Bound by
// memory: along both axes (16384, 4608) bf16 takes 73 us, 4.2 TB/s, (16384, 768) 13.9, (5003, 1536) fp32
// 12.4; along the rows alone the first 50 us, 4.6 TB/s.
template <class T, bool kTiles>
__global__ __launch_bounds__(256) void k_fp8_quantize(Fp8QuantizeArgs a) {
  __shared__ uint32_t s_t[128 * 32];             // transposed codes: a column's 128 bytes a row
  __shared__ uint32_t s_top[4][128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int cc = tid & 15, rr = tid >> 4;        // columns 8 cc .., rows 4 rr .. and 64 + 4 rr ..
  const int64_t tiles_c = (a.C + 127) / 128, rb = blockIdx.x / tiles_c, cb = blockIdx.x - rb * tiles_c;
  const int64_t r0 = rb * 128, c0 = cb * 128, c = c0 + 8 * cc;
  const T* x = static_cast<const T*>(a.x);
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + (i >> 2) * 64 + rr * 4 + (i & 3);
    if (r < a.R) {
      fp8_load8(x + r * a.row_stride, c, a.C, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  auto bits = [](float f) { return __float_as_uint(f) & 0x7fffffffu; };
  auto lanes16 = [](uint32_t t) { return lanes_max<16>(t); };
  uint32_t tile_top = 0u;
  if constexpr (kTiles) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) tile_top = umax(tile_top, bits(v[i][j]));
    tile_top = lanes_max<64>(tile_top);
    if (lane == 0) s_top[0][wave] = tile_top;
    __syncthreads();
    tile_top = umax(umax(s_top[0][0], s_top[0][1]), umax(s_top[0][2], s_top[0][3]));
  }
  const Fp8Scale tile(tile_top);
  if (kTiles && tid == 0) a.row_scales[rb * a.row_rs + cb * a.row_ks] = tile.scale;
  if (a.row_codes) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = r0 + (i >> 2) * 64 + rr * 4 + (i & 3);
      Fp8Scale s = tile;
      if constexpr (!kTiles) {
        uint32_t top = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = umax(top, bits(v[i][j]));
        s = Fp8Scale(lanes16(top));
      }
      if (r >= a.R) continue;
      if (!kTiles && cc == 0) a.row_scales[r * a.row_rs + cb * a.row_ks] = s.scale;
      uint2 q;
      q.x = pack_fp8x4(v[i][0] * s.inv, v[i][1] * s.inv, v[i][2] * s.inv, v[i][3] * s.inv);
      q.y = pack_fp8x4(v[i][4] * s.inv, v[i][5] * s.inv, v[i][6] * s.inv, v[i][7] * s.inv);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.row_codes) + r * a.row_bytes + c) = q;
    }
  }
  if (!a.col_codes) return;
  float inv[8];
  if constexpr (kTiles) {
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = tile.inv;
  } else {
    uint32_t top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      top[j] = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) top[j] = umax(top[j], bits(v[i][j]));
      top[j] = umax(top[j], __shfl_xor(top[j], 16));
      top[j] = umax(top[j], __shfl_xor(top[j], 32));
    }
    if (lane < 16)
#pragma unroll
      for (int j = 0; j < 8; ++j) s_top[wave][8 * cc + j] = top[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const Fp8Scale s(umax(umax(s_top[0][8 * cc + j], s_top[1][8 * cc + j]),
                            umax(s_top[2][8 * cc + j], s_top[3][8 * cc + j])));
      inv[j] = s.inv;
      if (rr == 0 && c + j < a.C)
        a.col_scales[(c + j) * a.col_rs + rb * a.col_ks] = s.scale;
    }
  }
  // word (column, four rows) at chunk ^ (column / 8): the 64 words that a wave writes at once
  // lie in 32 banks, and a column's 16-byte chunks are read whole
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int word = h * 16 + rr;
      s_t[(8 * cc + j) * 32 + ((((word >> 2) ^ (cc & 7)) << 2) | (word & 3))] =
          pack_fp8x4(v[4 * h][j] * inv[j], v[4 * h + 1][j] * inv[j], v[4 * h + 2][j] * inv[j],
                     v[4 * h + 3][j] * inv[j]);
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = tid + i * 256, col = q >> 3, ch = q & 7;
    if (c0 + col < a.C)
      *reinterpret_cast<u32x4*>(static_cast<uint8_t*>(a.col_codes) + (c0 + col) * a.col_bytes + r0 + ch * 16) =
          *reinterpret_cast<const u32x4*>(s_t + col * 32 + ((ch ^ ((col >> 3) & 7)) << 2));
  }
}

// ---- the product -------------------------------------------------------------------

// eight codes as bf16, which holds each of them
__device__ __forceinline__ bf16x8 bf16_of(int lo, int hi) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  return __builtin_bit_cast(bf16x8, r);
}
// The 8-bit instruction adds its products in groups (of 16 at most) in which each is cut at 2^-13
// of the largest: measured, a product of 2^-13 of its neighbour counts and one of 2^-14 is lost,
// while 2^-23 counts between groups and to the accumulator. Random rows of 128 come out 4e-6 of
// their magnitudes' sum off, a five-hundredth of the rounding of a bf16 result, which take it: with
// fp32 sums they are as far from the float64 product (1.662e-3 in the norm at M = N = K = 4096, 1.657e-3 at
// 16384 x 4608 x 768, either way) and take 159 us instead of 79 there, 144 instead of 85 here (one
// row of 1536 to 6144: 5.2 and 4.9). fp32 results (kExact) are summed in fp32: the codes as bf16, whose
// instruction keeps all 24 bits, at half the rate.
template <bool kExact>
__device__ __forceinline__ f32x16 mma_fp8(i32x8 a, i32x8 b, f32x16 c) {
  if constexpr (kExact) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bf16_of(a[2 * j], a[2 * j + 1]), bf16_of(b[2 * j], b[2 * j + 1]),
                                                  c, 0, 0, 0);
    return c;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
  }
}
__device__ __forceinline__ i32x8 join8(u32x4 lo, u32x4 hi) {
  i32x8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r[j] = (int)lo[j];
    r[4 + j] = (int)hi[j];
  }
  return r;
}

// Stores a wave's 32 x (32 FN) block from its own LDS, rows in the lanes' order of acc (lane: row
// l & 31, elements: columns 8 q + 4 (l >> 5) ..): 16-byte pieces of rows where all of them are
// aligned, else elements. Past the caches (M = 16384, N = 2304, K = 1024 with its quantisation 66 us, 71
// through them; the step at 768 to 4608 347 and 376): the next launches' operands stay there.
template <class T, int FN>
__device__ __forceinline__ void fp8_store(const f32x16 (&acc)[FN], char* stage, T* out, int64_t ld,
                                          int64_t row0, int64_t rows, int64_t col0, int64_t cols, bool wide) {
  constexpr int RB = 32 * FN * (int)sizeof(T) + 16, CPR = 32 * FN * (int)sizeof(T) / 16;
  constexpr int EPC = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 63;
  char* mine = stage + (lane & 31) * RB;
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = j * 32 + 8 * q + 4 * (lane >> 5);
      if constexpr (sizeof(T) == 2) {
        uint2 v;
        v.x = pack_bf16x2(acc[j][4 * q], acc[j][4 * q + 1]);
        v.y = pack_bf16x2(acc[j][4 * q + 2], acc[j][4 * q + 3]);
        *reinterpret_cast<uint2*>(mine + col * 2) = v;
      } else {
        *reinterpret_cast<float4*>(mine + col * 4) =
            float4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
      }
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (wide) {
    for (int c = lane; c < 32 * CPR; c += 64) {
      const int r = c / CPR, ch = c % CPR;
      if (row0 + r < rows && col0 + ch * EPC < cols)
        __builtin_nontemporal_store(*reinterpret_cast<const u32x4*>(stage + r * RB + ch * 16),
                                    reinterpret_cast<u32x4*>(out + (row0 + r) * ld + col0 + ch * EPC));
    }
  } else {
    for (int c = lane; c < 32 * 32 * FN; c += 64) {
      const int r = c / (32 * FN), e = c % (32 * FN);
      if (row0 + r < rows && col0 + e < cols)
        out[(row0 + r) * ld + col0 + e] = *reinterpret_cast<const T*>(stage + r * RB + e * sizeof(T));
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// BM x BN tiles, WM x WN waves, two LDS stages filled by direct loads: tile kt + 1 is on its way
// while tile kt is computed.
template <int BM, int BN, int WM, int WN, bool kBRows>
struct Fp8Tile {
  static constexpr int kThreads = 64 * WM * WN, W = WM * WN;
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
  static constexpr int kScales = BM + (kBRows ? BN : 64);       // floats
  static constexpr int kStageBytes = (BM + BN) * 128 + kScales * 4;
  static constexpr int kLdsBytes = 2 * kStageBytes;
  static constexpr int kStoreBytes = W * 32 * (32 * FN * 4 + 16);
  static constexpr int kSmem = kLdsBytes > kStoreBytes ? kLdsBytes : kStoreBytes;
  static_assert(BM % (32 * WM) == 0 && BN % (32 * WN) == 0 && BN / WN <= 128 && 128 % (BN / WN) == 0, "");
  static_assert((BM + BN) / 8 % W == 0 && kSmem <= 160 * 1024, "");
};

// A tile's product: a K tile's two matrix instructions for each block of 32 x 32 begin from zero and
// what they give is added with its scales. Of 128 x 128 two work-groups share a compute unit, so that
// one computes while the other waits or stores; of 256 x 256 (alone there, for its stages) the LDS
// reads a product are half. Bound by those reads and the scales' multiply-adds beside the matrix units
// (at work 32 to 39% of the time, the vector units 39 to 57%): M = N = K = 4096 66 us, 2.1 PFLOP/s; M =
// 16384, N = 2304, K = 1024 59, 1.3, its results 75 of its 95 MB; M = 768, N = 4608, K = 16384 by rows 97 with
// the planes' sum.
template <int BM, int BN, int WM, int WN, bool kBRows, bool kExact>
__global__ __launch_bounds__(64 * WM * WN) void k_fp8_gemm(Fp8GemmArgs a) {
  using TL = Fp8Tile<BM, BN, WM, WN, kBRows>;
  constexpr int FM = TL::FM, FN = TL::FN, W = TL::W;
  __shared__ u32x4 s_mem[TL::kSmem / 16];
  char* smem = reinterpret_cast<char*>(s_mem);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_n = (int)((a.N + BN - 1) / BN), tiles = tiles_n * (int)((a.M + BM - 1) / BM);
  const int slice = blockIdx.x / tiles;
  int tm, tn;
  tile_coords_of(blockIdx.x - slice * tiles, tiles_n, tiles, tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int kt0 = slice * a.slice_blocks, kt1 = cmin_dev(kt0 + a.slice_blocks, a.blocks);
  const int mv = (int)(a.M - m0 < BM ? a.M - m0 : BM), nv = (int)(a.N - n0 < BN ? a.N - n0 : BN);
  const char* ap = static_cast<const char*>(a.a) + m0 * a.a_bytes;
  const char* bp = static_cast<const char*>(a.b) + n0 * a.b_bytes;

  auto load = [&](int kt, int st) __attribute__((always_inline)) {
    char* s = smem + st * TL::kStageBytes;
#pragma unroll
    for (int i = 0; i < (BM + BN) / 8 / W; ++i) {
      const int blk = wave + i * W;              // 8 rows; A's first
      const int ch = dma_chunk(lane, blk);
      const bool isa = blk < BM / 8;
      const int r = (isa ? blk : blk - BM / 8) * 8 + (lane >> 3);
      const int rc = cmin_dev(r, (isa ? mv : nv) - 1);
      const char* g = (isa ? ap : bp) + ((uint32_t)rc * (uint32_t)(isa ? a.a_bytes : a.b_bytes) +
                                         (uint32_t)(kt * 128 + ch * 16));
      __builtin_amdgcn_global_load_lds((gbl_cvptr)g, (lds_vptr)(s + blk * 1024), 16, 0, 0);
    }
    char* sc = s + (BM + BN) * 128;
    constexpr int kA = BM / 64, kB = kBRows ? BN / 64 : 1;
#pragma unroll
    for (int i = 0; i < (kA + kB + W - 1) / W; ++i) {
      const int q = wave + i * W;
      if (q < kA) {
        const int64_t r = m0 + cmin_dev(q * 64 + lane, mv - 1);
        const float* g = a.sa + (a.a_tiles ? r / kFp8Block : r) * a.sa_rs + kt * a.sa_ks;
        __builtin_amdgcn_global_load_lds((gbl_cvptr)g, (lds_vptr)(sc + q * 256), 4, 0, 0);
      } else if (q < kA + kB) {
        const int64_t r = n0 + cmin_dev(kBRows ? (q - kA) * 64 + lane : cmin_dev(lane, BN / 128 - (BN < 128 ? 0 : 1)) * 128, nv - 1);
        const float* g = a.sb + (kBRows ? r : r / kFp8Block) * a.sb_rs + kt * a.sb_ks;
        __builtin_amdgcn_global_load_lds((gbl_cvptr)g, (lds_vptr)(sc + BM * 4 + (q - kA) * 256), 4, 0, 0);
      }
    }
  };

  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = zero16();

  load(kt0, 0);
  for (int kt = kt0; kt < kt1; ++kt) {
    const int st = (kt - kt0) & 1;
    wait_vm_lds<0>();
    lds_barrier();
    if (kt + 1 < kt1) load(kt + 1, st ^ 1);
    const u32x4* s = reinterpret_cast<const u32x4*>(smem + st * TL::kStageBytes);
    const float* sc = reinterpret_cast<const float*>(smem + st * TL::kStageBytes + (BM + BN) * 128);
    i32x8 bf[FN][2];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = BM + wn * FN * 32 + j * 32 + (lane & 31);
        bf[j][k] = join8(s[lds_slot(r, 4 * k + (lane >> 5))], s[lds_slot(r, 4 * k + 2 + (lane >> 5))]);
      }
    // B's scales: one, or those of the columns that the lane's elements lie in. These are read by
    // assembly with its wait: the compiler takes them for what the loads in flight write and waits
    // for those (M = 768, N = 4608, K = 16384: 120 us so, 103 as it is).
    float sb1 = 0.f;
    u32x4 sb[kBRows ? FN : 1][4];
    if constexpr (kBRows) {
      static_assert(FN == 2, "the reads below");
      const uint32_t at = (uint32_t)(size_t)(lds_vptr)(smem + st * TL::kStageBytes + (BM + BN) * 128) +
                          (BM + wn * FN * 32) * 4 + (lane >> 5) * 16;
      asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:32\n\tds_read_b128 %2, %8 offset:64\n\t"
                   "ds_read_b128 %3, %8 offset:96\n\tds_read_b128 %4, %8 offset:128\n\tds_read_b128 %5, %8 offset:160\n\t"
                   "ds_read_b128 %6, %8 offset:192\n\tds_read_b128 %7, %8 offset:224\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(sb[0][0]), "=&v"(sb[0][1]), "=&v"(sb[0][2]), "=&v"(sb[0][3]), "=&v"(sb[1][0]),
                     "=&v"(sb[1][1]), "=&v"(sb[1][2]), "=&v"(sb[1][3])
                   : "v"(at) : "memory");
    } else {
      sb1 = sc[BM + wn * FN * 32 / 128];
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      i32x8 af[2];
      const int r = wm * FM * 32 + i * 32 + (lane & 31);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        af[k] = join8(s[lds_slot(r, 4 * k + (lane >> 5))], s[lds_slot(r, 4 * k + 2 + (lane >> 5))]);
      const float sa1 = kBRows ? sc[r] : sc[r] * sb1;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        f32x16 t = mma_fp8<kExact>(bf[j][0], af[0], zero16());
        t = mma_fp8<kExact>(bf[j][1], af[1], t);
        if constexpr (kBRows) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            acc[i][j][e] = fmaf(t[e], sa1 * __uint_as_float(sb[j][e / 4][e % 4]), acc[i][j][e]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] = fmaf(t[e], sa1, acc[i][j][e]);
        }
      }
    }
  }
  wait_vm_lds<0>();
  lds_barrier();                                 // the stages are read: the stores may use them
  char* mine = smem + wave * 32 * (32 * FN * 4 + 16);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t row0 = m0 + wm * FM * 32 + i * 32, col0 = n0 + wn * FN * 32;
    if (a.planes) {
      float* p = a.planes + (int64_t)slice * a.M * a.N;
      fp8_store<float, FN>(acc[i], mine, p, a.N, row0, a.M, col0, a.N, a.N % 4 == 0);
    } else if (a.dtype == TMOE_BF16) {
      fp8_store<uint16_t, FN>(acc[i], mine, static_cast<uint16_t*>(a.out), a.N, row0, a.M, col0, a.N, a.N % 8 == 0);
    } else {
      fp8_store<float, FN>(acc[i], mine, static_cast<float*>(a.out), a.N, row0, a.M, col0, a.N, a.N % 4 == 0);
    }
  }
}

// out = the sum of the planes, in their order; 4.2 us for ten of 1536 x 256, 8 for two of 768 x 4608
template <class T>
__global__ __launch_bounds__(256) void k_fp8_sum(const float* __restrict__ planes, int n, int64_t count,
                                                 T* __restrict__ out) {
  const int64_t step = (int64_t)gridDim.x * 256 * 4;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += step) {
    if (i + 4 <= count && count % 4 == 0) {
      float4 t = *reinterpret_cast<const float4*>(planes + i);
      for (int p = 1; p < n; p += 5) {           // five loads at once
        float4 u[5];
#pragma unroll
        for (int k = 0; k < 5; ++k)
          u[k] = p + k < n ? *reinterpret_cast<const float4*>(planes + (p + k) * count + i) : float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 5; ++k) {
          t.x += u[k].x; t.y += u[k].y; t.z += u[k].z; t.w += u[k].w;
        }
      }
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(out + i) = uint2{pack_bf16x2(t.x, t.y), pack_bf16x2(t.z, t.w)};
      else
        *reinterpret_cast<float4*>(out + i) = t;
    } else {
      for (int64_t e = i; e < count && e < i + 4; ++e) {
        float t = planes[e];
        for (int p = 1; p < n; ++p) t += planes[p * count + e];
        store_from_f32(out + e, t);
      }
    }
  }
}

// Up to 32 rows against all of B, read once straight into registers: a work-group takes 32
// columns, its waves a K tile each, the next one's codes on their way. A's rows are codes, or (T)
// bf16 or fp32 values of kFp8Held blocks at most, which the work-group first quantises into LDS (by
// each wave for itself, from its rows' lanes, that took 3.2 us a K tile; W tiles at a time between
// the products it waited for B's codes too). Bound by latency: M = 1, K = 1536, N = 6144 takes 5.3 us, of
// which the launch is 2 and reading 9.4 MB 1.8.
template <class T, int W, bool kExact>
__global__ __launch_bounds__(64 * W) void k_fp8_skinny(Fp8GemmArgs a) {
  constexpr bool kCodes = sizeof(T) == 1;
  __shared__ u32x4 s_codes[kCodes ? 1 : kFp8Held * 8 + 32];
  __shared__ float s_scales[kCodes ? 1 : kFp8Held];
  __shared__ float s_part[W][32][33];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, h = lane >> 5;
  const int M = (int)a.M, blocks = a.blocks;
  const int64_t n0 = (int64_t)blockIdx.x * 32;
  const int64_t n = n0 + r < a.N ? n0 + r : a.N - 1;
  const bool live = r < M;
  // the codes of a row's K tile that the lane holds
  auto codes = [&](const void* row, int64_t at, i32x8 (&f)[2]) __attribute__((always_inline)) {
    const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const char*>(row) + at);
#pragma unroll
    for (int k = 0; k < 2; ++k) f[k] = join8(p[4 * k + h], p[4 * k + 2 + h]);
  };
  const char* bp = static_cast<const char*>(a.b) + n * a.b_bytes;
  i32x8 next[2] = {};
  if (wave < blocks) codes(bp, (int64_t)wave * 128, next);
  const int row_bytes = blocks * 128 + 16;       // of LDS (rows in other banks)
  if constexpr (!kCodes) {                       // 16 lanes to a block, the blocks of a K tile neighbours
    const int c = 8 * (tid & 15);
    int blk = (tid >> 4) / M, row = (tid >> 4) - blk * M;
#pragma unroll 1
    while (blk < blocks) {
      float v[8];
      fp8_load8(static_cast<const T*>(a.a) + row * a.a_bytes, (int64_t)blk * 128 + c, a.K, v);
      uint32_t top = 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = umax(top, __float_as_uint(v[j]) & 0x7fffffffu);
      const Fp8Scale s(lanes_max<16>(top));
      *reinterpret_cast<uint2*>(reinterpret_cast<char*>(s_codes) + row * row_bytes + blk * 128 + c) =
          uint2{pack_fp8x4(v[0] * s.inv, v[1] * s.inv, v[2] * s.inv, v[3] * s.inv),
                pack_fp8x4(v[4] * s.inv, v[5] * s.inv, v[6] * s.inv, v[7] * s.inv)};
      if (c == 0) s_scales[blk * M + row] = s.scale;
      row += 4 * W % M;
      blk += 4 * W / M;
      if (row >= M) {
        row -= M;
        ++blk;
      }
    }
    wait_vm_lds<63>();                           // (LDS alone: B's codes stay on their way)
    lds_barrier();
  }
  f32x16 acc = zero16();
#pragma unroll 1
  for (int kt = wave; kt < blocks; kt += W) {
    const i32x8 bf[2] = {next[0], next[1]};
    if (kt + W < blocks) codes(bp, (int64_t)(kt + W) * 128, next);
    float sb[16];
    if (a.b_tiles) {
      sb[0] = a.sb[n0 / kFp8Block * a.sb_rs + kt * a.sb_ks];
#pragma unroll
      for (int e = 1; e < 16; ++e) sb[e] = sb[0];
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t col = n0 + 8 * (e >> 2) + 4 * h + (e & 3);
        sb[e] = a.sb[(col < a.N ? col : a.N - 1) * a.sb_rs + kt * a.sb_ks];
      }
    }
    i32x8 af[2] = {};
    float sa = 0.f;
    if (live) {
      if constexpr (kCodes) {
        codes(a.a, r * a.a_bytes + (int64_t)kt * 128, af);
        sa = a.sa[(a.a_tiles ? 0 : r) * a.sa_rs + kt * a.sa_ks];
      } else {
        codes(s_codes, r * row_bytes + kt * 128, af);
        sa = s_scales[kt * M + r];
      }
    }
    f32x16 t = mma_fp8<kExact>(bf[0], af[0], zero16());
    t = mma_fp8<kExact>(bf[1], af[1], t);
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = fmaf(t[e], sa * sb[e], acc[e]);
  }
  if (live)
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) s_part[wave][r][8 * q + 4 * h + e] = acc[4 * q + e];
  __syncthreads();
  // an output of 32 columns a thread, the waves' sums in their order
  for (int i = threadIdx.x; i < a.M * 32; i += 64 * W) {
    const int row = i >> 5, col = i & 31;
    if (n0 + col >= a.N) continue;
    float t = s_part[0][row][col];
#pragma unroll
    for (int w = 1; w < W; ++w) t += s_part[w][row][col];
    if (a.dtype == TMOE_BF16) store_from_f32(static_cast<uint16_t*>(a.out) + row * a.N + n0 + col, t);
    else store_from_f32(static_cast<float*>(a.out) + row * a.N + n0 + col, t);
  }
}

}  // namespace dev
}  // namespace tmoe
