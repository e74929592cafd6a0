// The Muon step over many tensors, and orthogonalisation alone. For a matrix of a parameter with
// gradient g and momentum m:
//   m = mu m + g;  u = g + mu m (nesterov) or m;  X = u / (|u| + eps), transposed where it is tall
//   steps times: A = X X^T;  B = b A + c A A;  X = a X + B X
//   p = p (1 - lr wd) - lr rms sqrt(max(rows, cols)) X
//
// The polynomial a x + b x^3 + c x^5 takes every singular value towards one, the small ones by
// its slope at zero: 3.4445^5 = 485 in five steps, and with them what X was rounded by. So X, A
// and B are held as two fp16 numbers each (22 bits; all of them times 2^11, which keeps the
// second one out of fp16's smallest numbers), and a product is three matrix instructions: high
// high, high low and low high, fp32 sums. One bf16 number instead puts the update 1e-2 off.
//
// A launch takes all matrices of a group of tensors: a work-group finds its tile's tensor in a
// table in the workspace. A and B, symmetric, are computed by half and stored twice. X lies as its
// parameter does, its symmetric products along either axis: what is summed over rows (a tall
// matrix's X^T X, a wide one's B X) is read transposed from LDS. B holds a on its diagonal as well,
// so that X' = B X and nothing else is read.
//
// Small groups are bound by launches: a step of three matrices of up to 256 x 1024 is 22 of them, of
// 4 to 6 us. Large ones by memory and matrix units together: 66 layers (2112 matrices of 256 x 512
// and 139 M elements of wider ones, in float32) take 14.3 ms, of it the third products 6.6 (the bytes
// of X, X' and the parameters alone 3.5 at a copy's rate, three fp16 products at the library's rate 3.2), the Gram
// products 3.6, B 2.1, and the two passes before them 1.8.
#pragma once

#include "tmoe_mma.hpp"
#include "tmoe_step.h"

namespace tmoe {
namespace dev {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMuonThreads = 256;
constexpr float kMuonOne = 2048.f;             // what 1 is stored as
constexpr int kMuonChunk = 8192;               // elements of a work-group of k_muon_momentum

__device__ __forceinline__ f32x16 mma_f16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                0, 0, 0);
}
// eight values as their high and low parts
__device__ __forceinline__ void split8(const float (&v)[8], u32x4& hi, u32x4& lo) {
  f16x8 h, l;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // Both parts of one rounded value. Where it is a product, the compiler otherwise makes the high
    // part of the unrounded one too, and beside a tie the two lie on different sides.
    float x = v[j];
    asm volatile("" : "+v"(x));
    h[j] = (_Float16)x;
    l[j] = (_Float16)(x - (float)h[j]);
  }
  hi = __builtin_bit_cast(u32x4, h);
  lo = __builtin_bit_cast(u32x4, l);
}
__device__ __forceinline__ void join8f(u32x4 hi, u32x4 lo, float (&v)[8]) {
  const f16x8 h = __builtin_bit_cast(f16x8, hi), l = __builtin_bit_cast(f16x8, lo);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)h[j] + (float)l[j];
}

// The last tensor whose first work-group (of the kind that `first` gives) is no later than `tile`. A
// whole wave's call: each lane loads one tensor's entry, and the one that a ballot finds is
// broadcast, so that no load waits for which it is.
template <class F>
__device__ __forceinline__ MuonDesc muon_take(const MuonDesc* t, int count, uint32_t tile, F first) {
  constexpr int W = sizeof(MuonDesc) / 4;
  static_assert(kMuonTensors <= 64 && sizeof(MuonDesc) % 4 == 0, "a lane a tensor");
  struct Words {
    uint32_t w[W];
  };
  const int lane = threadIdx.x & 63;
  const MuonDesc mine = t[cmin_dev(lane, count - 1)];
  const int k = 63 - __clzll(__ballot(lane < count && first(mine) <= tile));     // (lane 0's always is)
  Words u = __builtin_bit_cast(Words, mine);
#pragma unroll
  for (int i = 0; i < W; ++i) u.w[i] = __builtin_amdgcn_readlane(u.w[i], k);
  return __builtin_bit_cast(MuonDesc, u);
}

__device__ __forceinline__ float muon_u(float g, float m, float mu, bool nesterov) {
  return nesterov ? fmaf(mu, m, g) : m;
}

// eight consecutive elements of a row of which n are there (zeros, and nothing stored, past them),
// at any alignment
template <class T>
__device__ __forceinline__ void muon_load8(const T* p, int64_t n, float (&v)[8]) {
  constexpr int W = 8 * (int)sizeof(T) / 4;
  typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  if (n >= 8) {
    const vec q = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(q[j]);
      else v[j] = __uint_as_float(j & 1 ? q[j / 2] & 0xffff0000u : q[j / 2] << 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? load_as_f32(p + j) : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void muon_store8(T* p, int64_t n, const float (&v)[8]) {
  constexpr int W = 8 * (int)sizeof(T) / 4;
  typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  if (n >= 8) {
    vec q;
#pragma unroll
    for (int j = 0; j < W; ++j)
      if constexpr (sizeof(T) == 4) q[j] = __float_as_uint(v[j]);
      else q[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<vec*>(p) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) store_from_f32(p + j, v[j]);
  }
}

// a matrix's planes in the workspace: X (high, low) and X', then A and B
struct MuonPlanes {
  int rp, cp, m;           // X's rows and columns, padded to 64, and the smaller of them
  int64_t xs, as;          // elements of a plane of X, of A
  uint16_t *x0, *a, *b;
  __device__ __forceinline__ MuonPlanes(const MuonDesc& d, int64_t mat) {
    rp = (d.rows + 63) & ~63;
    cp = (d.cols + 63) & ~63;
    m = d.rows > d.cols ? cp : rp;
    xs = (int64_t)rp * cp;
    as = (int64_t)m * m;
    x0 = d.planes + mat * (4 * xs + 4 * as);
    a = x0 + 4 * xs;
    b = a + 2 * as;
  }
  // X or X' (an array of both would lie in memory, 2.7 us a launch)
  __device__ __forceinline__ uint16_t* x(int which) const { return x0 + which * 2 * xs; }
};

// m = mu m + g, and each chunk's sum of u^2, in 64 bits: a finite u's squares may be past fp32 at either
// end (1e20, or 1e-25 with an eps as small), and as many conversions are nothing beside the bytes; the first work-group leaves the tensors' table. Bound by
// memory, 5.5 TB/s (83 M elements in fp32: 172 us)
template <class T>
__global__ __launch_bounds__(kMuonThreads) void k_muon_momentum(MuonFirstArgs first) {
  const int tid = threadIdx.x;
  const MuonArgs& a = first.a;
  if (blockIdx.x == 0)
    for (int i = tid; i < a.count * (int)(sizeof(MuonDesc) / 4); i += kMuonThreads)
      reinterpret_cast<uint32_t*>(a.t)[i] = reinterpret_cast<const uint32_t*>(first.t)[i];
  const MuonDesc d = muon_take(first.t, a.count, blockIdx.x, [](const MuonDesc& t) { return t.chunk0; });
  const uint32_t c = blockIdx.x - d.chunk0;
  const int64_t n = (int64_t)d.rows * d.cols, mat = c / d.chunks, e0 = (int64_t)(c % d.chunks) * kMuonChunk;
  const T* g = static_cast<const T*>(d.g) + mat * n;
  float* m = d.m ? d.m + mat * n : nullptr;
  double sum = 0.0;
  const int64_t e1 = e0 + kMuonChunk < n ? e0 + kMuonChunk : n;
#pragma unroll 2
  for (int64_t e = e0 + tid * 8; e < e1; e += kMuonThreads * 8) {
    float v[8], q[8];
    muon_load8(g + e, e1 - e, v);
    if (m) {
      muon_load8(m + e, e1 - e, q);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        q[j] = fmaf(a.mu, q[j], v[j]);
        v[j] = muon_u(v[j], q[j], a.mu, a.nesterov);
      }
      muon_store8(m + e, e1 - e, q);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fma((double)v[j], (double)v[j], sum);
  }
  sum = lanes_sum64<64>(sum);
  __shared__ double s[kMuonThreads / 64];
  if ((tid & 63) == 0) s[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) a.sums[blockIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
}

// X = u / (|u| + eps) in its padded planes, zeros past the matrix; a work-group takes 8192 elements.
// Bound by memory, 5.1 TB/s (199 us): u is formed again from g and m, 8 bytes, where a plane of it would be
// 4 written and 4 read
template <class T>
__global__ __launch_bounds__(kMuonThreads) void k_muon_start(MuonArgs a) {
  __shared__ double s_part[kMuonThreads / 64];
  const int tid = threadIdx.x;
  const MuonDesc d = muon_take(a.t, a.count, blockIdx.x, [](const MuonDesc& t) { return t.tile0; });
  const int64_t padded = (int64_t)((d.rows + 63) & ~63) * ((d.cols + 63) & ~63);
  const uint32_t per = (uint32_t)((padded + kMuonChunk - 1) / kMuonChunk), t = blockIdx.x - d.tile0;
  const int64_t mat = t / per;
  const MuonPlanes w(d, mat);
  double sum = 0.0;
  for (uint32_t c = tid; c < d.chunks; c += kMuonThreads) sum += a.sums[d.chunk0 + mat * d.chunks + c];
  sum = lanes_sum64<64>(sum);
  if ((tid & 63) == 0) s_part[tid >> 6] = sum;
  __syncthreads();
  // 1 / (|u| + eps) as 2^-ex and a number in (1, 2], which fp32 holds whatever |u| is
  const double norm = sqrt((s_part[0] + s_part[1]) + (s_part[2] + s_part[3])) + (double)a.eps;
  int ex = 0;
  const float f = norm < INFINITY ? (float)(kMuonOne / frexp(norm, &ex)) : NAN;
  const int64_t n = (int64_t)d.rows * d.cols;
  const T* g = static_cast<const T*>(d.g) + mat * n;
  const float* m = d.m ? d.m + mat * n : nullptr;
  const int cpr = w.cp / 8;
#pragma unroll
  for (int i = 0; i < kMuonChunk / 8 / kMuonThreads; ++i) {
    const int64_t q = (int64_t)(t % per) * (kMuonChunk / 8) + i * kMuonThreads + tid;
    const int64_t r = q / cpr;
    const int c = (int)(q - r * cpr) * 8;
    if (r >= w.rp) break;
    float v[8] = {};
    if (r < d.rows && c < d.cols) {
      muon_load8(g + r * d.cols + c, d.cols - c, v);
      if (m) {
        float u[8];
        muon_load8(m + r * d.cols + c, d.cols - c, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = muon_u(v[j], u[j], a.mu, a.nesterov);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ldexpf(v[j], -ex) * f;
    u32x4 hi, lo;
    split8(v, hi, lo);
    *reinterpret_cast<u32x4*>(w.x0 + q * 8) = hi;
    *reinterpret_cast<u32x4*>(w.x0 + w.xs + q * 8) = lo;
  }
}

// ---- the products --------------------------------------------------------------------
// An operand's tile in LDS is BT of its rows by 32 of the summed axis, in two planes. Where the
// summed axis is the contiguous one a row is 64 bytes, chunk ch of row r at ch ^ (r / 4): any 16
// rows of one chunk lie in 16 different 16-byte banks. Where it is the other one (K-major) the
// tile is 32 rows of BT, read transposed (ds_read_b64_tr_b16: 16 lanes read 4 rows x 16 columns
// and get a column each): the 32-byte units of row k at unit ^ swz(k), so that the four rows and
// two units that 32 lanes touch are eight banks of 32 bytes.
constexpr int kMuonK = 32;

template <int BT>
__device__ __forceinline__ int muon_swz(int k) {
  return BT == 128 ? ((k & 3) << 1) | ((k >> 1) & 1) : ((k >> 1) & 1) << 1;
}
struct MuonOperand {
  const uint16_t* base;    // its tile's first row or column at the summed axis' beginning
  int64_t plane;           // elements from the high part to the low one
  int ld, valid;           // elements of a row in memory; the tile's rows or columns that exist
};
// the 16-byte piece of an operand's K tile 0 that lane `lane` of 1 KB block `blk` brings
template <int BT, bool kMajor>
__device__ __forceinline__ const uint16_t* muon_piece(const MuonOperand& o, int blk, int lane) {
  if constexpr (!kMajor) {
    const int r = cmin_dev(blk * 16 + (lane >> 2), o.valid - 1);
    return o.base + ((int64_t)r * o.ld + ((lane & 3) ^ ((lane >> 4) & 3)) * 8);
  } else {
    constexpr int CPR = BT / 8;                  // pieces of a row
    const int k = blk * (64 / CPR) + lane / CPR, ch = lane % CPR;
    const int lc = (((ch >> 1) ^ muon_swz<BT>(k)) << 1) | (ch & 1);
    return o.base + ((int64_t)k * o.ld + cmin_dev(lc * 8, o.valid - 8));
  }
}

// Fragments of a K tile: f[u][ks][part], 16 of the summed axis (step ks) of the rows 32 u .., eight of
// one row a lane. at(): the addresses that a lane reads from in stage 0 (rows: of step 0 and 1;
// K-major: of block 0 and 1).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int F, bool kMajor>
struct MuonFrags {
  u32x4 f[F][2][2];
  uint32_t a0, a1;
  template <int BT>
  __device__ __forceinline__ void at(uint32_t tile, int u0, int lane) {
    if constexpr (!kMajor) {
      const int r = u0 * 32 + (lane & 31), h = lane >> 5, x = (r >> 2) & 3;
      a0 = tile + r * 64 + ((h ^ x) << 4);
      a1 = tile + r * 64 + (((2 + h) ^ x) << 4);
    } else {
      const int l = lane & 15, g = lane >> 4, k = 8 * (g >> 1) + (l >> 2), z = muon_swz<BT>(k);
      const uint32_t row = tile + k * (BT * 2) + ((l & 3) << 3);
      a0 = row + (((u0 * 2 + (g & 1)) ^ z) << 5);
      a1 = row + (((u0 * 2 + 2 + (g & 1)) ^ z) << 5);
    }
  }
};
__device__ __forceinline__ u32x4 join4(u32x2 a, u32x2 b) {
  u32x4 r;
  r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
  return r;
}

// Both operands' fragments of a stage, in one block of assembly with its wait: the compiler takes
// the loads to LDS that are in flight for aliases of a transposed read and would wait for all of
// them. Rows are read 16 bytes at a time, K-major ones in two transposed halves.
#define TMOE_MR(o, a, off) "ds_read_b128 %[" #o "], %[" #a "] offset:%c[" #off "]\n\t"
#define TMOE_MT(o, a, off) "ds_read_b64_tr_b16 %[" #o "], %[" #a "] offset:%c[" #off "]\n\t"
template <int BM, int BN, int FM, int FN, bool LK, bool RK>
__device__ __forceinline__ void muon_read(MuonFrags<FM, LK>& l, MuonFrags<FN, RK>& r, uint32_t stage) {
  const uint32_t l0 = l.a0 + stage, l1 = l.a1 + stage, r0 = r.a0 + stage, r1 = r.a1 + stage;
  u32x2 lw[FM][2][2][2], rw[FN][2][2][2];
  if constexpr (!LK && !RK && FM == 1 && FN == 1)
    asm volatile(TMOE_MR(l000, lp, L00) TMOE_MR(l001, lp, L01) TMOE_MR(l010, lq, L00) TMOE_MR(l011, lq, L01)
                 TMOE_MR(r000, rp, R00) TMOE_MR(r001, rp, R01) TMOE_MR(r010, rq, R00)
                 TMOE_MR(r011, rq, R01) "s_waitcnt lgkmcnt(0)"
                 : [l000] "=&v"(l.f[0][0][0]), [l001] "=&v"(l.f[0][0][1]), [l010] "=&v"(l.f[0][1][0]),
                 [l011] "=&v"(l.f[0][1][1]),
                   [r000] "=&v"(r.f[0][0][0]), [r001] "=&v"(r.f[0][0][1]), [r010] "=&v"(r.f[0][1][0]),
                 [r011] "=&v"(r.f[0][1][1])
                 : [lp] "v"(l0), [lq] "v"(l1), [rp] "v"(r0), [rq] "v"(r1), [L00] "n"(0 * 2048 + 0 * BM * 64),
                 [L01] "n"(0 * 2048 + 1 * BM * 64),
                   [R00] "n"(0 * 2048 + 0 * BN * 64), [R01] "n"(0 * 2048 + 1 * BN * 64)
                 : "memory");
  else if constexpr (!LK && !RK && FM == 1 && FN == 2)
    asm volatile(TMOE_MR(l000, lp, L00) TMOE_MR(l001, lp, L01) TMOE_MR(l010, lq, L00) TMOE_MR(l011, lq, L01)
                 TMOE_MR(r000, rp, R00) TMOE_MR(r001, rp, R01) TMOE_MR(r010, rq, R00) TMOE_MR(r011, rq, R01)
                 TMOE_MR(r100, rp, R10) TMOE_MR(r101, rp, R11) TMOE_MR(r110, rq, R10)
                 TMOE_MR(r111, rq, R11) "s_waitcnt lgkmcnt(0)"
                 : [l000] "=&v"(l.f[0][0][0]), [l001] "=&v"(l.f[0][0][1]), [l010] "=&v"(l.f[0][1][0]),
                 [l011] "=&v"(l.f[0][1][1]),
                   [r000] "=&v"(r.f[0][0][0]), [r001] "=&v"(r.f[0][0][1]), [r010] "=&v"(r.f[0][1][0]),
                 [r011] "=&v"(r.f[0][1][1]), [r100] "=&v"(r.f[1][0][0]), [r101] "=&v"(r.f[1][0][1]),
                 [r110] "=&v"(r.f[1][1][0]), [r111] "=&v"(r.f[1][1][1])
                 : [lp] "v"(l0), [lq] "v"(l1), [rp] "v"(r0), [rq] "v"(r1), [L00] "n"(0 * 2048 + 0 * BM * 64),
                 [L01] "n"(0 * 2048 + 1 * BM * 64),
                   [R00] "n"(0 * 2048 + 0 * BN * 64), [R01] "n"(0 * 2048 + 1 * BN * 64),
                 [R10] "n"(1 * 2048 + 0 * BN * 64), [R11] "n"(1 * 2048 + 1 * BN * 64)
                 : "memory");
  else if constexpr (!LK && !RK && FM == 2 && FN == 2)
    asm volatile(TMOE_MR(l000, lp, L00) TMOE_MR(l001, lp, L01) TMOE_MR(l010, lq, L00) TMOE_MR(l011, lq, L01)
                 TMOE_MR(l100, lp, L10) TMOE_MR(l101, lp, L11) TMOE_MR(l110, lq, L10) TMOE_MR(l111, lq, L11)
                 TMOE_MR(r000, rp, R00) TMOE_MR(r001, rp, R01) TMOE_MR(r010, rq, R00) TMOE_MR(r011, rq, R01)
                 TMOE_MR(r100, rp, R10) TMOE_MR(r101, rp, R11) TMOE_MR(r110, rq, R10)
                 TMOE_MR(r111, rq, R11) "s_waitcnt lgkmcnt(0)"
                 : [l000] "=&v"(l.f[0][0][0]), [l001] "=&v"(l.f[0][0][1]), [l010] "=&v"(l.f[0][1][0]),
                 [l011] "=&v"(l.f[0][1][1]), [l100] "=&v"(l.f[1][0][0]), [l101] "=&v"(l.f[1][0][1]),
                 [l110] "=&v"(l.f[1][1][0]), [l111] "=&v"(l.f[1][1][1]),
                   [r000] "=&v"(r.f[0][0][0]), [r001] "=&v"(r.f[0][0][1]), [r010] "=&v"(r.f[0][1][0]),
                 [r011] "=&v"(r.f[0][1][1]), [r100] "=&v"(r.f[1][0][0]), [r101] "=&v"(r.f[1][0][1]),
                 [r110] "=&v"(r.f[1][1][0]), [r111] "=&v"(r.f[1][1][1])
                 : [lp] "v"(l0), [lq] "v"(l1), [rp] "v"(r0), [rq] "v"(r1), [L00] "n"(0 * 2048 + 0 * BM * 64),
                 [L01] "n"(0 * 2048 + 1 * BM * 64), [L10] "n"(1 * 2048 + 0 * BM * 64),
                 [L11] "n"(1 * 2048 + 1 * BM * 64),
                   [R00] "n"(0 * 2048 + 0 * BN * 64), [R01] "n"(0 * 2048 + 1 * BN * 64),
                 [R10] "n"(1 * 2048 + 0 * BN * 64), [R11] "n"(1 * 2048 + 1 * BN * 64)
                 : "memory");
  else if constexpr (LK && RK && FM == 1 && FN == 1)
    asm volatile(TMOE_MT(l000x, lp, L00x) TMOE_MT(l000y, lp, L00y) TMOE_MT(l001x, lp, L01x)
                 TMOE_MT(l001y, lp, L01y) TMOE_MT(l010x, lp, L10x) TMOE_MT(l010y, lp, L10y)
                 TMOE_MT(l011x, lp, L11x) TMOE_MT(l011y, lp, L11y)
                 TMOE_MT(r000x, rp, R00x) TMOE_MT(r000y, rp, R00y) TMOE_MT(r001x, rp, R01x)
                 TMOE_MT(r001y, rp, R01y) TMOE_MT(r010x, rp, R10x) TMOE_MT(r010y, rp, R10y)
                 TMOE_MT(r011x, rp, R11x) TMOE_MT(r011y, rp, R11y) "s_waitcnt lgkmcnt(0)"
                 : [l000x] "=&v"(lw[0][0][0][0]), [l000y] "=&v"(lw[0][0][0][1]), [l001x] "=&v"(lw[0][0][1][0]),
                 [l001y] "=&v"(lw[0][0][1][1]), [l010x] "=&v"(lw[0][1][0][0]), [l010y] "=&v"(lw[0][1][0][1]),
                 [l011x] "=&v"(lw[0][1][1][0]), [l011y] "=&v"(lw[0][1][1][1]),
                   [r000x] "=&v"(rw[0][0][0][0]), [r000y] "=&v"(rw[0][0][0][1]), [r001x] "=&v"(rw[0][0][1][0]),
                 [r001y] "=&v"(rw[0][0][1][1]), [r010x] "=&v"(rw[0][1][0][0]), [r010y] "=&v"(rw[0][1][0][1]),
                 [r011x] "=&v"(rw[0][1][1][0]), [r011y] "=&v"(rw[0][1][1][1])
                 : [lp] "v"(l0), [rp] "v"(r0), [L00x] "n"(0 * BM * 64 + 0 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L00y] "n"(0 * BM * 64 + 0 * 16 * BM * 2 + 1 * 4 * BM * 2),
                 [L01x] "n"(1 * BM * 64 + 0 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L01y] "n"(1 * BM * 64 + 0 * 16 * BM * 2 + 1 * 4 * BM * 2),
                 [L10x] "n"(0 * BM * 64 + 1 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L10y] "n"(0 * BM * 64 + 1 * 16 * BM * 2 + 1 * 4 * BM * 2),
                 [L11x] "n"(1 * BM * 64 + 1 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L11y] "n"(1 * BM * 64 + 1 * 16 * BM * 2 + 1 * 4 * BM * 2),
                   [R00x] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R00y] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R01x] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R01y] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R10x] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R10y] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R11x] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R11y] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2)
                 : "memory");
  else if constexpr (LK && RK && FM == 1 && FN == 2)
    asm volatile(TMOE_MT(l000x, lp, L00x) TMOE_MT(l000y, lp, L00y) TMOE_MT(l001x, lp, L01x)
                 TMOE_MT(l001y, lp, L01y) TMOE_MT(l010x, lp, L10x) TMOE_MT(l010y, lp, L10y)
                 TMOE_MT(l011x, lp, L11x) TMOE_MT(l011y, lp, L11y)
                 TMOE_MT(r000x, rp, R00x) TMOE_MT(r000y, rp, R00y) TMOE_MT(r001x, rp, R01x)
                 TMOE_MT(r001y, rp, R01y) TMOE_MT(r010x, rp, R10x) TMOE_MT(r010y, rp, R10y)
                 TMOE_MT(r011x, rp, R11x) TMOE_MT(r011y, rp, R11y) TMOE_MT(r100x, rq, R00x)
                 TMOE_MT(r100y, rq, R00y) TMOE_MT(r101x, rq, R01x) TMOE_MT(r101y, rq, R01y)
                 TMOE_MT(r110x, rq, R10x) TMOE_MT(r110y, rq, R10y) TMOE_MT(r111x, rq, R11x)
                 TMOE_MT(r111y, rq, R11y) "s_waitcnt lgkmcnt(0)"
                 : [l000x] "=&v"(lw[0][0][0][0]), [l000y] "=&v"(lw[0][0][0][1]), [l001x] "=&v"(lw[0][0][1][0]),
                 [l001y] "=&v"(lw[0][0][1][1]), [l010x] "=&v"(lw[0][1][0][0]), [l010y] "=&v"(lw[0][1][0][1]),
                 [l011x] "=&v"(lw[0][1][1][0]), [l011y] "=&v"(lw[0][1][1][1]),
                   [r000x] "=&v"(rw[0][0][0][0]), [r000y] "=&v"(rw[0][0][0][1]), [r001x] "=&v"(rw[0][0][1][0]),
                 [r001y] "=&v"(rw[0][0][1][1]), [r010x] "=&v"(rw[0][1][0][0]), [r010y] "=&v"(rw[0][1][0][1]),
                 [r011x] "=&v"(rw[0][1][1][0]), [r011y] "=&v"(rw[0][1][1][1]), [r100x] "=&v"(rw[1][0][0][0]),
                 [r100y] "=&v"(rw[1][0][0][1]), [r101x] "=&v"(rw[1][0][1][0]), [r101y] "=&v"(rw[1][0][1][1]),
                 [r110x] "=&v"(rw[1][1][0][0]), [r110y] "=&v"(rw[1][1][0][1]), [r111x] "=&v"(rw[1][1][1][0]),
                 [r111y] "=&v"(rw[1][1][1][1])
                 : [lp] "v"(l0), [rp] "v"(r0), [rq] "v"(r1),
                 [L00x] "n"(0 * BM * 64 + 0 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L00y] "n"(0 * BM * 64 + 0 * 16 * BM * 2 + 1 * 4 * BM * 2),
                 [L01x] "n"(1 * BM * 64 + 0 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L01y] "n"(1 * BM * 64 + 0 * 16 * BM * 2 + 1 * 4 * BM * 2),
                 [L10x] "n"(0 * BM * 64 + 1 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L10y] "n"(0 * BM * 64 + 1 * 16 * BM * 2 + 1 * 4 * BM * 2),
                 [L11x] "n"(1 * BM * 64 + 1 * 16 * BM * 2 + 0 * 4 * BM * 2),
                 [L11y] "n"(1 * BM * 64 + 1 * 16 * BM * 2 + 1 * 4 * BM * 2),
                   [R00x] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R00y] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R01x] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R01y] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R10x] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R10y] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R11x] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R11y] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2)
                 : "memory");
  else if constexpr (!LK && RK && FM == 1 && FN == 1)
    asm volatile(TMOE_MR(l000, lp, L00) TMOE_MR(l001, lp, L01) TMOE_MR(l010, lq, L00) TMOE_MR(l011, lq, L01)
                 TMOE_MT(r000x, rp, R00x) TMOE_MT(r000y, rp, R00y) TMOE_MT(r001x, rp, R01x)
                 TMOE_MT(r001y, rp, R01y) TMOE_MT(r010x, rp, R10x) TMOE_MT(r010y, rp, R10y)
                 TMOE_MT(r011x, rp, R11x) TMOE_MT(r011y, rp, R11y) "s_waitcnt lgkmcnt(0)"
                 : [l000] "=&v"(l.f[0][0][0]), [l001] "=&v"(l.f[0][0][1]), [l010] "=&v"(l.f[0][1][0]),
                 [l011] "=&v"(l.f[0][1][1]),
                   [r000x] "=&v"(rw[0][0][0][0]), [r000y] "=&v"(rw[0][0][0][1]), [r001x] "=&v"(rw[0][0][1][0]),
                 [r001y] "=&v"(rw[0][0][1][1]), [r010x] "=&v"(rw[0][1][0][0]), [r010y] "=&v"(rw[0][1][0][1]),
                 [r011x] "=&v"(rw[0][1][1][0]), [r011y] "=&v"(rw[0][1][1][1])
                 : [lp] "v"(l0), [lq] "v"(l1), [rp] "v"(r0), [L00] "n"(0 * 2048 + 0 * BM * 64),
                 [L01] "n"(0 * 2048 + 1 * BM * 64),
                   [R00x] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R00y] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R01x] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R01y] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R10x] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R10y] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R11x] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R11y] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2)
                 : "memory");
  else if constexpr (!LK && RK && FM == 2 && FN == 2)
    asm volatile(TMOE_MR(l000, lp, L00) TMOE_MR(l001, lp, L01) TMOE_MR(l010, lq, L00) TMOE_MR(l011, lq, L01)
                 TMOE_MR(l100, lp, L10) TMOE_MR(l101, lp, L11) TMOE_MR(l110, lq, L10) TMOE_MR(l111, lq, L11)
                 TMOE_MT(r000x, rp, R00x) TMOE_MT(r000y, rp, R00y) TMOE_MT(r001x, rp, R01x)
                 TMOE_MT(r001y, rp, R01y) TMOE_MT(r010x, rp, R10x) TMOE_MT(r010y, rp, R10y)
                 TMOE_MT(r011x, rp, R11x) TMOE_MT(r011y, rp, R11y) TMOE_MT(r100x, rq, R00x)
                 TMOE_MT(r100y, rq, R00y) TMOE_MT(r101x, rq, R01x) TMOE_MT(r101y, rq, R01y)
                 TMOE_MT(r110x, rq, R10x) TMOE_MT(r110y, rq, R10y) TMOE_MT(r111x, rq, R11x)
                 TMOE_MT(r111y, rq, R11y) "s_waitcnt lgkmcnt(0)"
                 : [l000] "=&v"(l.f[0][0][0]), [l001] "=&v"(l.f[0][0][1]), [l010] "=&v"(l.f[0][1][0]),
                 [l011] "=&v"(l.f[0][1][1]), [l100] "=&v"(l.f[1][0][0]), [l101] "=&v"(l.f[1][0][1]),
                 [l110] "=&v"(l.f[1][1][0]), [l111] "=&v"(l.f[1][1][1]),
                   [r000x] "=&v"(rw[0][0][0][0]), [r000y] "=&v"(rw[0][0][0][1]), [r001x] "=&v"(rw[0][0][1][0]),
                 [r001y] "=&v"(rw[0][0][1][1]), [r010x] "=&v"(rw[0][1][0][0]), [r010y] "=&v"(rw[0][1][0][1]),
                 [r011x] "=&v"(rw[0][1][1][0]), [r011y] "=&v"(rw[0][1][1][1]), [r100x] "=&v"(rw[1][0][0][0]),
                 [r100y] "=&v"(rw[1][0][0][1]), [r101x] "=&v"(rw[1][0][1][0]), [r101y] "=&v"(rw[1][0][1][1]),
                 [r110x] "=&v"(rw[1][1][0][0]), [r110y] "=&v"(rw[1][1][0][1]), [r111x] "=&v"(rw[1][1][1][0]),
                 [r111y] "=&v"(rw[1][1][1][1])
                 : [lp] "v"(l0), [lq] "v"(l1), [rp] "v"(r0), [rq] "v"(r1), [L00] "n"(0 * 2048 + 0 * BM * 64),
                 [L01] "n"(0 * 2048 + 1 * BM * 64), [L10] "n"(1 * 2048 + 0 * BM * 64),
                 [L11] "n"(1 * 2048 + 1 * BM * 64),
                   [R00x] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R00y] "n"(0 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R01x] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R01y] "n"(1 * BN * 64 + 0 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R10x] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R10y] "n"(0 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2),
                 [R11x] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 0 * 4 * BN * 2),
                 [R11y] "n"(1 * BN * 64 + 1 * 16 * BN * 2 + 1 * 4 * BN * 2)
                 : "memory");
  else
    static_assert(FM == 0, "no such tile");
  if constexpr (LK)
#pragma unroll
    for (int i = 0; i < 4 * FM; ++i) l.f[i / 4][i / 2 & 1][i & 1] = join4(lw[i / 4][i / 2 & 1][i & 1][0], lw[i / 4][i / 2 & 1][i & 1][1]);
  if constexpr (RK)
#pragma unroll
    for (int i = 0; i < 4 * FN; ++i) r.f[i / 4][i / 2 & 1][i & 1] = join4(rw[i / 4][i / 2 & 1][i & 1][0], rw[i / 4][i / 2 & 1][i & 1][1]);
}
#undef TMOE_MR
#undef TMOE_MT

// BM x BN tiles, WM x WN waves, NS LDS stages of both operands' planes
template <int BM_, int BN_, int WM_, int WN_, int NS_>
struct MuonTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_, W = WM * WN, kThreads = 64 * W;
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
  static constexpr int kStage = 2 * (BM + BN) * 64, kRow = 32 * FN + 4;   // floats of a row of a wave's result
  static constexpr int kStore = W * 32 * kRow * 4;
  static constexpr int kSmem = NS * kStage > kStore ? NS * kStage : kStore;
  static constexpr int LB = 2 * BM * 64 / 1024 / W, RB = 2 * BN * 64 / 1024 / W;   // blocks that a wave brings
  static_assert(FM <= 2 && FN <= 2 && kSmem <= 160 * 1024 && LB >= 1 && RB >= 1, "");
  static_assert(BM * 64 / 1024 % LB == 0 && BN * 64 / 1024 % RB == 0, "a wave's blocks are of one part");
};

// acc (transposed blocks: a lane's row of lhs, columns of rhs in its elements) of nkt tiles of the
// summed axis. Tile kt + NS - 1 is on its way while tile kt is computed; past the last one the last
// is fetched again, into a stage that nothing reads, so that every wait counts alike.
//
// Eight waves work in two groups, one of each on every SIMD, the second a barrier behind the first:
// while one reads its fragments the other has its matrix instructions, and its loads between those
// (ahead of the reads they kept them waiting for the vector memory queue: 2760 instead of 1980
// cycles a K tile of 256 x 128). With phases between barriers, group 0 reads tile kt in phase 2 kt
// and computes in 2 kt + 1, group 1 in 2 kt + 1 and 2 kt + 2. Tile kt's stage is read last in phase
// 2 kt + 1: in its computing phase of tile kt group 0 loads tile kt + NS - 1, into the stage of tile
// kt - 1, and group 1 tile kt + NS, into that of tile kt. Before phase 2 kt both have waited for
// their loads of tile kt, in phase 2 kt - 1: group 0 at the end of its computing of tile kt - 1, when
// tiles up to kt + NS - 2 are on their way, group 1 of its reading of tile kt - 1, likewise.
//
// kSame: rhs is lhs (a tile on the diagonal of a symmetric product), loaded once: 66 layers' step
// 14.78 -> 14.33 ms, two of three tiles of a 256 x 256 product being such.
template <class TL, bool LK, bool RK, bool kSame = false>
__device__ __forceinline__ void muon_product(f32x16 (&acc)[TL::FM][TL::FN], const MuonOperand& l,
                                             const MuonOperand& r, int nkt, char* smem) {
  constexpr int NS = TL::NS, D = TL::LB + (kSame ? 0 : TL::RB);
  constexpr bool kTwo = TL::W == 8;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / TL::WN, wn = wave % TL::WN;
  const uint32_t base = (uint32_t)(size_t)(lds_vptr)smem;
  MuonFrags<TL::FM, LK> af;
  MuonFrags<TL::FN, RK> bf;
  af.template at<TL::BM>(base, wm * TL::FM, lane);
  bf.template at<TL::BN>(base + (kSame ? 0 : 2 * TL::BM * 64), wn * TL::FN, lane);
  // this wave's blocks: LB neighbours of one part of lhs, RB of rhs
  constexpr int kLhs = TL::BM * 64 / 1024, kRhs = TL::BN * 64 / 1024;
  const int lq = wave * TL::LB, rq = wave * TL::RB;
  // where their pieces lie in K tile 0, and the step to the next one
  const uint16_t* lp[TL::LB];
  const uint16_t* rp[TL::RB];
#pragma unroll
  for (int i = 0; i < TL::LB; ++i)
    lp[i] = muon_piece<TL::BM, LK>(l, lq % kLhs + i, lane) + (lq >= kLhs ? l.plane : 0);
#pragma unroll
  for (int i = 0; i < TL::RB; ++i)
    rp[i] = muon_piece<TL::BN, RK>(r, rq % kRhs + i, lane) + (rq >= kRhs ? r.plane : 0);
  const int64_t lstep = LK ? (int64_t)kMuonK * l.ld : kMuonK, rstep = RK ? (int64_t)kMuonK * r.ld : kMuonK;
  // piece i of K tile kt into a stage
  auto piece = [&](int i, int kt, int st) __attribute__((always_inline)) {
    char* s = smem + st * TL::kStage;
    if (i < TL::LB)
      __builtin_amdgcn_global_load_lds((gbl_cvptr)(lp[i] + kt * lstep), (lds_vptr)(s + (lq + i) * 1024), 16, 0, 0);
    else
      __builtin_amdgcn_global_load_lds((gbl_cvptr)(rp[i - TL::LB] + kt * rstep),
                                       (lds_vptr)(s + 2 * TL::BM * 64 + (rq + i - TL::LB) * 1024), 16, 0, 0);
  };
  // the products of the fragments, K tile kt's pieces loaded in between
  auto compute = [&](int kt, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 6; ++q) {                // steps 0 and 1: low high, high low, high high
#pragma unroll
      for (int i = 0; i < TL::FM; ++i)
#pragma unroll
        for (int j = 0; j < TL::FN; ++j)
          acc[i][j] = mma_f16(bf.f[j][q / 3][q % 3 == 0], af.f[i][q / 3][q % 3 == 1], acc[i][j]);
      if (q < 5) {
#pragma unroll
        for (int i = q * D / 5; i < (q + 1) * D / 5; ++i) piece(i, kt, st);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int group = kTwo ? wave >> 2 : 0;
#pragma unroll
  for (int t = 0; t < NS; ++t)
    if (t < NS - 1 || group)
#pragma unroll
      for (int i = 0; i < D; ++i) piece(i, cmin_dev(t, nkt - 1), t);
  int st = 0;                                    // the stage of tile kt
  auto next = [](int s) { return s + 1 < NS ? s + 1 : 0; };
  if (group) wait_vm_lds<(NS - 1) * D>();
  else wait_vm_lds<(NS - 2) * D>();
  if constexpr (kTwo) {
    lds_barrier();
    if (group) lds_barrier();
    int to = group ? 0 : NS - 1;
    for (int kt = 0; kt < nkt; ++kt) {
      muon_read<TL::BM, TL::BN>(af, bf, st * TL::kStage);
      if (group) wait_vm_lds<(NS - 2) * D>();
      lds_barrier();
      compute(cmin_dev(kt + NS - 1 + group, nkt - 1), to);
      if (!group) wait_vm_lds<(NS - 2) * D>();
      lds_barrier();
      st = next(st);
      to = next(to);
    }
    if (!group) lds_barrier();
  } else {
    int to = NS - 1;
    for (int kt = 0; kt < nkt; ++kt) {
      lds_barrier();
      muon_read<TL::BM, TL::BN>(af, bf, st * TL::kStage);
      compute(cmin_dev(kt + NS - 1, nkt - 1), to);
      wait_vm_lds<(NS - 2) * D>();
      st = next(st);
      to = next(to);
    }
  }
  mfma_drain();
  wait_vm_lds<0>();
  lds_barrier();
}

// tile number q of those on and below the diagonal, row by row
__device__ __forceinline__ void muon_pair(int q, int& tm, int& tn) {
  tm = (int)((sqrtf(8.f * q + 1.f) - 1.f) * 0.5f);
  while ((tm + 1) * (tm + 2) / 2 <= q) ++tm;
  while (tm * (tm + 1) / 2 > q) --tm;
  tn = q - tm * (tm + 1) / 2;
}
// Where a slice of the Gram product's summed axis leaves its sums of a tile, as the lanes hold
// them: in X', which is not in use then.
template <int BT>
__device__ __forceinline__ float* muon_part(uint16_t* next, int slice, int slices, int tile) {
  return reinterpret_cast<float*>(next) + ((int64_t)tile * slices + slice) * BT * BT;
}

constexpr int kMuonGram = 0, kMuonPoly = 1, kMuonApply = 2, kMuonLast = 3;

// One product for all matrices:
//   Gram   A = X X^T (wide), X^T X (tall)        Apply  X' = B X (wide), X B (tall)
//   Poly   B = a + b A + c A A                   Last   p = keep p - rate B X
// A launch for 83 M elements (435 matrices of 256 x 512 and larger ones): Gram 145 us, Poly 85, Apply 246,
// Last 329 in fp32. Gram and Poly are bound by LDS reads and starts of tiles of eight or sixteen K tiles (the
// matrix units at work 45% and 26% of the time), Apply by those (42%) and 700 MB of X and X'.
template <class TL, int PHASE, class T>
__global__ __launch_bounds__(TL::kThreads) void k_muon_gemm(MuonArgs a) {
  constexpr int BM = TL::BM, BN = TL::BN, FM = TL::FM, FN = TL::FN, kRow = TL::kRow;
  constexpr bool kSymmetric = PHASE == kMuonGram || PHASE == kMuonPoly;
  static_assert(!kSymmetric || BM == BN, "tiles below the diagonal");
  __shared__ u32x4 s_mem[TL::kSmem / 16];
  char* smem = reinterpret_cast<char*>(s_mem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / TL::WN, wn = wave % TL::WN;
  auto first = [](const MuonDesc& t) {
    return PHASE == kMuonGram ? t.gram0 : PHASE == kMuonPoly ? t.sym0 : t.app0;
  };
  // work-groups go round the eight XCDs: each gets a run of neighbours, which share X in its L2
  const uint32_t each = gridDim.x / 8, place = blockIdx.x < each * 8 ? blockIdx.x % 8 * each + blockIdx.x / 8 : blockIdx.x;
  const MuonDesc d = muon_take(a.t, a.count, place, first);
  const bool tall = d.rows > d.cols;
  uint32_t t = place - first(d);
  int64_t mat;
  int tm, tn, slice = 0;
  {
    const int rp = (d.rows + 63) & ~63, cp = (d.cols + 63) & ~63;
    if constexpr (kSymmetric) {                  // tiles on and below the diagonal
      const int side = ((tall ? cp : rp) + BM - 1) / BM, per = side * (side + 1) / 2;
      if constexpr (PHASE == kMuonGram) {
        slice = t % d.slices;
        t /= d.slices;
      }
      mat = t / per;
      muon_pair(t % per, tm, tn);
    } else {                                     // tiles that share X are neighbours
      const int tr = (rp + BM - 1) / BM, tc = (cp + BN - 1) / BN, per = tr * tc;
      mat = t / per;
      const int q = t % per;
      tm = tall ? q / tc : q % tr;
      tn = tall ? q % tc : q / tr;
    }
  }
  const MuonPlanes w(d, mat);
  const uint16_t* x = w.x(a.cur);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = zero16();
  const int mv = (int)((kSymmetric ? w.m : w.rp) - m0), nv = (int)((kSymmetric ? w.m : w.cp) - n0);
  const int lv = cmin_dev(mv, BM), rv = cmin_dev(nv, BN);
  if constexpr (PHASE == kMuonGram) {
    const int all = (tall ? w.rp : w.cp) / kMuonK, k0 = slice * d.slice_tiles;
    const int nkt = cmin_dev(d.slice_tiles, all - k0);
    const uint16_t* xk = x + (tall ? (int64_t)k0 * kMuonK * w.cp : k0 * kMuonK);
    const int64_t step = tall ? 1 : w.cp;        // from a row of A to the next one's
    const MuonOperand l{xk + m0 * step, w.xs, w.cp, lv}, r{xk + n0 * step, w.xs, w.cp, rv};
    if (tall) {
      if (tm == tn) muon_product<TL, true, true, true>(acc, l, r, nkt, smem);
      else muon_product<TL, true, true>(acc, l, r, nkt, smem);
    } else {
      if (tm == tn) muon_product<TL, false, false, true>(acc, l, r, nkt, smem);
      else muon_product<TL, false, false>(acc, l, r, nkt, smem);
    }
    if (d.slices > 1) {                          // k_muon_sum adds them
      float* part = muon_part<BM>(w.x(a.cur ^ 1), slice, d.slices, tm * (tm + 1) / 2 + tn);
      const float f = 1.f / kMuonOne;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(part + ((((wave * FM + i) * FN + j) * 4 + q) * 64 + lane) * 4) =
                float4{acc[i][j][4 * q] * f, acc[i][j][4 * q + 1] * f, acc[i][j][4 * q + 2] * f, acc[i][j][4 * q + 3] * f};
      return;
    }
  } else if constexpr (PHASE == kMuonPoly) {
    const MuonOperand l{w.a + m0 * w.m, w.as, w.m, lv}, r{w.a + n0 * w.m, w.as, w.m, rv};
    if (tm == tn) muon_product<TL, false, false, true>(acc, l, r, w.m / kMuonK, smem);
    else muon_product<TL, false, false>(acc, l, r, w.m / kMuonK, smem);
  } else {
    if (tall)
      muon_product<TL, false, false>(acc, {x + m0 * w.cp, w.xs, w.cp, lv}, {w.b + n0 * w.m, w.as, w.m, rv},
                                     w.m / kMuonK, smem);
    else
      muon_product<TL, false, true>(acc, {w.b + m0 * w.m, w.as, w.m, lv}, {x + n0, w.xs, w.cp, rv},
                                    w.m / kMuonK, smem);
  }
  // a wave's blocks of 32 rows through its own LDS: a lane has row l & 31, elements 4 q .. of
  // columns 8 q + 4 (l >> 5)
  float* res = reinterpret_cast<float*>(smem) + wave * 32 * kRow;
  const float f = (PHASE == kMuonPoly ? a.c : 1.f) / kMuonOne;
  const int64_t c0 = n0 + wn * 32 * FN;
  const int ld = kSymmetric ? w.m : w.cp;        // of what is written
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t r0 = m0 + wm * 32 * FM + i * 32;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(res + (lane & 31) * kRow + j * 32 + 8 * q + 4 * (lane >> 5)) =
            float4{acc[i][j][4 * q] * f, acc[i][j][4 * q + 1] * f, acc[i][j][4 * q + 2] * f, acc[i][j][4 * q + 3] * f};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < 2 * FN; ++it) {
      const int k = it * 64 + lane, r = k / (4 * FN), c = k % (4 * FN) * 8;
      const int64_t row = r0 + r, col = c0 + c;
      if (row - m0 >= mv || col - n0 >= nv) continue;
      float v[8], u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = res[r * kRow + c + j];
      if constexpr (PHASE == kMuonPoly) {
        const uint16_t* q = w.a + row * ld + col;
        join8f(*reinterpret_cast<const u32x4*>(q), *reinterpret_cast<const u32x4*>(q + w.as), u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = fmaf(a.b, u[j], v[j]) + (row == col + j ? a.a * kMuonOne : 0.f);
          res[r * kRow + c + j] = v[j];
        }
      }
      if constexpr (PHASE != kMuonLast) {
        u32x4 hi, lo;
        split8(v, hi, lo);
        uint16_t* o = (PHASE == kMuonGram ? w.a : PHASE == kMuonPoly ? w.b : w.x(a.cur ^ 1)) + row * ld + col;
        *reinterpret_cast<u32x4*>(o) = hi;
        *reinterpret_cast<u32x4*>(o + (kSymmetric ? w.as : w.xs)) = lo;
      } else if (row < d.rows && col < d.cols) {
        T* p = static_cast<T*>(d.p) + (mat * d.rows + row) * d.cols + col;
        const float rate = d.rate / kMuonOne;
        if (!a.write_only) {
          muon_load8(p, d.cols - col, u);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = fmaf(a.keep, u[j], -rate * v[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= -rate;
        }
        muon_store8(p, d.cols - col, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (kSymmetric && tm != tn) {                // the other half: four lanes take a column, a row of it
      const int r = lane % 4 * 8;
#pragma unroll
      for (int it = 0; it < 2 * FN; ++it) {
        const int c = it * 16 + lane / 4;
        if (c0 + c - n0 >= nv || r0 + r - m0 >= mv) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = res[(r + j) * kRow + c];
        u32x4 hi, lo;
        split8(v, hi, lo);
        uint16_t* o = (PHASE == kMuonGram ? w.a : w.b) + (c0 + c) * ld + r0 + r;
        *reinterpret_cast<u32x4*>(o) = hi;
        *reinterpret_cast<u32x4*>(o + w.as) = lo;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// A of the slices' sums, in their order: a wave takes 32 rows and columns of a tile; a launch's 4 to 6 us
template <class TL>
__global__ __launch_bounds__(64) void k_muon_sum(MuonArgs a) {
  constexpr int BT = TL::BM, kBlocks = TL::W * TL::FM * TL::FN;      // of 32 x 32 in a tile
  __shared__ float s_res[32][33];
  const int lane = threadIdx.x;
  const MuonDesc d = muon_take(a.t, a.count, blockIdx.x, [](const MuonDesc& t) { return t.sum0; });
  uint32_t t = blockIdx.x - d.sum0;
  const int blk = t % kBlocks;
  t /= kBlocks;
  const int m = ((d.rows > d.cols ? d.cols : d.rows) + 63) & ~63, side = (m + BT - 1) / BT;
  const int per = side * (side + 1) / 2, tile = t % per;
  const MuonPlanes w(d, t / per);
  int tm, tn;
  muon_pair(tile, tm, tn);
  // block (i, j) of wave (wm, wn), as k_muon_gemm's accumulators lie
  const int wave = blk / (TL::FM * TL::FN), i = blk / TL::FN % TL::FM, j = blk % TL::FN;
  const int64_t r0 = (int64_t)tm * BT + (wave / TL::WN * TL::FM + i) * 32;
  const int64_t c0 = (int64_t)tn * BT + (wave % TL::WN * TL::FN + j) * 32;
  if (r0 >= m || c0 >= m) return;
  float v[16] = {};
  for (int s = 0; s < d.slices; ++s) {
    const float* p = muon_part<BT>(w.x(a.cur ^ 1), s, d.slices, tile) + blk * 1024 + lane * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 u = *reinterpret_cast<const float4*>(p + q * 256);
      v[4 * q] += u.x; v[4 * q + 1] += u.y; v[4 * q + 2] += u.z; v[4 * q + 3] += u.w;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) s_res[lane & 31][8 * q + 4 * (lane >> 5) + e] = v[4 * q + e];
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int k = it * 64 + lane, r = k / 4, c = k % 4 * 8;
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s_res[r][c + e];
      y[e] = s_res[c + e][r];
    }
    u32x4 hi, lo;
    split8(x, hi, lo);
    uint16_t* o = w.a + (r0 + r) * m + c0 + c;
    *reinterpret_cast<u32x4*>(o) = hi;
    *reinterpret_cast<u32x4*>(o + w.as) = lo;
    if (tm == tn) continue;
    split8(y, hi, lo);
    o = w.a + (c0 + r) * m + r0 + c;
    *reinterpret_cast<u32x4*>(o) = hi;
    *reinterpret_cast<u32x4*>(o + w.as) = lo;
  }
}

}  // namespace dev
}  // namespace tmoe
