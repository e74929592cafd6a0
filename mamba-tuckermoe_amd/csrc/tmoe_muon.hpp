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
// Bound by the matrix units: three times the products' work, of which A and B, symmetric, are
// computed by half and stored twice.
//
// A launch takes all matrices of all tensors: a work-group finds its tile's tensor in a table
// that the first kernels leave in the workspace. X is held both ways round, so that both
// operands of each product lie along its summed axis.
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
    h[j] = (_Float16)v[j];
    l[j] = (_Float16)(v[j] - (float)h[j]);
  }
  hi = __builtin_bit_cast(u32x4, h);
  lo = __builtin_bit_cast(u32x4, l);
}
__device__ __forceinline__ void join8f(u32x4 hi, u32x4 lo, float (&v)[8]) {
  const f16x8 h = __builtin_bit_cast(f16x8, hi), l = __builtin_bit_cast(f16x8, lo);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)h[j] + (float)l[j];
}

// The last tensor whose first tile (of the kind that `first` gives) is no later than `tile`: 64
// entries at a time, by ballots. A whole wave's call.
template <class F>
__device__ __forceinline__ int muon_find(int count, uint32_t tile, F first) {
  int lo = 0, n = count;
  const int lane = threadIdx.x & 63;
  while (n > 1) {
    const int step = (n + 63) / 64, at = lo + lane * step;
    const bool before = lane * step < n && first(at) <= tile;
    const int k = 63 - __clzll(__ballot(before));     // (lane 0's always is)
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

__device__ __forceinline__ float muon_u(float g, float m, float mu, bool nesterov) {
  return nesterov ? fmaf(mu, m, g) : m;
}

// m = mu m + g, and each chunk's sum of u^2; the first work-group writes the tensors' entries of
// the table
template <class T>
__global__ __launch_bounds__(kMuonThreads) void k_muon_momentum(MuonChunkArgs a) {
  const int tid = threadIdx.x;
  if (blockIdx.x == 0) {
    for (int i = tid; i < a.count * (int)(sizeof(MuonDesc) / 4); i += kMuonThreads)
      reinterpret_cast<uint32_t*>(a.table + a.first)[i] = reinterpret_cast<const uint32_t*>(a.t)[i];
  }
  const int i = muon_find(a.count, blockIdx.x, [&](int k) { return a.t[k].chunk0 - a.t[0].chunk0; });
  const MuonDesc& d = a.t[i];
  const uint32_t c = blockIdx.x - (d.chunk0 - a.t[0].chunk0);
  const int64_t n = (int64_t)d.rows * d.cols, mat = c / d.chunks, e0 = (int64_t)(c % d.chunks) * kMuonChunk;
  const T* g = static_cast<const T*>(d.g) + mat * n;
  float* m = d.m ? d.m + mat * n : nullptr;
  float sum = 0.f;
  const int64_t e1 = e0 + kMuonChunk < n ? e0 + kMuonChunk : n;
  for (int64_t e = e0 + tid * 4; e < e1; e += kMuonThreads * 4) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint16_t h4 __attribute__((ext_vector_type(4), aligned(2)));
    if (e + 4 <= e1) {
      float gv[4];
      if constexpr (sizeof(T) == 2) {
        const h4 q = *reinterpret_cast<const h4*>(g + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) gv[j] = bf16_bits_to_f32(q[j]);
      } else {
        const f4 q = *reinterpret_cast<const f4*>(g + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) gv[j] = q[j];
      }
      if (m) {
        f4 q = *reinterpret_cast<const f4*>(m + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[j] = fmaf(a.mu, q[j], gv[j]);
          gv[j] = muon_u(gv[j], q[j], a.mu, a.nesterov);
        }
        *reinterpret_cast<f4*>(m + e) = q;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fmaf(gv[j], gv[j], sum);
    } else {
      for (int64_t k = e; k < e1; ++k) {
        float v = load_as_f32(g + k);
        if (m) {
          const float q = fmaf(a.mu, m[k], v);
          m[k] = q;
          v = muon_u(v, q, a.mu, a.nesterov);
        }
        sum = fmaf(v, v, sum);
      }
    }
  }
  sum = lanes_sum<64>(sum);
  __shared__ float s[kMuonThreads / 64];
  if ((tid & 63) == 0) s[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) a.sums[d.chunk0 + c] = (s[0] + s[1]) + (s[2] + s[3]);
}

// X and its transpose of u, by 64 x 64 tiles of the padded X; zeros past the matrix
template <class T>
__global__ __launch_bounds__(kMuonThreads) void k_muon_start(MuonArgs a) {
  __shared__ float s_x[64][65];
  __shared__ float s_part[kMuonThreads / 64];
  const int tid = threadIdx.x;
  const int i = muon_find(a.count, blockIdx.x, [&](int k) { return a.table[k].tile0; });
  const MuonDesc d = a.table[i];
  const uint32_t t = blockIdx.x - d.tile0;
  const int tn = d.np / 64, per = tn * (d.mp / 64);
  const int64_t mat = t / per;
  const int q = t % per, i0 = q / tn * 64, j0 = q % tn * 64;     // of X
  float sum = 0.f;
  for (uint32_t c = tid; c < d.chunks; c += kMuonThreads) sum += a.sums[d.chunk0 + mat * d.chunks + c];
  sum = lanes_sum<64>(sum);
  if ((tid & 63) == 0) s_part[tid >> 6] = sum;
  __syncthreads();
  const float f = kMuonOne / (sqrtf((s_part[0] + s_part[1]) + (s_part[2] + s_part[3])) + a.eps);
  const int64_t n = (int64_t)d.rows * d.cols;
  const T* g = static_cast<const T*>(d.g) + mat * n;
  const float* m = d.m ? d.m + mat * n : nullptr;
  const bool tall = d.rows > d.cols;
  // rows of the matrix as it lies: of X, or of its transpose
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
  for (int k = tid; k < 64 * 64; k += kMuonThreads) {
    const int r = k >> 6, c = k & 63;
    float v = 0.f;
    if (r0 + r < d.rows && c0 + c < d.cols) {
      const int64_t e = (int64_t)(r0 + r) * d.cols + c0 + c;
      v = load_as_f32(g + e);
      if (m) v = muon_u(v, m[e], a.mu, a.nesterov);
    }
    if (tall) s_x[c][r] = v * f;
    else s_x[r][c] = v * f;
  }
  __syncthreads();
  const int64_t plane = (int64_t)d.mp * d.np;
  uint16_t* x = d.x[0] + mat * 2 * plane;
  uint16_t* xt = d.xt[0] + mat * 2 * plane;
  for (int k = tid; k < 64 * 8; k += kMuonThreads) {
    const int r = k >> 3, c = (k & 7) * 8;
    float v[8], w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = s_x[r][c + j];
      w[j] = s_x[c + j][r];
    }
    u32x4 hi, lo;
    split8(v, hi, lo);
    uint16_t* p = x + (int64_t)(i0 + r) * d.np + j0 + c;
    *reinterpret_cast<u32x4*>(p) = hi;
    *reinterpret_cast<u32x4*>(p + plane) = lo;
    split8(w, hi, lo);
    p = xt + (int64_t)(j0 + r) * d.mp + i0 + c;
    *reinterpret_cast<u32x4*>(p) = hi;
    *reinterpret_cast<u32x4*>(p + plane) = lo;
  }
}

constexpr int kMuonGram = 0, kMuonPoly = 1, kMuonApply = 2, kMuonLast = 3;

// One product for all matrices, in tiles of BT x BT, four waves, two LDS stages of both operands'
// high and low parts:
//   Gram   A = X X^T            Apply  X' = a X + B X
//   Poly   B = b A + c A A      Last   p = keep p - rate (a X + B X)
template <int BT, int PHASE, class T>
__global__ __launch_bounds__(kMuonThreads) void k_muon_gemm(MuonArgs a) {
  constexpr int F = BT / 64;                     // blocks of 32 of a wave, each way
  constexpr int kStage = 4 * BT * 128;           // bytes: a high, a low, b high, b low
  constexpr int kRow = BT + 4;                   // floats of a row of the result in LDS
  constexpr int kBytes = 2 * kStage > BT * kRow * 4 ? 2 * kStage : BT * kRow * 4;
  constexpr bool kSymmetric = PHASE == kMuonGram || PHASE == kMuonPoly;
  __shared__ u32x4 s_mem[kBytes / 16];
  char* smem = reinterpret_cast<char*>(s_mem);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
  const int which = muon_find(a.count, blockIdx.x, [&](int k) { return kSymmetric ? a.table[k].sym0 : a.table[k].app0; });
  const MuonDesc& d = a.table[which];
  const int mp = d.mp, np = d.np;
  uint32_t t = blockIdx.x - (kSymmetric ? d.sym0 : d.app0);
  const int tm_n = (mp + BT - 1) / BT, tn_n = (np + BT - 1) / BT;
  int64_t mat;
  int tm, tn;
  if constexpr (kSymmetric) {                    // tiles on and below the diagonal
    const int per = tm_n * (tm_n + 1) / 2;
    mat = t / per;
    const int q = t % per;
    tm = (int)((sqrtf(8.f * q + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= q) ++tm;
    while (tm * (tm + 1) / 2 > q) --tm;
    tn = q - tm * (tm + 1) / 2;
  } else {
    const int per = tm_n * tn_n;
    mat = t / per;
    tm = t % per % tm_n;                         // tiles that share X's rows are neighbours
    tn = t % per / tm_n;
  }
  const int64_t xp = (int64_t)mp * np, ap = (int64_t)mp * mp;
  const uint16_t* x = d.x[a.cur] + mat * 2 * xp;
  const uint16_t* xt = d.xt[a.cur] + mat * 2 * xp;
  uint16_t* A = d.a + mat * 2 * ap;
  uint16_t* B = d.b + mat * 2 * ap;
  // operands: rows along the summed axis of length kl
  const uint16_t *lhs, *rhs;
  int64_t lp, rp;
  int kl, rrows;
  if constexpr (PHASE == kMuonGram) { lhs = rhs = x; lp = rp = xp; kl = np; rrows = mp; }
  else if constexpr (PHASE == kMuonPoly) { lhs = rhs = A; lp = rp = ap; kl = mp; rrows = mp; }
  else { lhs = B; lp = ap; rhs = xt; rp = xp; kl = mp; rrows = np; }
  const int lv = mp - tm * BT, rv = rrows - tn * BT;      // rows from the tile's first on
  const char* lb = reinterpret_cast<const char*>(lhs + (int64_t)tm * BT * kl);
  const char* rb = reinterpret_cast<const char*>(rhs + (int64_t)tn * BT * kl);

  auto load = [&](int kt, int st) __attribute__((always_inline)) {
    char* s = smem + st * kStage;
#pragma unroll
    for (int i = 0; i < 4 * BT / 8 / 4; ++i) {
      const int blk = wave + i * 4;              // of 8 rows: BT / 8 of each part
      const int part = blk / (BT / 8), in = blk % (BT / 8);
      const bool left = part < 2;
      const int r = cmin_dev(in * 8 + (lane >> 3), (left ? lv : rv) - 1);
      const char* g = (left ? lb : rb) + (part & 1 ? (left ? lp : rp) * 2 : 0) +
                      ((uint32_t)r * (uint32_t)(kl * 2) + (uint32_t)(kt * 128 + dma_chunk(lane, blk) * 16));
      __builtin_amdgcn_global_load_lds((gbl_cvptr)g, (lds_vptr)(s + blk * 1024), 16, 0, 0);
    }
  };
  f32x16 acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = zero16();
  const int nkt = kl / 64;
  load(0, 0);
  for (int kt = 0; kt < nkt; ++kt) {
    wait_vm_lds<0>();
    lds_barrier();
    if (kt + 1 < nkt) load(kt + 1, (kt + 1) & 1);
    const u32x4* s = reinterpret_cast<const u32x4*>(smem + (kt & 1) * kStage);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const int ch = 2 * ks + (lane >> 5);
      u32x4 ah[F], al[F], bh[F], bl[F];
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int r = wm * F * 32 + i * 32 + (lane & 31), c = wn * F * 32 + i * 32 + (lane & 31);
        ah[i] = s[lds_slot(r, ch)];
        al[i] = s[lds_slot(BT + r, ch)];
        bh[i] = s[lds_slot(2 * BT + c, ch)];
        bl[i] = s[lds_slot(3 * BT + c, ch)];
      }
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
          acc[i][j] = mma_f16(bl[j], ah[i], acc[i][j]);
          acc[i][j] = mma_f16(bh[j], al[i], acc[i][j]);
          acc[i][j] = mma_f16(bh[j], ah[i], acc[i][j]);
        }
    }
  }
  wait_vm_lds<0>();
  lds_barrier();
  // the result in LDS: a lane has row l & 31 of a block, elements 4 q .. of columns 8 q + 4 (l >> 5)
  float* res = reinterpret_cast<float*>(s_mem);
  const float f = (PHASE == kMuonPoly ? a.c : 1.f) / kMuonOne;
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(res + (wm * F * 32 + i * 32 + (lane & 31)) * kRow + wn * F * 32 + j * 32 +
                                   8 * q + 4 * (lane >> 5)) =
            float4{acc[i][j][4 * q] * f, acc[i][j][4 * q + 1] * f, acc[i][j][4 * q + 2] * f,
                   acc[i][j][4 * q + 3] * f};
  __syncthreads();
  const int i0 = tm * BT, j0 = tn * BT;
  // rows of eight: the sum with what is added, and its parts to where they lie along the row
  for (int k = tid; k < BT * BT / 8; k += kMuonThreads) {
    const int r = k / (BT / 8), c = k % (BT / 8) * 8;
    if (i0 + r >= mp || j0 + c >= (kSymmetric ? mp : np)) continue;
    float v[8], w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = res[r * kRow + c + j];
    u32x4 hi, lo;
    if constexpr (PHASE != kMuonGram) {
      const uint16_t* add = PHASE == kMuonPoly ? A + (int64_t)(i0 + r) * mp + j0 + c : x + (int64_t)(i0 + r) * np + j0 + c;
      join8f(*reinterpret_cast<const u32x4*>(add),
             *reinterpret_cast<const u32x4*>(add + (PHASE == kMuonPoly ? ap : xp)), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = fmaf(PHASE == kMuonPoly ? a.b : a.a, w[j], v[j]);
        res[r * kRow + c + j] = v[j];
      }
    }
    if constexpr (PHASE != kMuonLast) {
      split8(v, hi, lo);
      uint16_t* o;
      int64_t op;
      if constexpr (kSymmetric) { o = (PHASE == kMuonGram ? A : B) + (int64_t)(i0 + r) * mp + j0 + c; op = ap; }
      else { o = d.x[a.cur ^ 1] + mat * 2 * xp + (int64_t)(i0 + r) * np + j0 + c; op = xp; }
      *reinterpret_cast<u32x4*>(o) = hi;
      *reinterpret_cast<u32x4*>(o + op) = lo;
    }
  }
  if (kSymmetric && tm == tn) return;
  __syncthreads();
  if constexpr (PHASE != kMuonLast) {            // and along the column
    for (int k = tid; k < BT * BT / 8; k += kMuonThreads) {
      const int c = k % BT, r = k / BT * 8;
      if (i0 + r >= mp || j0 + c >= (kSymmetric ? mp : np)) continue;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = res[(r + j) * kRow + c];
      u32x4 hi, lo;
      split8(v, hi, lo);
      uint16_t* o;
      int64_t op;
      if constexpr (kSymmetric) { o = (PHASE == kMuonGram ? A : B) + (int64_t)(j0 + c) * mp + i0 + r; op = ap; }
      else { o = d.xt[a.cur ^ 1] + mat * 2 * xp + (int64_t)(j0 + c) * mp + i0 + r; op = xp; }
      *reinterpret_cast<u32x4*>(o) = hi;
      *reinterpret_cast<u32x4*>(o + op) = lo;
    }
  } else {
    const int64_t n = (int64_t)d.rows * d.cols;
    T* p = static_cast<T*>(d.p) + mat * n;
    const bool tall = d.rows > d.cols;
    const float rate = d.rate / kMuonOne;
    for (int k = tid; k < BT * BT; k += kMuonThreads) {
      const int fast = k % BT, slow = k / BT;    // the parameter's rows: X's, or its columns
      const int r = tall ? fast : slow, c = tall ? slow : fast;
      const int pr = tall ? j0 + c : i0 + r, pc = tall ? i0 + r : j0 + c;
      if (pr >= d.rows || pc >= d.cols) continue;
      T* e = p + (int64_t)pr * d.cols + pc;
      const float v = res[r * kRow + c];
      store_from_f32(e, a.keep == 0.f ? -rate * v : fmaf(a.keep, load_as_f32(e), -rate * v));
    }
  }
}

}  // namespace dev
}  // namespace tmoe
