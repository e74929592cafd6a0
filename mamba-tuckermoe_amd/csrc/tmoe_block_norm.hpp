// The norms before and after a block, fused with the block's gate and the residual's scale
// (pure_torch_mlx/model.py:258-260, :337-341 around a sub-block; every operand but y optional):
//   u = y silu(gate);  f = u / rms(u) post_w;  r = x + gamma f;  h = r / rms(r) next_w
// with rms(v) = sqrt(mean(v^2) + eps), and their gradient. With nu = u / rms(u),
// nr = r / rms(r), from dr and dh:
//   q = dh next_w;   D = dr + (q - nr mean(q nr)) / rms(r);   dx = D
//   df = D gamma;    v = df post_w;   du = (v - nu mean(v nu)) / rms(u)
//   dy = du silu(gate);  dgate = du y silu'(gate)
//   dnext_w = sum dh nr,  dgamma = sum D f,  dpost_w = sum df nu      (over the rows)
// All in fp32 from the stored inputs; h is taken from the unrounded r, and the backward
// forms r again from x and y, so that both see the same r; each output is rounded once.
//
// Bound by memory: every activation is read once and every output written once, a row's
// chunks of 16 bytes lie in the registers of its lanes between the two norms. Rows of at
// most kWaveChunks chunks a lane take one wave (no barrier), longer ones a work-group of
// as many waves as the row has chunks for. The weights' gradients are summed in registers
// over a work-group's rows, then in planes of `part` that k_block_norm_cols adds in order.
#pragma once

#include "tmoe_elem.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace dev {

// Threads of one row and where each of its elements lies. kVec: chunks of 16 bytes, one
// chunk a thread and step; else element by element, neighbours on neighbouring threads.
template <class T, int NCH, bool kVec>
struct RowMap {
  static constexpr int EPC = 16 / (int)sizeof(T), N = NCH * EPC;
  int tid, tpr;
  int64_t d;
  __device__ int64_t col(int k, int j) const {
    return kVec ? ((int64_t)k * tpr + tid) * EPC + j : ((int64_t)k * EPC + j) * tpr + tid;
  }
  __device__ bool in(int k, int j) const { return col(k, kVec ? 0 : j) < d; }
  __device__ void load(const void* base, float v[N]) const {
    const T* p = static_cast<const T*>(base);
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      if constexpr (kVec) {
        u32x4 q = {0u, 0u, 0u, 0u};
        if (in(k, 0)) q = *reinterpret_cast<const u32x4*>(p + col(k, 0));
        const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int j = 0; j < EPC; ++j) v[k * EPC + j] = load_as_f32(e + j);
      } else {
#pragma unroll
        for (int j = 0; j < EPC; ++j) v[k * EPC + j] = in(k, j) ? load_as_f32(p + col(k, j)) : 0.f;
      }
    }
  }
  __device__ void store(void* base, const float v[N]) const {
    T* p = static_cast<T*>(base);
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      if constexpr (kVec) {
        if (!in(k, 0)) continue;
        u32x4 q;
        T* e = reinterpret_cast<T*>(&q);
#pragma unroll
        for (int j = 0; j < EPC; ++j) store_from_f32(e + j, v[k * EPC + j]);
        *reinterpret_cast<u32x4*>(p + col(k, 0)) = q;
      } else {
#pragma unroll
        for (int j = 0; j < EPC; ++j)
          if (in(k, j)) store_from_f32(p + col(k, j), v[k * EPC + j]);
      }
    }
  }
};

// Sum over a row's threads, the same value in all of them.
template <bool kWave>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (!kWave) {
    const int W = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < W; ++w) v += lds[w];
    __syncthreads();
  }
  return v;
}

__device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + __expf(-g)); }

template <class T>
__device__ __forceinline__ const void* row_at(const void* p, int64_t row, int64_t stride) {
  return static_cast<const T*>(p) + row * stride;
}
template <class T>
__device__ __forceinline__ void* row_at(void* p, int64_t row, int64_t stride) {
  return static_cast<T*>(p) + row * stride;
}

constexpr int kNormThreads = 256;   // of a work-group whose rows take a wave each

template <class T, int NCH, bool kWave, bool kVec>
__global__ __launch_bounds__(kWave ? kNormThreads : 1024) void k_block_norm_fwd(BlockNormArgs a) {
  using M = RowMap<T, NCH, kVec>;
  constexpr int N = M::N;
  __shared__ float lds[16];
  const M m = {kWave ? (int)(threadIdx.x & 63) : (int)threadIdx.x, kWave ? 64 : (int)blockDim.x, a.d};
  const int teams = kWave ? kNormThreads / 64 : 1;
  const int64_t first = (int64_t)blockIdx.x * teams + (kWave ? threadIdx.x >> 6 : 0);
  const float inv_d = 1.f / (float)a.d;
  for (int64_t b = first; b < a.T; b += (int64_t)gridDim.x * teams) {
    float f[N], x[N];
    m.load(row_at<T>(a.y, b, a.y_rs), f);
    if (a.x) m.load(row_at<T>(a.x, b, a.x_rs), x);
    if (a.gate) {
      float g[N];
      m.load(row_at<T>(a.gate, b, a.gate_rs), g);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= g[i] * sigmoid(g[i]);
    }
    if (a.post_w) {
      float w[N], ss = 0.f;
      m.load(a.post_w, w);
#pragma unroll
      for (int i = 0; i < N; ++i) ss += f[i] * f[i];
      const float inv = 1.f / sqrtf(row_sum<kWave>(ss, lds) * inv_d + a.eps);
      if (a.inv && m.tid == 0) a.inv[b] = inv;
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= inv * w[i];
    }
    if (a.gamma) {
      float w[N];
      m.load(a.gamma, w);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= w[i];
    }
    if (a.x) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] += x[i];
    }
    if (a.r) m.store(row_at<T>(a.r, b, a.d), f);
    if (a.next_w) {
      float w[N], ss = 0.f;
      m.load(a.next_w, w);
#pragma unroll
      for (int i = 0; i < N; ++i) ss += f[i] * f[i];
      const float inv = 1.f / sqrtf(row_sum<kWave>(ss, lds) * inv_d + a.eps);
      if (a.inv && m.tid == 0) a.inv[a.T + b] = inv;
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= inv * w[i];
      m.store(row_at<T>(a.h, b, a.d), f);
    }
  }
}

template <class T, int NCH, bool kWave, bool kVec>
__global__ __launch_bounds__(kWave ? kNormThreads : 1024) void k_block_norm_bwd(BlockNormArgs a) {
  using M = RowMap<T, NCH, kVec>;
  constexpr int N = M::N;
  __shared__ float lds[16];
  const M m = {kWave ? (int)(threadIdx.x & 63) : (int)threadIdx.x, kWave ? 64 : (int)blockDim.x, a.d};
  const int teams = kWave ? kNormThreads / 64 : 1;
  const int64_t first = (int64_t)blockIdx.x * teams + (kWave ? threadIdx.x >> 6 : 0);
  const float inv_d = 1.f / (float)a.d;
  float s_post[N], s_gamma[N], s_next[N];
#pragma unroll
  for (int i = 0; i < N; ++i) s_post[i] = s_gamma[i] = s_next[i] = 0.f;
  for (int64_t b = first; b < a.T; b += (int64_t)gridDim.x * teams) {
    // u (in f), then f
    float y[N], f[N], D[N];
    m.load(row_at<T>(a.y, b, a.y_rs), y);
    if (a.dr) m.load(row_at<T>(a.dr, b, a.dr_rs), D);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f[i] = y[i];
      if (!a.dr) D[i] = 0.f;
    }
    if (a.gate) {
      float g[N];
      m.load(row_at<T>(a.gate, b, a.gate_rs), g);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= g[i] * sigmoid(g[i]);
    }
    float inv_u = 0.f;
    if (a.post_w) {
      float w[N];
      m.load(a.post_w, w);
      inv_u = a.inv[b];
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= inv_u * w[i];
    }
    float gm[N];
    if (a.gamma) m.load(a.gamma, gm);
    if (a.dh) {
      float r[N], w[N], dh[N];
      m.load(row_at<T>(a.dh, b, a.dh_rs), dh);
      m.load(a.next_w, w);
      if (a.x) m.load(row_at<T>(a.x, b, a.x_rs), r);
      const float inv_r = a.inv[a.T + b];
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = a.gamma ? f[i] * gm[i] : f[i];
        r[i] = (a.x ? r[i] + v : v) * inv_r;       // nr
        s_next[i] += dh[i] * r[i];
        dh[i] *= w[i];
        dot += dh[i] * r[i];
      }
      dot = row_sum<kWave>(dot, lds) * inv_d;
#pragma unroll
      for (int i = 0; i < N; ++i) D[i] += (dh[i] - r[i] * dot) * inv_r;
    }
    if (a.dx) m.store(row_at<T>(a.dx, b, a.d), D);
    if (a.gamma) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s_gamma[i] += D[i] * f[i];
        D[i] *= gm[i];
      }
    }
    if (a.post_w) {
      // nu from y and the gate again: f has the weight in it, which may be zero
      float w[N], g[N], dot = 0.f;
      m.load(a.post_w, w);
      if (a.gate) m.load(row_at<T>(a.gate, b, a.gate_rs), g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        f[i] = (a.gate ? y[i] * (g[i] * sigmoid(g[i])) : y[i]) * inv_u;
        s_post[i] += D[i] * f[i];
        D[i] *= w[i];
        dot += D[i] * f[i];
      }
      dot = row_sum<kWave>(dot, lds) * inv_d;
#pragma unroll
      for (int i = 0; i < N; ++i) D[i] = (D[i] - f[i] * dot) * inv_u;
    }
    if (a.gate) {
      float g[N];
      m.load(row_at<T>(a.gate, b, a.gate_rs), g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float s = sigmoid(g[i]);
        y[i] *= D[i] * (s * (1.f + g[i] * (1.f - s)));
        D[i] *= g[i] * s;
      }
      if (a.dgate) m.store(row_at<T>(a.dgate, b, a.d), y);
    }
    if (a.dy) m.store(row_at<T>(a.dy, b, a.d), D);
  }
  // part: (3, planes, d); a plane for each row of threads
  if (!a.part) return;
  const int64_t planes = (int64_t)gridDim.x * teams;
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int j = 0; j < M::EPC; ++j) {
      const int64_t c = m.col(k, j);
      if (c >= a.d) continue;
      const int i = k * M::EPC + j;
      if (a.dpost_w) a.part[(0 * planes + first) * a.d + c] = s_post[i];
      if (a.dgamma) a.part[(1 * planes + first) * a.d + c] = s_gamma[i];
      if (a.dnext_w) a.part[(2 * planes + first) * a.d + c] = s_next[i];
    }
}

// The weights' gradients from the backward's planes: 64 columns of one weight a work-group.
template <class T>
__global__ __launch_bounds__(1024) void k_block_norm_cols(BlockNormArgs a, int64_t planes) {
  T* out = static_cast<T*>(blockIdx.y == 0 ? a.dpost_w : blockIdx.y == 1 ? a.dgamma : a.dnext_w);
  if (!out) return;   // uniform over the work-group
  __shared__ float s[16][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float* p = a.part + blockIdx.y * planes * a.d + c;
  float v = 0.f;
  if (c < a.d)
#pragma unroll 8
    for (int64_t i = threadIdx.x >> 6; i < planes; i += 16) v += p[i * a.d];
  s[threadIdx.x >> 6][threadIdx.x & 63] = v;
  __syncthreads();
  if (threadIdx.x < 64 && c < a.d) {
    v = 0.f;
#pragma unroll
    for (int g = 0; g < 16; ++g) v += s[g][threadIdx.x];
    store_from_f32(out + c, v);
  }
}

}  // namespace dev
}  // namespace tmoe
