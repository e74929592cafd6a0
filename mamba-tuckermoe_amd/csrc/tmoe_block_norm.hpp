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
// Bound by memory: every activation is read once (but for k_block_norm_bwd_wide's rows) and
// every output written once; a row lies in the registers of its threads between its two
// norms, and the next row is on its way meanwhile. Rows of at most 1024 elements take a
// wave, or a half or a quarter of one (no barrier), four neighbours a lane and step; longer
// ones a work-group, 16 bytes a thread and step. The weights' gradients are summed in
// registers over a work-group's rows, then in planes of `part` that k_block_norm_cols adds
// in a fixed order; one work-group alone has them whole. Measured, bf16, T = 16384: d = 768
// with residual, gamma and next norm 17.1 us forward and 25.6 + 4.0 backward (5.9 TB/s of
// what each moves), d = 2304 with every operand 76.8 and 123.2 + 5.2 us (4.9 TB/s; its
// 981 MB don't fit the cache).
#pragma once

#include "tmoe_elem.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace dev {

// Elements a thread holds of a row: NCH steps of EPC neighbours, each one load of any
// alignment (a row of odd width begins anywhere). Where d is no multiple of EPC (kOverlap)
// the last step's are the row's last EPC: the first `dup` of them are its neighbour's too,
// computed and stored alike by both, and left out of the row's sums here. Rows of fewer than
// EPC elements (kTiny) go element by element.
enum RowEnd { kWhole, kOverlap, kTiny };

template <class T, int EPC_, int NCH_, RowEnd kEnd_>
struct RowMap {
  static constexpr int EPC = EPC_, NCH = NCH_, N = NCH * EPC, kWords = EPC * (int)sizeof(T) / 4;
  static constexpr RowEnd kEnd = kEnd_;
  typedef uint32_t vec __attribute__((ext_vector_type(kWords), aligned(sizeof(T))));
  int tid, tpr;
  int64_t d;
  __device__ int64_t first(int k) const { return ((int64_t)k * tpr + tid) * EPC; }
  __device__ bool in(int k) const { return first(k) < d; }
  __device__ int64_t col(int k) const {
    const int64_t c = first(k);
    return kEnd == kOverlap && c > d - EPC ? d - EPC : c;
  }
  // whether element i of the thread's is this thread's to count
  __device__ bool mine(int i) const {
    return kEnd != kOverlap || col(i / EPC) + i % EPC >= first(i / EPC);
  }
};

// A word of ones.
template <class T>
constexpr uint32_t kOneWords = sizeof(T) == 2 ? 0x3f803f80u : 0x3f800000u;

// A row's elements in registers as they are stored.
template <class M, class T>
struct RowRegs {
  uint32_t q[M::NCH][M::kWords];
  __device__ void load(const M& m, const void* base, int64_t row, int64_t stride) {
    const T* p = static_cast<const T*>(base) + row * stride;
#pragma unroll
    for (int k = 0; k < M::NCH; ++k) {
      typename M::vec v = (uint32_t)0;
      if constexpr (M::kEnd == kTiny) {
        for (int j = 0; j < M::EPC; ++j)
          if (m.first(k) + j < m.d) {
            if constexpr (sizeof(T) == 2) v[j / 2] |= (uint32_t)p[m.first(k) + j] << 16 * (j & 1);
            else v[j] = __float_as_uint(p[m.first(k) + j]);
          }
      } else if (m.in(k)) {
        v = *reinterpret_cast<const typename M::vec*>(p + m.col(k));
      }
#pragma unroll
      for (int j = 0; j < M::kWords; ++j) q[k][j] = v[j];
    }
  }
  __device__ void fill(uint32_t word) {
#pragma unroll
    for (int k = 0; k < M::NCH; ++k)
#pragma unroll
      for (int j = 0; j < M::kWords; ++j) q[k][j] = word;
  }
  __device__ float operator[](int i) const {
    const int k = i / M::EPC, j = i % M::EPC;
    if constexpr (sizeof(T) == 4) return __uint_as_float(q[k][j]);
    else return __uint_as_float(j & 1 ? q[k][j / 2] & 0xffff0000u : q[k][j / 2] << 16);
  }
};

template <class T, class M, int N>
__device__ __forceinline__ void row_store(const M& m, void* base, int64_t row, const float (&v)[N]) {
  T* p = static_cast<T*>(base) + row * m.d;
#pragma unroll
  for (int k = 0; k < M::NCH; ++k) {
    if constexpr (M::kEnd == kTiny) {
      for (int j = 0; j < M::EPC; ++j)
        if (m.first(k) + j < m.d) store_from_f32(p + m.first(k) + j, v[k * M::EPC + j]);
    } else if (m.in(k)) {
      typename M::vec q;
#pragma unroll
      for (int j = 0; j < M::kWords; ++j)
        if constexpr (sizeof(T) == 2)
          q[j] = pack_bf16x2(v[k * M::EPC + 2 * j], v[k * M::EPC + 2 * j + 1]);
        else
          q[j] = __float_as_uint(v[k * M::EPC + j]);
      *reinterpret_cast<typename M::vec*>(p + m.col(k)) = q;
    }
  }
}

// Sum over a row's threads (kLanes of a wave, or 0: the work-group), the same value in all of
// them. lds: sixteen floats, zero past
// the work-group's waves, that nobody else has written to since the barrier before the last
// (one barrier a sum).
template <int kLanes>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  v = lanes_sum<kLanes ? kLanes : 64>(v);
  if constexpr (kLanes == 0) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lanes_sum<16>(lds[threadIdx.x & 15]);
  }
  return v;
}
__device__ __forceinline__ void row_sum_clear(float (*lds)[16]) {
  if (threadIdx.x < 64) lds[threadIdx.x >> 4][threadIdx.x & 15] = 0.f;
  __syncthreads();
}

// 1 / (1 + exp(-g)) to about 3 steps of fp32 (the hardware's reciprocal and exponential: an
// exact division would be a third of the gated kernels' instructions)
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
}

constexpr int kNormThreads = 256;   // of a work-group whose rows take at most a wave each

// The step of a kernel over the rows, and its threads' place in a row.
template <class M, int kLanes>
struct RowWalk {
  static constexpr int kTeams = kLanes ? kNormThreads / kLanes : 1;   // rows at a time
  M m;
  int team;
  int64_t row, step;
  __device__ explicit RowWalk(int64_t d)
      : m{kLanes ? (int)(threadIdx.x & (kLanes - 1)) : (int)threadIdx.x,
          kLanes ? kLanes : (int)blockDim.x, d},
        team(kLanes ? (int)(threadIdx.x / (kLanes ? kLanes : 1)) : 0),
        row((int64_t)blockIdx.x * kTeams + team), step((int64_t)gridDim.x * kTeams) {}
};

template <class T, int EPC, int NCH, int kLanes, RowEnd kEnd, int kThreads>
__global__ __launch_bounds__(kThreads) void k_block_norm_fwd(BlockNormArgs a) {
// the same roundings for an element wherever it lies in a thread: fused where it is written
#pragma clang fp contract(off)
  using M = RowMap<T, EPC, NCH, kEnd>;
  using R = RowRegs<M, T>;
  constexpr int N = M::N;
  __shared__ float lds[4][16];
  RowWalk<M, kLanes> w(a.d);
  const M& m = w.m;
  const float inv_d = 1.f / (float)a.d;
  if (kLanes == 0) row_sum_clear(lds);
  R ny, nx, ng;
  nx.fill(0u);
  if (w.row < a.T) {
    ny.load(m, a.y, w.row, a.y_rs);
    if (a.x) nx.load(m, a.x, w.row, a.x_rs);
    if (a.gate) ng.load(m, a.gate, w.row, a.gate_rs);
  }
  int par = 0;
  for (int64_t b = w.row; b < a.T; b += w.step, par ^= 2) {
    const R y = ny, x = nx, g = ng;
    if (b + w.step < a.T) {
      ny.load(m, a.y, b + w.step, a.y_rs);
      if (a.x) nx.load(m, a.x, b + w.step, a.x_rs);
      if (a.gate) ng.load(m, a.gate, b + w.step, a.gate_rs);
    }
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = y[i];
    if (a.gate) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= g[i] * sigmoid(g[i]);
    }
    if (a.post_w) {
      R pw;
      pw.load(m, a.post_w, 0, 0);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) ss = m.mine(i) ? fmaf(f[i], f[i], ss) : ss;
      const float inv = 1.f / sqrtf(row_sum<kLanes>(ss, lds[par]) * inv_d + a.eps);
      if (a.inv && m.tid == 0) a.inv[b] = inv;
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= inv * pw[i];
    }
    R gm;
    if (a.gamma) gm.load(m, a.gamma, 0, 0);
    else gm.fill(kOneWords<T>);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = fmaf(f[i], gm[i], x[i]);
    if (a.r) row_store<T>(m, a.r, b, f);
    if (a.next_w) {
      R nw;
      nw.load(m, a.next_w, 0, 0);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) ss = m.mine(i) ? fmaf(f[i], f[i], ss) : ss;
      const float inv = 1.f / sqrtf(row_sum<kLanes>(ss, lds[par + 1]) * inv_d + a.eps);
      if (a.inv && m.tid == 0) a.inv[a.T + b] = inv;
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= inv * nw[i];
      row_store<T>(m, a.h, b, f);
    }
  }
}

// A work-group's sums of one weight's gradient: its plane of part (3, work-groups, d), or
// the gradient itself of the only work-group.
template <class T, class M, int N>
__device__ __forceinline__ void put_sums(const M& m, const BlockNormArgs& a, const float (&v)[N],
                                         int which, void* out) {
  if (!out) return;
  if (gridDim.x == 1) return row_store<T>(m, out, 0, v);
  float* p = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.d;
#pragma unroll
  for (int k = 0; k < M::NCH; ++k)
#pragma unroll
    for (int j = 0; j < M::EPC; ++j)
      if (m.in(k) && m.col(k) + j < a.d) p[m.col(k) + j] = v[k * M::EPC + j];
}

// What a backward's rows load and store as the bits of F: known when it is compiled, with
// dr (and dh with kNext) there and every row's gradient wanted, so that the loads and stores
// have their places and none waits for another (a load of the next row that may or may not
// be followed by a store is waited for with that store); F = -1 looks at the pointers.
// kFull: with a gate or a norm after the block; without, neither's registers are held.
constexpr int kGate = 1, kRes = 2, kNext = 4, kPost = 8;

template <class T, int EPC, int NCH, int kLanes, RowEnd kEnd, int kThreads, bool kFull, int F>
__global__ __launch_bounds__(kThreads) void k_block_norm_bwd(BlockNormArgs a) {
// the same roundings for an element wherever it lies, and whichever gradients are wanted:
// fused where it is written
#pragma clang fp contract(off)
  using M = RowMap<T, EPC, NCH, kEnd>;
  using R = RowRegs<M, T>;
  constexpr int N = M::N;
  constexpr bool kAny = F < 0;
  __shared__ float lds[4][16];
  RowWalk<M, kLanes> w(a.d);
  const M& m = w.m;
  const float inv_d = 1.f / (float)a.d;
  if (kLanes == 0) row_sum_clear(lds);
  const bool gated = kFull && (kAny ? a.gate != nullptr : (F & kGate) != 0);
  const bool post = kFull && (kAny ? a.post_w != nullptr : (F & kPost) != 0);
  const bool res = kAny ? a.x != nullptr : (F & kRes) != 0;
  const bool next = kAny ? a.dh != nullptr : (F & kNext) != 0;
  const bool dr_in = kAny ? a.dr != nullptr : true;
  float s_post[kFull ? N : 1], s_gamma[N], s_next[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (kFull) s_post[i] = 0.f;
    s_gamma[i] = s_next[i] = 0.f;
  }
  R pw, gm, nw;
  if (post) pw.load(m, a.post_w, 0, 0);
  if (a.gamma) gm.load(m, a.gamma, 0, 0);
  else gm.fill(kOneWords<T>);   // a product by one: the same bits as without it
  if (next) nw.load(m, a.next_w, 0, 0);
  R ny, nx, ng, ndr, ndh;
  float n_u = 1.f, n_r = 0.f;
  auto fetch = [&](int64_t b) {
    ny.load(m, a.y, b, a.y_rs);
    if (gated) ng.load(m, a.gate, b, a.gate_rs);
    if (next) {
      ndh.load(m, a.dh, b, a.dh_rs);
      if (res) nx.load(m, a.x, b, a.x_rs);
      n_r = a.inv[a.T + b];
    }
    if (dr_in) ndr.load(m, a.dr, b, a.dr_rs);
    if (post) n_u = a.inv[b];
  };
  constexpr bool kAhead = kThreads <= 512;   // past that a thread's registers hold one row only
  if (kAhead && w.row < a.T) fetch(w.row);
  int par = 0;
  for (int64_t b = w.row; b < a.T; b += w.step, par ^= 2) {
    if (!kAhead) fetch(b);
    const R y = ny, x = nx, g = ng, dr = ndr, dh = ndh;
    const float inv_u = n_u, inv_r = n_r;
    if (kAhead) fetch(b + w.step < a.T ? b + w.step : b);
    // sigmoid(gate); nu (u where no norm follows the block); D
    float sg[kFull ? N : 1], nu[N], D[N];
#pragma unroll
    for (int i = 0; i < N; ++i) nu[i] = y[i];
    if constexpr (kFull) {
      if (gated) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sg[i] = sigmoid(g[i]);
          nu[i] *= g[i] * sg[i];
        }
      }
      if (post) {
#pragma unroll
        for (int i = 0; i < N; ++i) nu[i] *= inv_u;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) D[i] = 0.f;
    if (dr_in) {
#pragma unroll
      for (int i = 0; i < N; ++i) D[i] = dr[i];
    }
    if (next) {
      float nr[N], dot = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) nr[i] = nu[i];
      if constexpr (kFull)
        if (post) {
#pragma unroll
          for (int i = 0; i < N; ++i) nr[i] *= pw[i];
        }
#pragma unroll
      for (int i = 0; i < N; ++i) nr[i] = res ? fmaf(nr[i], gm[i], x[i]) : nr[i] * gm[i];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        nr[i] *= inv_r;
        const float t = dh[i] * nr[i];
        s_next[i] += t;
        dot = m.mine(i) ? fmaf(t, nw[i], dot) : dot;
      }
      dot = row_sum<kLanes>(dot, lds[par]) * inv_d * inv_r;
#pragma unroll
      for (int i = 0; i < N; ++i) D[i] = fmaf(-nr[i], dot, fmaf(dh[i] * nw[i], inv_r, D[i]));
    }
    if (kAny ? a.dx != nullptr : res) row_store<T>(m, a.dx, b, D);
    if (post) {
      if constexpr (kFull) {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          s_gamma[i] = fmaf(D[i], nu[i] * pw[i], s_gamma[i]);
          D[i] *= gm[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float t = D[i] * nu[i];
          s_post[i] += t;
          dot = m.mine(i) ? fmaf(t, pw[i], dot) : dot;
        }
        dot = row_sum<kLanes>(dot, lds[par + 1]) * inv_d * inv_u;
#pragma unroll
        for (int i = 0; i < N; ++i) D[i] = fmaf(-nu[i], dot, D[i] * pw[i] * inv_u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s_gamma[i] = fmaf(D[i], nu[i], s_gamma[i]);
        D[i] *= gm[i];
      }
    }
    if constexpr (kFull)
      if (gated) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          // silu' = s (1 + g (1 - s))
          nu[i] = D[i] * y[i] * (sg[i] * fmaf(g[i], 1.f - sg[i], 1.f));
          D[i] *= g[i] * sg[i];
        }
        if (kAny ? a.dgate != nullptr : true) row_store<T>(m, a.dgate, b, nu);
      }
    if (kAny ? a.dy != nullptr : true) row_store<T>(m, a.dy, b, D);
  }
  if (!a.dpost_w && !a.dgamma && !a.dnext_w) return;
  // a work-group's rows apart: their sums over it first, in the order of the teams
  if constexpr (kLanes > 0) {
    constexpr int kTeams = RowWalk<M, kLanes>::kTeams;
    __shared__ float s[kTeams][N * kLanes];
    auto join = [&](float (&v)[N]) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) s[w.team][i * kLanes + m.tid] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int t = 0; t < kTeams; ++t) v[i] += s[t][i * kLanes + m.tid];
      }
    };
    if constexpr (kFull)
      if (a.dpost_w) join(s_post);
    if (a.dgamma) join(s_gamma);
    if (a.dnext_w) join(s_next);
    if (w.team > 0) return;
  }
  if constexpr (kFull) put_sums<T>(m, a, s_post, 0, a.dpost_w);
  put_sums<T>(m, a, s_gamma, 1, a.dgamma);
  put_sums<T>(m, a, s_next, 2, a.dnext_w);
}

// The backward of rows whose fp32 values no thread's registers hold: a row is read twice,
// the second time from the cache, some neighbours a thread at a time; only the weights'
// sums stay. One pass takes what both norms need of the row (D's parts by themselves, since
// D is not known yet):
//   s1 = sum q nr;  s2 = sum (dr + q / rms(r)) e,  s3 = sum nr e,  e = nu gamma post_w
//   sum D e = s2 - s1 s3 / (d rms(r))
// and the other one forms the gradients. Without a norm there is that one alone. Four
// elements a thread and step: eight hold more than the registers left beside the sums.
// d = 9216, bf16, T = 4096: 73 us with a gate alone (5.2 TB/s of what has to be moved), 182
// with every operand (3.3 TB/s); d = 16384, T = 2048, residual and next norm 118 (3.4 TB/s).
template <class T, int NCH, RowEnd kEnd, int F>
__global__ __launch_bounds__(1024) void k_block_norm_bwd_wide(BlockNormArgs a) {
#pragma clang fp contract(off)
  constexpr int N = 4;
  using M = RowMap<T, N, 1, kEnd>;
  using R = RowRegs<M, T>;
  constexpr bool kAny = F < 0;
  __shared__ float lds[6][16];
  if (threadIdx.x < 96) lds[threadIdx.x >> 4][threadIdx.x & 15] = 0.f;
  __syncthreads();
  const int tid = threadIdx.x, tpr = blockDim.x;
  const float inv_d = 1.f / (float)a.d;
  const bool gated = kAny ? a.gate != nullptr : (F & kGate) != 0;
  const bool post = kAny ? a.post_w != nullptr : (F & kPost) != 0;
  const bool res = kAny ? a.x != nullptr : (F & kRes) != 0;
  const bool next = kAny ? a.dh != nullptr : (F & kNext) != 0;
  const bool dr_in = kAny ? a.dr != nullptr : true;
  const bool sums = a.dpost_w || a.dgamma || a.dnext_w;
  float s_post[NCH][N] = {}, s_gamma[NCH][N] = {}, s_next[NCH][N] = {};
  int par = 0;
  for (int64_t b = blockIdx.x; b < a.T; b += gridDim.x, par ^= 3) {
    const float inv_u = post ? a.inv[b] : 1.f, inv_r = next ? a.inv[a.T + b] : 0.f;
    R y, x, g, dr, dh, pw, gm, nw;
    x.fill(0u), dr.fill(0u), gm.fill(kOneWords<T>), pw.fill(kOneWords<T>);
    const auto fetch = [&](const M& m) {
      y.load(m, a.y, b, a.y_rs);
      if (gated) g.load(m, a.gate, b, a.gate_rs);
      if (next) {
        dh.load(m, a.dh, b, a.dh_rs);
        nw.load(m, a.next_w, 0, 0);
        if (res) x.load(m, a.x, b, a.x_rs);
      }
      if (dr_in) dr.load(m, a.dr, b, a.dr_rs);
      if (post) pw.load(m, a.post_w, 0, 0);
      if (a.gamma) gm.load(m, a.gamma, 0, 0);
    };
    // nu and nr of the thread's elements, and D without the norm's mean
    float sg[N], nu[N], nr[N], D[N];
    const auto form = [&]() {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        nu[i] = y[i];
        D[i] = dr[i];
      }
      if (gated) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sg[i] = sigmoid(g[i]);
          nu[i] *= g[i] * sg[i];
        }
      }
      if (post) {
#pragma unroll
        for (int i = 0; i < N; ++i) nu[i] *= inv_u;
      }
      if (next) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          nr[i] = fmaf(nu[i] * pw[i], gm[i], x[i]) * inv_r;
          D[i] = fmaf(dh[i] * nw[i], inv_r, D[i]);
        }
      }
    };
    float s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (next || post) {
#pragma unroll 1
      for (int k = 0; k < NCH; ++k) {
        const M m{tid + k * tpr, tpr, a.d};
        fetch(m);
        form();
        if (next) {
#pragma unroll
          for (int i = 0; i < N; ++i) s1 = m.mine(i) ? fmaf(dh[i] * nr[i], nw[i], s1) : s1;
        }
        if (post) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float e = nu[i] * gm[i] * pw[i];
            s2 = m.mine(i) ? fmaf(D[i], e, s2) : s2;
            if (next) s3 = m.mine(i) ? fmaf(nr[i], e, s3) : s3;
          }
        }
      }
      s1 = lanes_sum<64>(s1), s2 = lanes_sum<64>(s2), s3 = lanes_sum<64>(s3);
      if ((tid & 63) == 0) {
        lds[par][tid >> 6] = s1;
        lds[par + 1][tid >> 6] = s2;
        lds[par + 2][tid >> 6] = s3;
      }
      __syncthreads();
      s1 = lanes_sum<16>(lds[par][tid & 15]) * inv_d * inv_r;
      s3 = lanes_sum<16>(lds[par + 2][tid & 15]);
      s2 = fmaf(-s1, s3, lanes_sum<16>(lds[par + 1][tid & 15])) * inv_d * inv_u;
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const M m{tid + k * tpr, tpr, a.d};
      fetch(m);
      form();
      if (next) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          s_next[k][i] += dh[i] * nr[i];
          D[i] = fmaf(-nr[i], s1, D[i]);
        }
      }
      if (kAny ? a.dx != nullptr : res) row_store<T>(m, a.dx, b, D);
#pragma unroll
      for (int i = 0; i < N; ++i) s_gamma[k][i] = fmaf(D[i], nu[i] * pw[i], s_gamma[k][i]);
#pragma unroll
      for (int i = 0; i < N; ++i) D[i] *= gm[i];
      if (post) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          s_post[k][i] += D[i] * nu[i];
          D[i] = fmaf(-nu[i], s2, D[i] * pw[i] * inv_u);
        }
      }
      if (gated) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          nu[i] = D[i] * y[i] * (sg[i] * fmaf(g[i], 1.f - sg[i], 1.f));
          D[i] *= g[i] * sg[i];
        }
        if (kAny ? a.dgate != nullptr : true) row_store<T>(m, a.dgate, b, nu);
      }
      if (kAny ? a.dy != nullptr : true) row_store<T>(m, a.dy, b, D);
      __builtin_amdgcn_sched_barrier(0);      // one step's registers at a time
    }
  }
  if (!sums) return;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const M m{tid + k * tpr, tpr, a.d};
    put_sums<T>(m, a, s_post[k], 0, a.dpost_w);
    put_sums<T>(m, a, s_gamma[k], 1, a.dgamma);
    put_sums<T>(m, a, s_next[k], 2, a.dnext_w);
  }
}

// The weights' gradients from the backward's planes: 32 columns of one weight a work-group,
// its 32 groups of threads to the planes.
template <class T>
__global__ __launch_bounds__(1024) void k_block_norm_cols(BlockNormArgs a, int64_t planes) {
  T* out = static_cast<T*>(blockIdx.y == 0 ? a.dpost_w : blockIdx.y == 1 ? a.dgamma : a.dnext_w);
  if (!out) return;   // uniform over the work-group
  __shared__ float s[32][33];
  const int g = threadIdx.x >> 5, l = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * 32 + l;
  const float* p = a.part + blockIdx.y * planes * a.d + c;
  float v = 0.f;
  if (c < a.d)
#pragma unroll 8
    for (int64_t i = g; i < planes; i += 32) v += p[i * a.d];
  s[g][l] = v;
  __syncthreads();
  v = s[l][g];          // column g's sums in the lanes of half a wave
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  const int64_t col = (int64_t)blockIdx.x * 32 + g;
  if (l == 0 && col < a.d) store_from_f32(out + col, v);
}

}  // namespace dev
}  // namespace tmoe
