// The training layer's router with its losses (sft_cot_bundle/scripts/model.py:318-332) and
// their gradient. For a token's logits raw (E), c = cap, tau = temperature:
//   a = c tanh(raw / c);  P = softmax(a / tau);  idx = the k largest raw, the lowest index
//   on ties (the cap and the temperature are monotone);  s = sum_j P[idx_j] + 1e-6;
//   w_j = P[idx_j] / s
//   lb = E sum_e (n_e / N) (sum_b P_be / N),  z = sum_b lse(a_b)^2 / N
// over the N tokens that no mask leaves out, n_e of which select e. A masked token has
// idx -1 (which selects nothing in the contraction), w 0 and no gradient.
//   G_e  = dlb E n_e / N^2,  A_e = [e = idx_j] (dw_j - sum_i dw_i w_i) / s
//   draw = (1 - tanh^2) (P_e (G_e + A_e - sum_f P_f (G_f + A_f)) / tau + dz 2 lse softmax(a)_e / N)
// where differences of G and dw are taken from the likeliest expert's (G_0, dw_0): with its P
// near 1 the sums are next to those, and the differences what is left of two equals. The mean
// of A is 1e-6 / s sum_i dw_i w_i, since the weights lack 1e-6 / s of one. So with
// D = sum_i w_i (dw_i - dw_0), S and U the selected and the other P's sums, no sum is taken
// from one that may be next to it:
//   A_e - mean = ((dw_j - dw_0) - D + 1e-6 (dw_0 U / s - D)) / s where selected, else
//                -1e-6 (dw_0 S / s + D) / s
//
// With Q = exp(-2 raw / c) and R = 1 / (1 + Q), tanh = 1 - 2 Q R, 1 - tanh^2 = 4 Q R^2 and
//   a_e - a_m = 2 c R_m R_e (Q_m - Q_e)
// for the largest logit m: the exponents of both softmaxes without the cancellation of two
// capped logits near the cap. raw / c is cut at +-20, past which tanh is +-1 in fp32. A Q near
// 1 has cap 2^-24 of a logit as its last place: for caps past 16 the capped logits' own
// differences are taken (the backward's 1 - tanh^2 stays of Q).
//
// A token's logits lie in L lanes, V to a lane (L a power of two, V L >= E; V = 8, or 4 where
// that is all of them): what a token needs of them is exchanged by lane permutations, what
// k lanes store or read is handed through shared memory, so that idx, w and dw are moved
// side by side. Eight to a lane rather than four: the exchanges, and not the exponentials,
// are most of the instructions (forward 29 against 32 us when that was measured). Bound by
// instructions (the vector units work 74% and 72% of the time): E = 64, k = 6, B = 131072
// (fp32) takes 22.3 us forward (1.9 TB/s of what it moves) and 21.9 backward (3.5 TB/s);
// B = 16384, E = 8, k = 2 5.3 and 5.4 us. The column
// sums over the tokens (sum_b P_be in registers, n_e in shared memory) are a work-group's
// own until its plane of `part`, and k_router_finish adds the planes in a fixed order: the
// losses do not depend on which work-group ends first.
#pragma once

#include "tmoe_elem.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace dev {

constexpr int kRouterThreads = 256;
constexpr int kRouterTopK = 16;       // slots of a token at most
constexpr int kFinishCols = 16;       // experts of a work-group of k_router_finish

// raw[e0 .. e0 + V - 1] of a row of E logits (-inf past its end), at any alignment
template <class T, int V>
__device__ __forceinline__ void router_load(const T* row, int e0, int E, float v[V]) {
  constexpr int W = V * (int)sizeof(T) / 4;
  typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  if (e0 + V <= E) {
    const vec q = *reinterpret_cast<const vec*>(row + e0);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(q[j]);
      else v[j] = __uint_as_float(j & 1 ? q[j / 2] & 0xffff0000u : q[j / 2] << 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = e0 + j < E ? load_as_f32(row + e0 + j) : -INFINITY;
  }
}

template <int V>
__device__ __forceinline__ uint32_t max_of(const uint32_t (&k)[V]) {
  uint32_t m = max(k[0], k[1]);
#pragma unroll
  for (int j = 2; j < V; j += 2) m = max(m, max(k[j], k[j + 1]));
  return m;
}

// An unsigned key in the order of the floats: NaN above +inf, -0 equal to 0, never 0; and
// the float of a key.
__device__ __forceinline__ uint32_t order_key(float f) {
  const int32_t b = (int32_t)__float_as_uint(f + 0.f);
  return f != f ? 0xffffffffu : (uint32_t)(b ^ (b >> 31 | (int32_t)0x80000000));
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct Capped {
  float Q, R;
};
// u = raw c1, c1 = -2 log2(e) / cap
__device__ __forceinline__ Capped capped_of(float u) {
  const float Q = __builtin_amdgcn_exp2f(u);
  return {Q, __builtin_amdgcn_rcpf(1.f + Q)};
}
constexpr float kCut = 20.f * 2.8853900817779268f;
// of a token's largest logit: a NaN stays one, and makes all that is taken from it NaN
__device__ __forceinline__ Capped capped_top(float raw, float c1) {
  const float u = raw * c1;
  return capped_of(u > kCut ? kCut : u < -kCut ? -kCut : u);
}
__device__ __forceinline__ Capped capped(float raw, float c1) {
  return capped_of(__builtin_amdgcn_fmed3f(raw * c1, -kCut, kCut));
}

// cap tanh(raw / cap) to the last places, for the logsumexp: once a token
__device__ __forceinline__ float capped_value(float raw, float c1, float cap) {
  const float q = __builtin_amdgcn_exp2f(-fabsf(raw * c1)), d = 1.f + q;
  const float r = __builtin_amdgcn_rcpf(d);
  return copysignf(cap * ((1.f - q) * fmaf(r, fmaf(-d, r, 1.f), r)), raw);
}
// The same to the last places of itself, also where the cap is far off: below a quarter of it
// tanh's series, the terms up to x^9 (the next is under 2^-26 of the sum).
__device__ __forceinline__ float capped_far(float raw, float c1, float cap) {
  const float x = raw * c1 * -0.34657359028f, s = x * x;     // raw / cap and its square
  const float p = fmaf(s, fmaf(s, fmaf(s, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f);
  return fabsf(x) < 0.25f ? fmaf(raw * s, p, raw) : capped_value(raw, c1, cap);
}

// Where a token's lanes keep expert e's word among them: the lanes' j-th words are
// neighbours, and tokens lie (V + 1) L words apart, so that a wave meets every bank alike.
template <int L, int V>
__device__ __forceinline__ uint32_t place(uint32_t e) {
  return e % V * L + e / V;
}

// The largest key below `best`; one exists, or a key of 0 is none.
template <int L, int V>
__device__ __forceinline__ uint32_t key_below(const uint32_t (&key)[V], uint32_t best) {
  uint32_t below[V];
#pragma unroll
  for (int j = 0; j < V; ++j) below[j] = key[j] - best;
  return lanes_max<L>(max_of(below)) + best;
}

// Past this cap the differences of Q lose more places (the cap's) than those of the capped
// logits, which are then taken themselves.
constexpr float kFarCap = 16.f;

struct RouterScales {
  float c1, cap, k_z, k_p;   // exponents in base 2 of a token's distances, of both softmaxes
  bool far;
  __device__ RouterScales(const RouterArgs& a) {
    const float tau = a.tau_dev ? *a.tau_dev : a.tau;
    far = a.cap > kFarCap;
    c1 = -2.8853900817779268f / a.cap;
    cap = a.cap;
    k_z = far ? 1.4426950408889634f : 2.8853900817779268f * a.cap;
    k_p = k_z / tau;
  }
  __device__ float value(float raw) const {
    return far ? capped_far(raw, c1, cap) : capped_value(raw, c1, cap);
  }
};
// The distances of a token's capped logits from its largest's, as they stand (far), or without
// the factor that k_z and k_p get here: R_e (Q_m - Q_e) of 2 c R_m R_e (Q_m - Q_e).
template <int V>
struct RouterToken {
  float k_z, k_p, d[V];
  __device__ __forceinline__ RouterToken(const RouterScales& s, const float (&v)[V],
                                         const Capped (&t)[V], float top)
      : k_z(s.k_z), k_p(s.k_p) {
    if (s.far) {
      const float most = capped_far(top, s.c1, s.cap);
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = capped_far(v[j], s.c1, s.cap) - most;
    } else {
      const Capped m = capped_top(top, s.c1);
      k_z *= m.R;
      k_p *= m.R;
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = (m.Q - t[j].Q) * t[j].R;
    }
  }
};

// counts, lb, z and N of column sums that are whole: ps, cn of expert e in the lanes of
// this wave (nothing past E), every lane the same z and n. lb's part of these experts.
__device__ __forceinline__ float router_finish_wave(const RouterArgs& a, int e, float ps, uint32_t cn,
                                                    float inv_n) {
  float t = 0.f;
  if (e < a.E) {
    a.counts[e] = cn;
    t = ((float)cn * inv_n) * (ps * inv_n);
  }
  return lanes_sum<64>(t);
}

template <class T, int L, int V>
__global__ __launch_bounds__(kRouterThreads) void k_router_fwd(RouterArgs a) {
  constexpr int G = kRouterThreads / L;
  const T* raw = static_cast<const T*>(a.raw);
  const int E = a.E, k = a.k, l = threadIdx.x & (L - 1), e0 = V * l;
  const RouterScales sc(a);
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t b = (int64_t)blockIdx.x * G + threadIdx.x / L;
  float ps[V] = {}, zs = 0.f;
  uint32_t low[V], n = 0u;
#pragma unroll
  for (int j = 0; j < V; ++j) low[j] = 255u - (uint32_t)(e0 + j);
  // a token's selected keys, by rank, and its exponentials: handed from the lanes that
  // hold them to those that store the routing, neighbours side by side; and the counts
  __shared__ uint32_t s_slot[G][kRouterTopK + 1], s_c[V * L];
  __shared__ float s_exp[G][(V + 1) * L];
  uint32_t* slot = s_slot[threadIdx.x / L];
  float* exps = s_exp[threadIdx.x / L];
  for (int e = threadIdx.x; e < V * L; e += kRouterThreads) s_c[e] = 0u;
  __syncthreads();
  float next[V];
  bool next_on = true;
  if (b < a.B) {
    router_load<T, V>(raw + b * a.row_stride, e0, E, next);
    if (a.mask) next_on = a.mask[b] != 0;
  }
  for (; b < a.B; b += step) {
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = next[j];
    const bool on = next_on;
    if (b + step < a.B) {     // the next token's row is on its way under this one's work
      router_load<T, V>(raw + (b + step) * a.row_stride, e0, E, next);
      if (a.mask) next_on = a.mask[b + step] != 0;
    }
    if (!on) {
      for (int j = l; j < k; j += L) {
        a.idx[b * k + j] = -1;
        a.w[b * k + j] = 0.f;
      }
      continue;
    }
    uint32_t key[V], full[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      full[j] = order_key(v[j]);
      key[j] = (full[j] & ~0xffu) | low[j];
    }
    // The k largest by keys with 255 - the expert in their low byte, one maximum each. The
    // largest key below `best` is the largest of key - best, unsigned, plus best: those
    // below wrap round to above all others. bf16 logits' keys end before that byte; of
    // fp32 ones two that differ in it alone, neighbours among the k + 1 largest, go to the
    // exact search.
    uint32_t best = lanes_max<L>(max_of(key)), top, apart = ~0u;
    if (sizeof(T) == 4) top = lanes_max<L>(max_of(full));
    else top = best & 0x80000000u ? best & 0xffff0000u : best | 0xffffu;
    slot[0] = best;
    for (int i = 1; i < k; ++i) {
      const uint32_t lower = key_below<L>(key, best);
      apart = min(apart, best ^ lower);
      slot[i] = best = lower;
    }
    if constexpr (sizeof(T) == 4) {
      if (k < E) apart = min(apart, best ^ key_below<L>(key, best));
      if (__any(apart < 256u)) {
#pragma unroll
        for (int j = 0; j < V; ++j) full[j] = order_key(v[j]);
        for (int i = 0; i < k; ++i) {
          // the largest key left, in the lowest lane that holds it, its first
          const uint32_t mine = max_of(full);
          const uint32_t most = lanes_max<L>(mine);
          if (lanes_min<L>(mine == most ? l : L) == l) {
            bool open = true;
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (open && full[j] == most) {
                open = false;
                full[j] = 0u;
                slot[i] = low[j];
              }
          }
        }
      }
    }
    Capped c[V];
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = capped(v[j], sc.c1);
    const RouterToken<V> tok(sc, v, c, key_value(top));
    float ep[V], sp = 0.f, sz = 0.f, ss = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = e0 + j < E ? tok.d[j] : -INFINITY;
      ep[j] = __builtin_amdgcn_exp2f(d * tok.k_p);
      sz += __builtin_amdgcn_exp2f(d * tok.k_z);
      sp += ep[j];
      exps[j * L + l] = ep[j];
    }
    sp = lanes_sum<L>(sp);
    sz = lanes_sum<L>(sz);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int i = l; i < k; i += L) ss += exps[place<L, V>(255u - (slot[i] & 255u))];
    ss = lanes_sum<L>(ss);
    const float inv_sp = __builtin_amdgcn_rcpf(sp);
    const float inv_s = __builtin_amdgcn_rcpf(fmaf(ss, inv_sp, 1e-6f));
#pragma unroll
    for (int j = 0; j < V; ++j) ps[j] += ep[j] * inv_sp;
    for (int i = l; i < k; i += L) {
      const uint32_t e = 255u - (slot[i] & 255u);
      a.idx[b * k + i] = e;
      a.w[b * k + i] = exps[place<L, V>(e)] * inv_sp * inv_s;
      atomicAdd(s_c + e, 1u);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (l == 0) {
      const float lse = sc.value(key_value(top)) + __logf(sz);
      zs += lse * lse;
      ++n;
    }
  }
  // this work-group's column sums: over the wave's tokens, then over its waves
#pragma unroll
  for (int o = L; o < 64; o <<= 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) ps[j] += __shfl_xor(ps[j], o);
    zs += __shfl_xor(zs, o);
    n += __shfl_xor(n, o);
  }
  constexpr int W = kRouterThreads / 64;
  __shared__ float s_p[W][V * L], s_z[W];
  __shared__ uint32_t s_n[W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (lane < L) {
#pragma unroll
    for (int j = 0; j < V; ++j) s_p[wave][e0 + j] = ps[j];
    if (l == 0) {
      s_z[wave] = zs;
      s_n[wave] = n;
    }
  }
  __syncthreads();
  float z = 0.f;
  uint32_t N = 0u;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    z += s_z[w];
    N += s_n[w];
  }
  if (gridDim.x == 1) {       // the sums are whole
    if (wave > 0) return;
    const float inv_n = N ? 1.f / (float)N : 0.f;
    float lb = 0.f;
    for (int e = lane; e - lane < E; e += 64) {
      float p = 0.f;
      uint32_t c = 0u;
      if (e < E)
#pragma unroll
        for (int w = 0; w < W; ++w) p += s_p[w][e];
      if (e < E) c = s_c[e];
      lb += router_finish_wave(a, e, p, c, inv_n);
    }
    if (lane == 0) {
      *a.lb = (float)E * lb;
      *a.z = z * inv_n;
      *a.tokens = (float)N;
    }
    return;
  }
  // part: (blocks, E) pairs of a sum of P and a count, (blocks) pairs of z and N, then
  // k_router_finish's own words
  float2* pairs = reinterpret_cast<float2*>(a.part);
  for (int e = threadIdx.x; e < E; e += kRouterThreads) {
    float p = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) p += s_p[w][e];
    pairs[(int64_t)blockIdx.x * E + e] = make_float2(p, __uint_as_float(s_c[e]));
  }
  if (threadIdx.x == 0) {
    pairs[(int64_t)gridDim.x * E + blockIdx.x] = make_float2(z, __uint_as_float(N));
    if (blockIdx.x == 0)      // k_router_finish counts its work-groups here
      *reinterpret_cast<uint32_t*>(pairs + (int64_t)gridDim.x * (E + 1)) = 0u;
  }
}

// counts, lb, z and N from the forward's planes: a work-group to kFinishCols experts, its
// 64 groups of lanes to the planes; with more than one the last to end adds lb's parts.
__global__ __launch_bounds__(1024) void k_router_finish(RouterArgs a) {
  const int E = a.E, nb = a.blocks;
  const float2* pairs = reinterpret_cast<const float2*>(a.part);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int c = threadIdx.x & (kFinishCols - 1), e = blockIdx.x * kFinishCols + c;
  __shared__ float s_p[16][kFinishCols], s_z[16];
  __shared__ uint32_t s_c[16][kFinishCols], s_n[16];
  float p = 0.f, z = 0.f;
  uint32_t cn = 0u, n = 0u;
  for (int i = threadIdx.x; i < nb; i += 1024) {
    const float2 q = pairs[(int64_t)nb * E + i];
    z += q.x;
    n += __float_as_uint(q.y);
  }
  if (e < E)
#pragma unroll 4
    for (int i = threadIdx.x / kFinishCols; i < nb; i += 1024 / kFinishCols) {
      const float2 q = pairs[(int64_t)i * E + e];
      p += q.x;
      cn += __float_as_uint(q.y);
    }
#pragma unroll
  for (int o = 32; o >= kFinishCols; o >>= 1) {
    p += __shfl_xor(p, o);
    cn += __shfl_xor(cn, o);
  }
  z = lanes_sum<64>(z);
  n = lanes_reduce<64>(n, [](uint32_t x, uint32_t y) { return x + y; });
  if (lane < kFinishCols) {
    s_p[wave][c] = p;
    s_c[wave][c] = cn;
  }
  if (lane == 0) {
    s_z[wave] = z;
    s_n[wave] = n;
  }
  __syncthreads();
  if (wave > 0) return;
  p = z = 0.f;
  cn = n = 0u;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    p += s_p[w][c];
    cn += s_c[w][c];
    z += s_z[w];
    n += s_n[w];
  }
  const float inv_n = n ? 1.f / (float)n : 0.f;
  const float lb = router_finish_wave(a, lane < kFinishCols ? e : E, p, cn, inv_n);
  if (lane > 0) return;
  if (blockIdx.x == 0) {
    *a.z = z * inv_n;
    *a.tokens = (float)n;
  }
  if (gridDim.x == 1) {
    *a.lb = (float)E * lb;
    return;
  }
  uint32_t* ended = reinterpret_cast<uint32_t*>(a.part + 2 * (int64_t)nb * (E + 1));
  float* parts = reinterpret_cast<float*>(ended + 1);
  __hip_atomic_store(parts + blockIdx.x, lb, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (__hip_atomic_fetch_add(ended, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) + 1u != gridDim.x)
    return;
  float sum = 0.f;
  for (unsigned i = 0; i < gridDim.x; ++i)
    sum += __hip_atomic_load(parts + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  *a.lb = (float)E * sum;
}

template <class T, int L, int V>
__global__ __launch_bounds__(kRouterThreads) void k_router_bwd(RouterArgs a) {
  constexpr int G = kRouterThreads / L;
  const T* raw = static_cast<const T*>(a.raw);
  T* draw = static_cast<T*>(a.draw);
  const int E = a.E, k = a.k, l = threadIdx.x & (L - 1), e0 = V * l;
  const RouterScales sc(a);
  const float inv_tau = 1.f / (a.tau_dev ? *a.tau_dev : a.tau);
  const float N = *a.tokens, inv_n = N > 0.f ? 1.f / N : 0.f;
  const float cg = a.dlb ? *a.dlb * (float)E * inv_n * inv_n : 0.f;
  const float cz = a.dz ? *a.dz * 2.f * inv_n : 0.f;
  float g0[V];
#pragma unroll
  for (int j = 0; j < V; ++j) g0[j] = e0 + j < E ? cg * (float)a.counts[e0 + j] : 0.f;
  // a token's selected experts, handed from the lanes that read them to those that hold them
  // (0 and dw's distance from the top's; 1 and 0 for all others)
  __shared__ float2 s_sel[G][(V + 1) * L];
  float2* sel = s_sel[threadIdx.x / L];
  const float2 none = make_float2(1.f, 0.f);
#pragma unroll
  for (int j = 0; j < V; ++j) sel[j * L + l] = none;
  for (int64_t b = (int64_t)blockIdx.x * G + threadIdx.x / L; b < a.B;
       b += (int64_t)gridDim.x * G) {
    float o[V] = {};
    // a masked token's row and indices (-1) are read too: the loads wait for no other
    float v[V];
    router_load<T, V>(raw + b * a.row_stride, e0, E, v);
    int64_t e_first = -1;
    float d_first = 0.f;
    if (l < k) {
      e_first = a.idx[b * k + l];
      if (a.dw) d_first = a.dw[b * k + l];
    }
    const int64_t e_top = a.idx[b * k];
    const float d_top = a.dw ? a.dw[b * k] : 0.f;
    if (!a.mask || a.mask[b]) {
      const float g_top = e_top >= 0 && e_top < E ? cg * (float)a.counts[e_top] : 0.f;
      const bool has = e_first >= 0 && e_first < E;
      const uint32_t first = place<L, V>((uint32_t)e_first);
      if (has) sel[first] = make_float2(0.f, d_first - d_top);
      for (int i = l + L; i < k; i += L) {
        const int64_t e = a.idx[b * k + i];
        if (e >= 0 && e < E)
          sel[place<L, V>((uint32_t)e)] = make_float2(0.f, (a.dw ? a.dw[b * k + i] : 0.f) - d_top);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      float off[V], dw[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 s = sel[j * L + l];
        off[j] = s.x;
        dw[j] = s.y;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (has) sel[first] = none;
      for (int i = l + L; i < k; i += L) {
        const int64_t e = a.idx[b * k + i];
        if (e >= 0 && e < E) sel[place<L, V>((uint32_t)e)] = none;
      }
      float top = v[0];         // NaN if one of them is
#pragma unroll
      for (int j = 1; j < V; ++j) top = __builtin_elementwise_maximum(top, v[j]);
      top = __uint_as_float(lanes_reduce<L>(__float_as_uint(top), [](uint32_t x, uint32_t y) {
        return __float_as_uint(
            __builtin_elementwise_maximum(__uint_as_float(x), __uint_as_float(y)));
      }));
      Capped t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] = capped(v[j], sc.c1);
      const RouterToken<V> tok(sc, v, t, top);
      float ep[V], ez[V], ss = 0.f, sz = 0.f, su = 0.f, sd = 0.f, sg = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = e0 + j < E ? tok.d[j] : -INFINITY;
        ep[j] = __builtin_amdgcn_exp2f(d * tok.k_p);
        ez[j] = __builtin_amdgcn_exp2f(d * tok.k_z);
        sz += ez[j];
        ss += off[j] == 0.f ? ep[j] : 0.f;
        su = fmaf(ep[j], off[j], su);
        sd = fmaf(ep[j], dw[j], sd);
        sg = fmaf(ep[j], g0[j] - g_top, sg);
      }
      // selected and not, each by itself: either may be a hundredth of the other
      ss = lanes_sum<L>(ss);
      sz = lanes_sum<L>(sz);
      su = lanes_sum<L>(su);
      sd = lanes_sum<L>(sd);
      sg = lanes_sum<L>(sg);
      const float inv_sp = __builtin_amdgcn_rcpf(ss + su);
      const float inv_s = __builtin_amdgcn_rcpf(fmaf(ss, inv_sp, 1e-6f));
      const float D = sd * inv_sp * inv_s;                         // sum_i w_i (dw_i - dw_0)
      const float pg = sg * inv_sp;                                // sum_e P_e (G_e - G_0)
      const float a_on = fmaf(1e-6f, fmaf(d_top, su * inv_sp * inv_s, -D), -D) * inv_s - pg;
      const float a_off = -1e-6f * fmaf(d_top, ss * inv_sp * inv_s, D) * inv_s - pg;
      const float c_p = 4.f * inv_sp * inv_tau;
      const float c_z = 4.f * cz * (sc.value(top) + __logf(sz)) * __builtin_amdgcn_rcpf(sz);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = fmaf(dw[j], inv_s, off[j] == 0.f ? a_on : a_off) + (g0[j] - g_top);
        o[j] = fmaf(c_z, ez[j], ep[j] * c_p * g) * (t[j].Q * t[j].R * t[j].R);
      }
    }
    T* row = draw + b * E;
    if (e0 + V <= E) {
      constexpr int W = V * (int)sizeof(T) / 4;
      typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
      vec q;
#pragma unroll
      for (int j = 0; j < W; ++j)
        if constexpr (sizeof(T) == 4) q[j] = __float_as_uint(o[j]);
        else q[j] = pack_bf16x2(o[2 * j], o[2 * j + 1]);
      *reinterpret_cast<vec*>(row + e0) = q;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j < E) store_from_f32(row + e0 + j, o[j]);
    }
  }
}

}  // namespace dev
}  // namespace tmoe
