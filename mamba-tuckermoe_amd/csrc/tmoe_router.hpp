// The training layer's router with its losses (sft_cot_bundle/scripts/model.py:318-332) and
// their gradient. For a token's logits raw (E), c = cap, tau = temperature:
//   a = c tanh(raw / c);  P = softmax(a / tau);  idx = the k largest raw, the lowest index
//   on ties (the cap and the temperature are monotone);  s = sum_j P[idx_j] + 1e-6;
//   w_j = P[idx_j] / s
//   lb = E sum_e (n_e / N) (sum_b P_be / N),  z = sum_b lse(a_b)^2 / N
// over the N tokens that no mask leaves out, n_e of which select e. A masked token has
// idx -1 (which selects nothing in the contraction), w 0 and no gradient.
//   g_e  = dlb E n_e / N^2 + [e = idx_j] (dw_j - sum_i dw_i w_i) / s
//   draw = (1 - tanh^2) ((P_e (g_e - sum_f P_f g_f)) / tau + dz 2 lse softmax(a)_e / N)
// where both differences are taken from the likeliest expert's (dw_0, g_0): with its
// P near 1 the sums are next to those, and the differences what is left of two equals.
//
// With Q = exp(-2 raw / c) and R = 1 / (1 + Q), tanh = 1 - 2 Q R, 1 - tanh^2 = 4 Q R^2 and
//   a_e - a_m = 2 c R_m R_e (Q_m - Q_e)
// for the largest logit m: the exponents of both softmaxes without the cancellation of two
// capped logits near the cap. raw / c is cut at +-20, past which tanh is +-1 in fp32.
//
// A token's logits lie in L lanes, V to a lane (L a power of two, V L >= E; V = 8, or 4 where
// that is all of them): what a token needs of them is exchanged by lane permutations. Eight
// to a lane rather than four: the exchanges, and not the exponentials, are most of the
// instructions (E = 64, B = 131072: forward 29 against 32 us). Bound by instructions: that
// size's forward takes 29.8 us (1.3 TB/s of what it moves), its backward 25.0 (3.1 TB/s);
// B = 16384, E = 8 5.8 and 5.5 us. The column sums over the tokens (n_e,
// sum_b P_be) stay in registers over a work-group's tokens, then in a plane of `part`, and
// k_router_finish adds the planes in a fixed order: the losses do not depend on which
// work-group ends first.
#pragma once

#include "tmoe_elem.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace dev {

constexpr int kRouterThreads = 256;
constexpr int kFinishCols = 16;       // experts of a work-group of k_router_finish

// raw[e0 .. e0 + V - 1] of a row of E logits (0 past its end), at any alignment
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
    for (int j = 0; j < V; ++j) v[j] = e0 + j < E ? load_as_f32(row + e0 + j) : 0.f;
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
  f += 0.f;
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct Capped {
  float Q, R;
};
// c1 = -2 log2(e) / cap; a NaN stays one
__device__ __forceinline__ Capped capped(float raw, float c1) {
  constexpr float kCut = 20.f * 2.8853900817779268f;
  float u = raw * c1;
  u = u > kCut ? kCut : u < -kCut ? -kCut : u;
  const float Q = __builtin_amdgcn_exp2f(u);
  return {Q, __builtin_amdgcn_rcpf(1.f + Q)};
}

// cap tanh(raw / cap) to the last places, for the logsumexp: once a token
__device__ __forceinline__ float capped_value(float raw, float c1, float cap) {
  const float q = __builtin_amdgcn_exp2f(-fabsf(raw * c1)), d = 1.f + q;
  const float r = __builtin_amdgcn_rcpf(d);
  return copysignf(cap * ((1.f - q) * fmaf(r, fmaf(-d, r, 1.f), r)), raw);
}

struct RouterScales {
  float c1, k_z, k_p;   // exponents in base 2 of R_m R_e (Q_m - Q_e): of both softmaxes
  __device__ RouterScales(const RouterArgs& a) {
    const float tau = a.tau_dev ? *a.tau_dev : a.tau;
    c1 = -2.8853900817779268f / a.cap;
    k_z = 2.8853900817779268f * a.cap;
    k_p = k_z / tau;
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
  uint32_t cn[V] = {}, n = 0u;
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
    uint32_t key[V], full[V], top = 0u, last = 0u;
    int pos[V];
    bool tied = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      full[j] = e0 + j < E ? order_key(v[j]) : 0u;
      key[j] = full[j] ? (full[j] & ~0xffu) | (255u - (uint32_t)(e0 + j)) : 0u;
      pos[j] = -1;
    }
    // The k largest by keys with the expert in their low byte: each is one lane's, and one
    // maximum finds it. bf16 logits' keys end before that byte; of fp32 ones two that
    // differ in it alone, neighbours among the k + 1 largest, go to the exact search.
    const int rounds = sizeof(T) == 4 && k < E ? k + 1 : k;
    for (int i = 0; i < rounds; ++i) {
      const uint32_t best = lanes_max<L>(max_of(key));
      if (sizeof(T) == 4) tied = tied || (best ^ last) < 256u;
      else if (i == 0) top = best & 0x80000000u ? best & 0xffff0000u : best | 0xffffu;
      last = best;
      if (i < k) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool it = key[j] == best;
          pos[j] = it ? i : pos[j];
          key[j] = it ? 0u : key[j];
        }
      }
    }
    if constexpr (sizeof(T) == 4) {
      top = lanes_max<L>(max_of(full));
      if (__any(tied)) {
#pragma unroll
        for (int j = 0; j < V; ++j) pos[j] = -1;
        for (int i = 0; i < k; ++i) {
          // the largest key left, in the lowest lane that holds it, its first
          const uint32_t mine = max_of(full);
          const uint32_t best = lanes_max<L>(mine);
          if (lanes_min<L>(mine == best ? l : L) == l) {
            bool open = true;
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (open && full[j] == best) {
                open = false;
                pos[j] = i;
                full[j] = 0u;
              }
          }
        }
      }
    }
    const Capped m = capped(key_value(top), sc.c1);
    float ep[V], sp = 0.f, sz = 0.f, ss = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const Capped c = capped(v[j], sc.c1);
      const float d = (m.Q - c.Q) * (m.R * c.R);
      const bool in = e0 + j < E;
      ep[j] = in ? __builtin_amdgcn_exp2f(d * sc.k_p) : 0.f;
      sz += in ? __builtin_amdgcn_exp2f(d * sc.k_z) : 0.f;
      sp += ep[j];
      ss += pos[j] >= 0 ? ep[j] : 0.f;
    }
    sp = lanes_sum<L>(sp);
    sz = lanes_sum<L>(sz);
    ss = lanes_sum<L>(ss);
    const float inv_sp = __builtin_amdgcn_rcpf(sp);
    const float inv_s = __builtin_amdgcn_rcpf(fmaf(ss, inv_sp, 1e-6f));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float P = ep[j] * inv_sp;
      ps[j] += P;
      if (pos[j] >= 0) {
        ++cn[j];
        a.idx[b * k + pos[j]] = e0 + j;
        a.w[b * k + pos[j]] = P * inv_s;
      }
    }
    if (l == 0) {
      const float lse = capped_value(key_value(top), sc.c1, a.cap) + __logf(sz);
      zs += lse * lse;
      ++n;
    }
  }
  // this work-group's column sums: over the wave's tokens, then over its waves
#pragma unroll
  for (int o = L; o < 64; o <<= 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      ps[j] += __shfl_xor(ps[j], o);
      cn[j] += __shfl_xor(cn[j], o);
    }
    zs += __shfl_xor(zs, o);
    n += __shfl_xor(n, o);
  }
  constexpr int W = kRouterThreads / 64;
  __shared__ float s_p[W][V * L], s_z[W];
  __shared__ uint32_t s_c[W][V * L], s_n[W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (lane < L) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s_p[wave][e0 + j] = ps[j];
      s_c[wave][e0 + j] = cn[j];
    }
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
        for (int w = 0; w < W; ++w) {
          p += s_p[w][e];
          c += s_c[w][e];
        }
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
    uint32_t c = 0u;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      p += s_p[w][e];
      c += s_c[w][e];
    }
    pairs[(int64_t)blockIdx.x * E + e] = make_float2(p, __uint_as_float(c));
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
  __shared__ float2 s_sel[G][V * L];
  float2* sel = s_sel[threadIdx.x / L];
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
#pragma unroll
      for (int j = 0; j < V; ++j) sel[e0 + j] = make_float2(0.f, 0.f);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const float g_top = e_top >= 0 && e_top < E ? cg * (float)a.counts[e_top] : 0.f;
      if (e_first >= 0 && e_first < E) sel[e_first] = make_float2(1.f, d_first - d_top);
      for (int i = l + L; i < k; i += L) {
        const int64_t e = a.idx[b * k + i];
        if (e >= 0 && e < E) sel[e] = make_float2(1.f, (a.dw ? a.dw[b * k + i] : 0.f) - d_top);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j < E) top = fmaxf(top, v[j]);
      top = __uint_as_float(lanes_reduce<L>(__float_as_uint(top), [](uint32_t x, uint32_t y) {
        return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
      }));
      const Capped m = capped(top, sc.c1);
      Capped t[V];
      float ep[V], ez[V], dw[V], on[V], sp = 0.f, sz = 0.f, su = 0.f, sd = 0.f, sg = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 s = sel[e0 + j];
        on[j] = s.x;
        dw[j] = s.y;
        t[j] = capped(v[j], sc.c1);
        const float d = (m.Q - t[j].Q) * (m.R * t[j].R);
        const bool in = e0 + j < E;
        ep[j] = in ? __builtin_amdgcn_exp2f(d * sc.k_p) : 0.f;
        ez[j] = in ? __builtin_amdgcn_exp2f(d * sc.k_z) : 0.f;
        sp += ep[j];
        sz += ez[j];
        su += on[j] != 0.f ? 0.f : ep[j];
        sd += on[j] != 0.f ? ep[j] * dw[j] : 0.f;
        sg += ep[j] * (g0[j] - g_top);
      }
      sp = lanes_sum<L>(sp);
      sz = lanes_sum<L>(sz);
      su = lanes_sum<L>(su);
      sd = lanes_sum<L>(sd);
      sg = lanes_sum<L>(sg);
      const float inv_sp = __builtin_amdgcn_rcpf(sp);
      const float inv_s = __builtin_amdgcn_rcpf((sp - su) * inv_sp + 1e-6f);
      // the top's own part of g beside the balance loss's: dw_0 - sum_i dw_i w_i, over s
      const float gs = (d_top * 1e-6f * inv_s - sd * inv_sp * inv_s) * inv_s;
      const float pg = (sg + sd * inv_s - su * gs) * inv_sp;       // sum_e P_e (g_e - g_0)
      const float zc = cz * (capped_value(top, sc.c1, a.cap) + __logf(sz)) * __builtin_amdgcn_rcpf(sz);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = g0[j] - g_top + (on[j] != 0.f ? dw[j] * inv_s : -gs);
        o[j] = (ep[j] * inv_sp * (g - pg) * inv_tau + zc * ez[j]) * (4.f * t[j].Q * t[j].R * t[j].R);
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
