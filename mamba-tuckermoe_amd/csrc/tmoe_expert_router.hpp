// Routing to experts by softmax or sigmoid scores, with a bias for balance, groups of experts
// and renormalised weights, and the gradient of the logits. For a token's logits raw (E):
//   s = softmax(raw) or 1 / (1 + exp(-raw));  b = s + bias
//   a group's worth = its two largest b added;  the top_groups worthiest groups are open
//   idx = the k largest b of the open groups;  w_j = scale s_j / (sum_i s_i + 1e-20), or scale s_j
// all of them compared as in float64, the lowest index first on ties. With neither bias nor
// groups b has the logits' own order, and those are compared. A masked token has idx -1, w 0
// and no gradient. Renormalised, with u = w / scale, r = 1 - sum u = 1e-20 / (sum s + 1e-20) in closed form
// and D = sum_i u_i (dw_i - dw_0), differences to dw_0 since one weight may be next to all:
//   t_j = dw_j - sum_i dw_i u_i = (dw_j - dw_0) - D + dw_0 r;  sum_j u_j t_j = r (D + (1 - r) dw_0)
//   sigmoid  draw_j = w_j t_j (1 - s_j) where selected, else 0
//   softmax  draw_e = w_e t_e (where selected) - scale s_e sum_j u_j t_j
// A softmax's r is next to nothing unless a bias selects scores of 1e-14 and less in all. There the row's
// logits are read for it; elsewhere sum w tells that it is below 2^-20, it is left out (16 roundings of
// what it stands beside), and the logits are not needed. Not renormalised t_j = dw_j, and
//   sigmoid  draw_j = w_j t_j (1 - s_j);  softmax  draw_e = scale s_e (t_e - sum_j s_j t_j)
//
// Ranks. A token's experts lie in L lanes, eight to a lane. Scores become whole numbers of 24
// bits over the range that the biases leave them ([-bm, 1 + bm]; softmax before its division,
// which is the same for all), with 255 - e below: one 32-bit maximum finds a score and its
// expert. A float's own bits in that place would leave 16 of them, and one token in a hundred
// with two scores that cannot be told apart. Where two numbers that the routing tells apart are
// closer than their error allows, the wave's tokens are ranked again in float64 (route_exact): one token in
// 600 of E = 256 with biases, one in 4000 of E = 64 in float32, which are 0.2 to 0.35% of the waves. Equal
// scores are such a pair as well: of bf16 softmax logits in groups without a bias (E = 64, k = 6), where
// equal logits are common, 9% of the tokens and half of the waves are ranked again.
#pragma once

#include "tmoe_router_keys.hpp"
#include "tmoe_step.h"

namespace tmoe {
namespace dev {

constexpr int kErThreads = 256;
constexpr int kErV = 8;                 // experts of a lane
constexpr int kErSoftmax = 0;           // ExpertRouterArgs::score
// The scores' numbers are off by under 8 of their units of 2^-24 of the range: 1 of the
// exponential, 1 of the quotient or 4 of the sum (a relative one, over 256 terms in a tree), 1
// of the addition, 1 cut off. Two of them: 16; a group's worth is two of those.
constexpr uint32_t kErNear = 20, kErNearGroups = 40;

// exp(x) to the last place or two at any x: hardware's exp2 of the rounded product, and the
// product's rounding put back
__device__ __forceinline__ float exp_close(float x) {
  const float h = x * 1.44269504f;
  const float lo = fmaf(x, 1.44269504f, -h) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(h);
  const float c = e * (lo * 0.69314718f);
  return e + (fabsf(h) < 150.f ? c : 0.f);   // past it e is 0 or inf, and lo may be none
}
// 1 / (1 + exp(-x))
__device__ __forceinline__ float sigmoid_close(float x) {
  const float d = 1.f + exp_close(-x), r = __builtin_amdgcn_rcpf(d);
  return d < 1e30f ? fmaf(r, fmaf(-d, r, 1.f), r) : exp_close(x);   // NaN: exp(NaN)
}

__device__ __forceinline__ uint64_t order_key64(double f) {
  const int64_t b = __double_as_longlong(f + 0.0);
  return f != f ? ~0ull : (uint64_t)(b ^ (b >> 63 | (int64_t)0x8000000000000000ull));
}
__device__ __forceinline__ double key_value64(uint64_t k) {
  return k == ~0ull ? (double)NAN
                    : __longlong_as_double((int64_t)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}
// the largest of L lanes' words, by halves
template <int L>
__device__ __forceinline__ uint64_t lanes_max64(uint64_t v) {
  const uint32_t hi = lanes_max<L>((uint32_t)(v >> 32));
  return (uint64_t)hi << 32 | lanes_max<L>((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}

// the largest of L lanes' floats, NaN if one of them is
template <int L>
__device__ __forceinline__ float lanes_top(float v) {
  return __uint_as_float(lanes_reduce<L>(__float_as_uint(v), [](uint32_t x, uint32_t y) {
    return __float_as_uint(__builtin_elementwise_maximum(__uint_as_float(x), __uint_as_float(y)));
  }));
}
__device__ __forceinline__ void er_order() {   // LDS of one wave: what was written is read after it
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A token's routing in float64: the ranks in slot[0 .. k - 1] (255 - the expert). `d` is the
// token's own V L doubles of shared memory, and its values pass through them one by one: in
// registers eight exponentials side by side took as many as the rest of the kernel together.
template <int L>
__device__ __forceinline__ void route_exact(const ExpertRouterArgs& a, const float (&v)[kErV], int l,
                                            bool by_logit, const float* bias, double* d, uint32_t* slot) {
  constexpr int V = kErV;
  const int E = a.E, e0 = V * l, mine = E - e0 < V ? E - e0 : V;    // (no expert: below 1)
  uint64_t* keys = reinterpret_cast<uint64_t*>(d);
  double unit = 1.0;
  float m = 0.f;
  if (!by_logit && a.score == kErSoftmax) {
    m = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = __builtin_elementwise_maximum(m, v[j]);
    m = lanes_top<L>(m);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) d[e0 + j] = v[j];
  if (!by_logit) {
    const bool softmax = a.score == kErSoftmax;
    double sum = 0.0;
#pragma unroll 1
    for (int j = 0; j < mine; ++j) {
      const double x = exp(softmax ? d[e0 + j] - (double)m : -d[e0 + j]);
      sum += x;
      d[e0 + j] = softmax ? x : 1.0 / (1.0 + x);
    }
    if (softmax) unit = lanes_sum64<L>(sum);
  }
#pragma unroll 1
  for (int j = 0; j < V; ++j) {
    const bool is = j < mine;
    const double x = d[e0 + j] / unit + (double)bias[e0 + j];
    keys[e0 + j] = is ? order_key64(x) : 0ull;
  }
  er_order();
  if (a.groups > 1 && a.top_groups < a.groups) {
    // group l + L i is this lane's i-th
    const int per = E / a.groups;
    uint64_t worth[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      worth[i] = 0ull;
      const int g = l + L * i;
      if (g < a.groups) {
        uint64_t top = 0ull, second = 0ull;
#pragma unroll 4
        for (int c = 0; c < per; ++c) {
          const uint64_t x = keys[g * per + c];
          second = x > top ? top : x > second ? x : second;
          top = x > top ? x : top;
        }
        worth[i] = per > 1 ? order_key64(key_value64(top) + key_value64(second)) : top;
      }
    }
    er_order();
    uint32_t kept = 0u;        // this lane's groups that are
    for (int r = 0; r < a.top_groups; ++r) {
      uint64_t best = 0ull;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (!(kept >> i & 1u) && worth[i] > best) best = worth[i];
      const uint64_t most = lanes_max64<L>(best);
      uint32_t g = 256u;
#pragma unroll
      for (int i = V - 1; i >= 0; --i)
        if (!(kept >> i & 1u) && l + L * i < a.groups && worth[i] == most) g = l + L * i;
      g = lanes_min<L>(g);
      if (g % L == (uint32_t)l) kept |= 1u << (g / L);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = l + L * i;
      if (g < a.groups && !(kept >> i & 1u))
        for (int c = 0; c < per; ++c) keys[g * per + c] = 0ull;
    }
    er_order();
  }
  uint64_t own[V];
#pragma unroll
  for (int j = 0; j < V; ++j) own[j] = keys[e0 + j];
  for (int i = 0; i < a.k; ++i) {
    uint64_t best = own[0];
#pragma unroll
    for (int j = 1; j < V; ++j) best = own[j] > best ? own[j] : best;
    const uint64_t most = lanes_max64<L>(best);
    uint32_t at = 255u;
#pragma unroll
    for (int j = V - 1; j >= 0; --j)
      if (own[j] == most && most) at = e0 + j;
    const uint32_t e = lanes_min<L>(at);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e == (uint32_t)(e0 + j)) own[j] = 0ull;
    slot[i] = 255u - e;
  }
}

// One pass over the logits, a token to L lanes: nothing but idx, w and the counts is written, and the
// next token's row is loaded under this one's work. Bound by the chain of a token's maxima, not by
// bytes: of (B, E) = (4096, 256), k = 8 in 4 of 8 groups, 8.8 us, and (16384, 64), k = 6 in 3 of 8, 7.0 us,
// where no token is ranked again, 16.9 and 13.2 us with random logits, of which 0.35% of the first's
// waves are and half of the second's, in bf16 (24.1 and 19.1 with the biases read from memory there and
// maxima of 64 bits by shuffles);
// (131072, 64), k = 6, a third of it masked, 24.5 us, 1.1 TB/s.
template <class T, int L>
__global__ __launch_bounds__(kErThreads) void k_expert_router_fwd(ExpertRouterArgs a) {
  constexpr int V = kErV, G = kErThreads / L;
  const T* raw = static_cast<const T*>(a.raw);
  const int E = a.E, k = a.k, l = threadIdx.x & (L - 1), e0 = V * l;
  const bool by_logit = !a.bias && a.groups == 1;
  const bool grouped = a.groups > 1 && a.top_groups < a.groups;
  const int per = E / a.groups;
  __shared__ uint32_t s_slot[G][kRouterTopK + 1], s_c[V * L];
  __shared__ float s_bias[V * L];
  __shared__ double s_wide[G][V * L];            // keys, worths and scores of a token
  uint32_t* slot = s_slot[threadIdx.x / L];
  double* wide = s_wide[threadIdx.x / L];
  uint32_t* words = reinterpret_cast<uint32_t*>(wide);          // V L keys or scores
  uint32_t* worths = words + V * L;
  for (int e = threadIdx.x; e < V * L; e += kErThreads) {
    s_c[e] = 0u;
    s_bias[e] = a.bias && e < E ? a.bias[e] : 0.f;
  }
  __syncthreads();
  float bias[V], bm = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    bias[j] = s_bias[e0 + j];
    bm = __builtin_elementwise_maximum(bm, fabsf(bias[j]));
  }
  bm = lanes_top<L>(bm);
  const bool wild = !(bm < 1e30f);               // biases that leave no range
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t b = (int64_t)blockIdx.x * G + threadIdx.x / L;
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
    // scores: s times `unit`
    float s[V], unit = 1.f;
    if (a.score == kErSoftmax) {
      float m = v[0], sum = 0.f;   // NaN if one of them is
#pragma unroll
      for (int j = 1; j < V; ++j) m = __builtin_elementwise_maximum(m, v[j]);
      m = lanes_top<L>(m);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[j] = e0 + j < E ? exp_close(v[j] - m) : 0.f;
        sum += s[j];
      }
      unit = lanes_sum<L>(sum);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = sigmoid_close(v[j]);
    }
    uint32_t key[V];
    bool near = wild;
    uint32_t least = kErNear << 8;               // keys closer than that are
    if (by_logit) {
      // bf16 logits' keys end before the expert's byte: equal ones are equal
      least = sizeof(T) == 4 ? 256u : 0u;
#pragma unroll
      for (int j = 0; j < V; ++j)
        key[j] = e0 + j < E ? (order_key(v[j]) & ~0xffu) | (255u - (uint32_t)(e0 + j)) : 0u;
    } else {
      const float lo = bm * unit, scale = 16777215.f / fmaf(2.f, lo, 1.f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float r = (fmaf(bias[j], unit, s[j]) + lo) * scale;
        near |= e0 + j < E && !(r < 16777216.f);       // NaN, or a logit of +inf
        const uint32_t q = min((uint32_t)fmaxf(r, 0.f), 0xffffffu);
        key[j] = e0 + j < E ? q << 8 | (255u - (uint32_t)(e0 + j)) : 0u;
      }
    }
    if (grouped) {
      er_order();              // the last token's reads of `words` are done
#pragma unroll
      for (int j = 0; j < V; ++j) words[e0 + j] = key[j] >> 8;
      er_order();
      uint32_t worth[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        worth[i] = 0u;
        const int g = l + L * i;
        if (g < a.groups) {
          uint32_t top = 0u, second = 0u;
#pragma unroll 2
          for (int c = 0; c < per; ++c) {
            const uint32_t x = words[g * per + c];
            second = max(second, min(top, x));
            top = max(top, x);
          }
          // 25 bits and 6 or 7 of the group, of which the lowest is the largest
          worth[i] = a.groups <= 64 ? (top + second) << 6 | (63u - (uint32_t)g) : 0u;
          worths[g] = worth[i];
        }
      }
      uint32_t t = lanes_max<L>(max_of(worth));
      for (int r = 1; r < a.top_groups; ++r) t = key_below<L>(worth, t);
      near |= a.groups > 64 || t - key_below<L>(worth, t) < kErNearGroups << 6;
      er_order();
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j < E && worths[(uint32_t)(e0 + j) / (uint32_t)per] < t) key[j] = 0u;
    }
    uint32_t best = lanes_max<L>(max_of(key)), apart = ~0u;
    slot[0] = best;
    for (int i = 1; i < k; ++i) {
      const uint32_t lower = key_below<L>(key, best);
      apart = min(apart, best - lower);
      slot[i] = best = lower;
    }
    if (k < E) apart = min(apart, best - key_below<L>(key, best));
    if (__any(near || apart < least)) {
      er_order();
      route_exact<L>(a, v, l, by_logit, s_bias, wide, slot);
    }
    er_order();
#pragma unroll
    for (int j = 0; j < V; ++j) words[e0 + j] = __float_as_uint(s[j]);
    er_order();
    const float inv_u = a.score == kErSoftmax ? 1.f / unit : 1.f;
    float total = 0.f;
    for (int i = l; i < k; i += L) total += __uint_as_float(words[255u - (slot[i] & 255u)]);
    total = lanes_sum<L>(total) * inv_u;
    const float f = a.renormalize ? a.scale / (total + 1e-20f) : a.scale;
    for (int i = l; i < k; i += L) {
      const uint32_t e = 255u - (slot[i] & 255u);
      a.idx[b * k + i] = e;
      a.w[b * k + i] = __uint_as_float(words[e]) * inv_u * f;
      atomicAdd(s_c + e, 1u);
    }
    er_order();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kErThreads) {
    if (gridDim.x == 1) a.counts[e] = s_c[e];
    else a.part[(int64_t)blockIdx.x * E + e] = s_c[e];
  }
}

// counts from the forward's planes, in place of atomics on counts that a launch would have to clear:
// 16 experts a work-group; 4 us, a launch's
__global__ __launch_bounds__(1024) void k_expert_router_counts(ExpertRouterArgs a) {
  __shared__ uint32_t s[64][16];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
  uint32_t n = 0u;
  if (e < a.E)
#pragma unroll 4
    for (int i = r; i < a.blocks; i += 64) n += a.part[(int64_t)i * a.E + e];
  s[r][c] = n;
  __syncthreads();
  if (threadIdx.x >= 16 || e >= a.E) return;
  n = 0u;
#pragma unroll
  for (int i = 0; i < 64; ++i) n += s[i][c];
  a.counts[e] = n;
}

// The gradient of a token from its k selected experts alone (but for a softmax that is not
// renormalised or whose r counts, where every expert has one): the row is put together in LDS and
// stored whole.
// Bound by those bytes where there are many tokens: (131072, 64) in float32 17 us, 2.3 TB/s with what it
// reads; (4096, 256) 4.7 us.
template <class T, int L>
__global__ __launch_bounds__(kErThreads) void k_expert_router_bwd(ExpertRouterArgs a) {
  constexpr int V = kErV, G = kErThreads / L;
  const T* raw = static_cast<const T*>(a.raw);
  T* draw = static_cast<T*>(a.draw);
  const int E = a.E, k = a.k, l = threadIdx.x & (L - 1), e0 = V * l;
  const bool softmax = a.score == kErSoftmax, dense = softmax && !a.renormalize;
  const float inv_c = 1.f / a.scale;
  __shared__ float s_sel[G][V * L];              // a token's gradients where selected, else 0
  float* sel = s_sel[threadIdx.x / L];
#pragma unroll
  for (int j = 0; j < V; ++j) sel[e0 + j] = 0.f;
  er_order();
  for (int64_t b = (int64_t)blockIdx.x * G + threadIdx.x / L; b < a.B; b += (int64_t)gridDim.x * G) {
    float o[V] = {};
    if (!a.mask || a.mask[b]) {
      const T* row = raw + b * a.row_stride;
      // the k selected, over the lanes; a lane's are in pieces of L
      const float top = a.dw[b * k];
      float D = 0.f, S = 0.f;
      for (int i = l; i < k; i += L) {
        const int64_t e = a.idx[b * k + i];
        const float w = a.w[b * k + i];
        D = fmaf(w * inv_c, a.renormalize ? a.dw[b * k + i] - top : a.dw[b * k + i], D);
        if (softmax) S = fmaf(w, inv_c, S);
        else if (e >= 0 && e < E) S += sigmoid_close(load_as_f32(row + e));
      }
      D = lanes_sum<L>(D);
      S = lanes_sum<L>(S);
      const bool small = softmax && a.renormalize && !(S >= 1.f - 0x1p-20f);
      float v[V], m = 0.f, unit = 1.f, f = 0.f;  // of a row whose every expert has a gradient
      if (dense || small) {
        float sum = 0.f;
        router_load<T, V>(row, e0, E, v);
        m = v[0];
#pragma unroll
        for (int j = 1; j < V; ++j) m = __builtin_elementwise_maximum(m, v[j]);
        m = lanes_top<L>(m);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[j] = e0 + j < E ? exp_close(v[j] - m) : 0.f;
          sum += v[j];
        }
        unit = lanes_sum<L>(sum);
        f = a.scale / unit;
      }
      if (small) {
        S = 0.f;
        for (int i = l; i < k; i += L) {
          const int64_t e = a.idx[b * k + i];
          if (e >= 0 && e < E) S += exp_close(load_as_f32(row + e) - m);
        }
        S = lanes_sum<L>(S) / unit;
      }
      // r, what 1e-20 leaves of one, and its part of t
      const float r = softmax && !small ? 0.f : 1e-20f / (S + 1e-20f), rest = top * r;
      for (int i = l; i < k; i += L) {
        const int64_t e = a.idx[b * k + i];
        if (e < 0 || e >= E) continue;
        const float w = a.w[b * k + i], g = a.dw[b * k + i];
        float t = a.renormalize ? ((g - top) - D) + rest : g;
        if (!softmax) t *= sigmoid_close(-load_as_f32(row + e));
        sel[e] = dense ? g : w * t;
      }
      er_order();
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = sel[e0 + j];
      er_order();
#pragma unroll
      for (int j = 0; j < V; ++j) sel[e0 + j] = 0.f;
      if (dense) {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = v[j] * f * (o[j] - D);
      } else if (small) {
        const float all = r * fmaf(S / (S + 1e-20f), top, D);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = fmaf(-v[j] * f, all, o[j]);
      }
      er_order();
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
