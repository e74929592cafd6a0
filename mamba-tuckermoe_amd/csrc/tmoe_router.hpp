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
//
// A token's logits lie in L lanes, four to a lane (L a power of two, 4 L >= E): everything a
// token needs is exchanged between those lanes. The column sums over the tokens (n_e,
// sum_b P_be) stay in registers over a work-group's tokens, then in a plane of `part`, and
// k_router_finish adds the planes in a fixed order: the losses do not depend on which
// work-group ends first.
#pragma once

#include "tmoe_elem.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace dev {

constexpr int kRouterThreads = 256;

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// raw[e0 .. e0 + 3] of a row of E logits (0 past its end)
template <class T>
__device__ __forceinline__ void router_load(const T* row, int e0, int E, bool vec, float v[4]) {
  if (vec && e0 + 4 <= E) {
    if constexpr (sizeof(T) == 4) {
      const float4 q = *reinterpret_cast<const float4*>(row + e0);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const uint2 q = *reinterpret_cast<const uint2*>(row + e0);
      v[0] = bf16_bits_to_f32(q.x & 0xffffu); v[1] = bf16_bits_to_f32(q.x >> 16);
      v[2] = bf16_bits_to_f32(q.y & 0xffffu); v[3] = bf16_bits_to_f32(q.y >> 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = e0 + j < E ? load_as_f32(row + e0 + j) : 0.f;
  }
}

// An unsigned key in the order of the floats: NaN above +inf, -0 equal to 0, never 0.
__device__ __forceinline__ uint32_t order_key(float f) {
  f += 0.f;
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Capped {
  float t, sech2;   // tanh(u) and 1 - tanh^2(u) without the cancellation near +-1
};
__device__ __forceinline__ Capped capped(float u) {
  const float q = __expf(-2.f * fabsf(u)), r = 1.f / (1.f + q);
  return {copysignf((1.f - q) * r, u), 4.f * q * r * r};
}

template <class T, int L>
__global__ __launch_bounds__(kRouterThreads) void k_router_fwd(RouterArgs a) {
  constexpr int G = kRouterThreads / L;
  const T* raw = static_cast<const T*>(a.raw);
  const int E = a.E, k = a.k, l = threadIdx.x & (L - 1), e0 = 4 * l;
  const float cap = a.cap, inv_cap = 1.f / cap;
  const float inv_tau = 1.f / (a.tau_dev ? *a.tau_dev : a.tau);
  const bool vec = (reinterpret_cast<uintptr_t>(raw) & (4 * sizeof(T) - 1)) == 0 &&
                   (a.row_stride & 3) == 0;
  float ps[4] = {0.f, 0.f, 0.f, 0.f}, zs = 0.f;
  uint32_t cn[4] = {0u, 0u, 0u, 0u}, n = 0u;
  for (int64_t b = (int64_t)blockIdx.x * G + threadIdx.x / L; b < a.B;
       b += (int64_t)gridDim.x * G) {
    if (a.mask && !a.mask[b]) {
      for (int j = l; j < k; j += L) {
        a.idx[b * k + j] = -1;
        a.w[b * k + j] = 0.f;
      }
      continue;
    }
    float v[4];
    router_load(raw + b * a.row_stride, e0, E, vec, v);
    uint32_t key[4];
    int pos[4] = {-1, -1, -1, -1};
#pragma unroll
    for (int j = 0; j < 4; ++j) key[j] = e0 + j < E ? order_key(v[j]) : 0u;
    float top = 0.f;
    for (int i = 0; i < k; ++i) {
      uint64_t best = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t c = (uint64_t)key[j] << 32 | (uint32_t)(kRouterMaxE - (e0 + j));
        best = c > best ? c : best;
      }
#pragma unroll
      for (int o = L / 2; o >= 1; o >>= 1) {
        const uint64_t c = (uint64_t)__shfl_xor((uint32_t)(best >> 32), o) << 32 |
                           __shfl_xor((uint32_t)best, o);
        best = c > best ? c : best;
      }
      const int e = (int)kRouterMaxE - (int)(uint32_t)best;
      if (i == 0) {
        const uint32_t kb = (uint32_t)(best >> 32);
        top = kb == 0xffffffffu ? __uint_as_float(0x7fc00000u)
                                : __uint_as_float(kb & 0x80000000u ? kb & 0x7fffffffu : ~kb);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e == e0 + j) {
          pos[j] = i;
          key[j] = 0u;
        }
    }
    const float amax = cap * capped(top * inv_cap).t;
    float ep[4], sp = 0.f, sz = 0.f, ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = cap * capped(v[j] * inv_cap).t - amax;
      const bool in = e0 + j < E;
      ep[j] = in ? __expf(d * inv_tau) : 0.f;
      sz += in ? __expf(d) : 0.f;
      sp += ep[j];
      ss += pos[j] >= 0 ? ep[j] : 0.f;
    }
    sp = lanes_sum<L>(sp);
    sz = lanes_sum<L>(sz);
    ss = lanes_sum<L>(ss);
    const float inv_sp = 1.f / sp, inv_s = 1.f / (ss * inv_sp + 1e-6f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float P = ep[j] * inv_sp;
      ps[j] += P;
      if (pos[j] >= 0) {
        ++cn[j];
        a.idx[b * k + pos[j]] = e0 + j;
        a.w[b * k + pos[j]] = P * inv_s;
      }
    }
    if (l == 0) {
      const float lse = amax + __logf(sz);
      zs += lse * lse;
      ++n;
    }
  }
  // this work-group's column sums: over the wave's tokens, then over its waves
#pragma unroll
  for (int o = L; o < 64; o <<= 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ps[j] += __shfl_xor(ps[j], o);
      cn[j] += __shfl_xor(cn[j], o);
    }
    zs += __shfl_xor(zs, o);
    n += __shfl_xor(n, o);
  }
  constexpr int W = kRouterThreads / 64;
  __shared__ float s_p[W][4 * L], s_z[W];
  __shared__ uint32_t s_c[W][4 * L], s_n[W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (lane < L) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s_p[wave][e0 + j] = ps[j];
      s_c[wave][e0 + j] = cn[j];
    }
    if (l == 0) {
      s_z[wave] = zs;
      s_n[wave] = n;
    }
  }
  __syncthreads();
  // part: (2 E + 2, blocks): sums of P, counts, then z and N
  const int64_t nb = gridDim.x;
  for (int c = threadIdx.x; c < 2 * E + 2; c += kRouterThreads) {
    if (c < E || c == 2 * E) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) v += c < E ? s_p[w][c] : s_z[w];
      a.part[c * nb + blockIdx.x] = v;
    } else {
      uint32_t v = 0u;
#pragma unroll
      for (int w = 0; w < W; ++w) v += c < 2 * E ? s_c[w][c - E] : s_n[w];
      a.part[c * nb + blockIdx.x] = __uint_as_float(v);
    }
  }
}

// counts, lb, z and N from the forward's planes; one work-group, a wave to a column.
__global__ __launch_bounds__(1024) void k_router_finish(RouterArgs a) {
  const int E = a.E, nb = a.blocks, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __shared__ float s_p[kRouterMaxE], s_c[kRouterMaxE], s_z, s_n;
  for (int c = wave; c < 2 * E + 2; c += 16) {
    const float* col = a.part + (int64_t)c * nb;
    if (c < E || c == 2 * E) {
      float v = 0.f;
      for (int i = lane; i < nb; i += 64) v += col[i];
      v = lanes_sum<64>(v);
      if (lane == 0) (c < E ? s_p[c] : s_z) = v;
    } else {
      uint32_t v = 0u;
      for (int i = lane; i < nb; i += 64) v += __float_as_uint(col[i]);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
      if (lane == 0) {
        if (c < 2 * E) {
          a.counts[c - E] = v;
          s_c[c - E] = (float)v;
        } else {
          s_n = (float)v;
        }
      }
    }
  }
  __syncthreads();
  if (wave == 0) {
    const float inv_n = s_n > 0.f ? 1.f / s_n : 0.f;
    float lb = 0.f;
    for (int e = lane; e < E; e += 64) lb += (s_c[e] * inv_n) * (s_p[e] * inv_n);
    lb = lanes_sum<64>(lb);
    if (lane == 0) {
      *a.lb = (float)E * lb;
      *a.z = s_z * inv_n;
      *a.tokens = s_n;
    }
  }
}

template <class T, int L>
__global__ __launch_bounds__(kRouterThreads) void k_router_bwd(RouterArgs a) {
  constexpr int G = kRouterThreads / L;
  const T* raw = static_cast<const T*>(a.raw);
  T* draw = static_cast<T*>(a.draw);
  const int E = a.E, k = a.k, l = threadIdx.x & (L - 1), e0 = 4 * l;
  const float cap = a.cap, inv_cap = 1.f / cap;
  const float inv_tau = 1.f / (a.tau_dev ? *a.tau_dev : a.tau);
  const bool vec = (reinterpret_cast<uintptr_t>(raw) & (4 * sizeof(T) - 1)) == 0 &&
                   (a.row_stride & 3) == 0;
  const bool vec_out = (E & 3) == 0 && (reinterpret_cast<uintptr_t>(draw) & (4 * sizeof(T) - 1)) == 0;
  const float N = *a.tokens, inv_n = N > 0.f ? 1.f / N : 0.f;
  const float cg = a.dlb ? *a.dlb * (float)E * inv_n * inv_n : 0.f;
  const float cz = a.dz ? *a.dz * 2.f * inv_n : 0.f;
  float g0[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) g0[j] = e0 + j < E ? cg * (float)a.counts[e0 + j] : 0.f;
  for (int64_t b = (int64_t)blockIdx.x * G + threadIdx.x / L; b < a.B;
       b += (int64_t)gridDim.x * G) {
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    if (!a.mask || a.mask[b]) {
      float v[4], dw[4] = {0.f, 0.f, 0.f, 0.f};
      bool sel[4] = {false, false, false, false};
      router_load(raw + b * a.row_stride, e0, E, vec, v);
      for (int i = 0; i < k; ++i) {
        const int64_t e = a.idx[b * k + i];
        const float d = a.dw ? a.dw[b * k + i] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e == e0 + j) {
            sel[j] = true;
            dw[j] = d;
          }
      }
      Capped t[4];
      float amax = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[j] = capped(v[j] * inv_cap);
        if (e0 + j < E) amax = fmaxf(amax, cap * t[j].t);
      }
#pragma unroll
      for (int s = L / 2; s >= 1; s >>= 1) amax = fmaxf(amax, __shfl_xor(amax, s));
      float ep[4], ez[4], sp = 0.f, sz = 0.f, ss = 0.f, sd = 0.f, sg = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = cap * t[j].t - amax;
        const bool in = e0 + j < E;
        ep[j] = in ? __expf(d * inv_tau) : 0.f;
        ez[j] = in ? __expf(d) : 0.f;
        sp += ep[j];
        sz += ez[j];
        ss += sel[j] ? ep[j] : 0.f;
        sd += sel[j] ? ep[j] * dw[j] : 0.f;
        sg += ep[j] * g0[j];
      }
      sp = lanes_sum<L>(sp);
      sz = lanes_sum<L>(sz);
      ss = lanes_sum<L>(ss);
      sd = lanes_sum<L>(sd);
      sg = lanes_sum<L>(sg);
      const float inv_sp = 1.f / sp;
      const float S = ss * inv_sp, inv_s = 1.f / (S + 1e-6f);
      const float dot = sd * inv_sp * inv_s;                       // sum_i dw_i w_i
      // sum_e P_e g_e: the balance loss's part and the selected ones'
      const float pg = sg * inv_sp + (sd * inv_sp - S * dot) * inv_s;
      const float zc = cz * (amax + __logf(sz)) / sz;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float g = g0[j] + (sel[j] ? (dw[j] - dot) * inv_s : 0.f);
        o[j] = (ep[j] * inv_sp * (g - pg) * inv_tau + zc * ez[j]) * t[j].sech2;
      }
    }
    T* row = draw + b * E;
    if (vec_out && e0 + 4 <= E) {
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(row + e0) = make_float4(o[0], o[1], o[2], o[3]);
      else
        *reinterpret_cast<uint2*>(row + e0) =
            make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e0 + j < E) store_from_f32(row + e0 + j, o[j]);
    }
  }
}

}  // namespace dev
}  // namespace tmoe
