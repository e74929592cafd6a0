// One AdamW step over many tensors (the reference trains with torch's AdamW,
// pre-train/train.py:1263-1268), with the moments in fp32 or in 8 bits:
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// 8-bit states hold m and r = sqrt(v) as e4m3 codes, each kAdamwBlock elements with one
// fp32 scale, the block's largest value / 448. Rounding to nearest would hold a slow
// average where it is: at b2 = 0.999 v moves by 1/1000 a step, half a code's step is 1/16.
// Codes are therefore rounded to the lower or the upper neighbour at random, so that the
// expected m, and the expected v = r^2, are the unrounded ones: m goes up with the chance
// (a - lo) / (hi - lo), r with (a^2 - lo^2) / (hi^2 - lo^2). The random bits are a hash of
// (seed, step, tensor, element), so a step repeated gives the same bits. A positive r is
// never coded as zero: its element's step would be m / eps.
//
// fp32 is bound by memory: 28 bytes an element, 417 M of them in 2265 us, 5.2 TB/s. 8 bits
// by instructions, 77 an element (the vector units work 94% of the time): 19.3 M bf16
// parameters in 49.3 us, 3.9 TB/s. A launch takes up to kAdamwTensors tensors, their addresses
// in its arguments: nothing is copied to the device, and a captured step holds them. A
// work-group takes `chunk` elements of one tensor.
#pragma once

#include "tmoe_elem.hpp"
#include "tmoe_train.h"

namespace tmoe {
namespace dev {

constexpr int kAdamwTensors = 56;     // a launch's arguments hold 4 KB at most
constexpr int kAdamwThreads = 256;
constexpr float kE4m3Max = 448.f;

struct AdamwTable {
  void* p[kAdamwTensors];
  const void* g[kAdamwTensors];
  void* m[kAdamwTensors];
  void* v[kAdamwTensors];
  float* ms[kAdamwTensors];
  float* vs[kAdamwTensors];
  int64_t n[kAdamwTensors];
  uint32_t end[kAdamwTensors];        // work-groups of this tensor and those before it
  const int64_t* step_dev;
  int64_t chunk;
  double beta1, beta2, lr;            // read where the step is on the device
  uint32_t seed, first;               // first: number of the launch's first tensor
  int count;
  float b1, ob1, b2, ob2, eps, keep, rate, inv_c2;
};

__host__ __device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

struct AdamwStep {
  float b1, ob1, b2, ob2, eps, keep, rate, inv_c2;
  uint32_t key;
  int64_t base;                       // the work-group's first element
  int t;                              // its tensor
};

// The step's numbers and the work-group's place.
__device__ __forceinline__ AdamwStep adamw_step(const AdamwTable& a) {
  AdamwStep s{a.b1, a.ob1, a.b2, a.ob2, a.eps, a.keep, a.rate, a.inv_c2, 0u, 0, 0};
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (blockIdx.x < a.end[mid]) hi = mid;
    else lo = mid + 1;
  }
  s.t = lo;
  s.base = (int64_t)(blockIdx.x - (lo ? a.end[lo - 1] : 0u)) * a.chunk;
  uint32_t step = 0u;
  if (a.step_dev) {
    __shared__ float c[2];
    __shared__ uint32_t st;
    if (threadIdx.x == 0) {
      const double n = (double)*a.step_dev;
      c[0] = (float)(a.lr / (1.0 - pow(a.beta1, n)));
      c[1] = 1.f / (float)sqrt(1.0 - pow(a.beta2, n));
      st = (uint32_t)*a.step_dev;
    }
    __syncthreads();
    s.rate = c[0];
    s.inv_c2 = c[1];
    step = st;
    s.key = mix32(a.seed + step * 0x9E3779B1u);
  } else {
    s.key = a.seed;                   // mixed on the host
  }
  return s;
}

// The new moments and parameter of one element, each operation rounded as it is written:
// the 8-bit codes of one step decide the next one's values.
__device__ __forceinline__ void adamw_moments(const AdamwStep& s, float g, float& m, float& v) {
#pragma clang fp contract(off)
  m = m * s.b1 + g * s.ob1;
  v = v * s.b2 + g * g * s.ob2;
}
__device__ __forceinline__ float adamw_param(const AdamwStep& s, float p, float m, float root) {
#pragma clang fp contract(off)
  return p * s.keep - (m / (root * s.inv_c2 + s.eps)) * s.rate;
}

// N neighbours at any alignment (a view may begin anywhere).
template <int N, class T>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
  constexpr int W = N * (int)sizeof(T) / 4;
  typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  const vec q = *reinterpret_cast<const vec*>(p);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(q[j]);
    else v[j] = __uint_as_float(j & 1 ? q[j / 2] & 0xffff0000u : q[j / 2] << 16);
}
template <int N, class T>
__device__ __forceinline__ void store_n(T* p, const float (&v)[N]) {
  constexpr int W = N * (int)sizeof(T) / 4;
  typedef uint32_t vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  vec q;
#pragma unroll
  for (int j = 0; j < W; ++j)
    if constexpr (sizeof(T) == 4) q[j] = __float_as_uint(v[j]);
    else q[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<vec*>(p) = q;
}
typedef uint32_t codes8 __attribute__((ext_vector_type(2), aligned(1)));

template <class T>
__global__ __launch_bounds__(kAdamwThreads) void k_adamw32(const AdamwTable a) {
  const AdamwStep s = adamw_step(a);
  T* p = static_cast<T*>(a.p[s.t]);
  const T* g = static_cast<const T*>(a.g[s.t]);
  float* m = static_cast<float*>(a.m[s.t]);
  float* v = static_cast<float*>(a.v[s.t]);
  const int64_t end = s.base + a.chunk < a.n[s.t] ? s.base + a.chunk : a.n[s.t];
  int64_t i = s.base + 4 * threadIdx.x;
  for (; i + 4 <= end; i += 4 * kAdamwThreads) {
    float pv[4], gv[4], mv[4], vv[4];
    load_n<4>(p + i, pv);
    load_n<4>(g + i, gv);
    load_n<4>(m + i, mv);
    load_n<4>(v + i, vv);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      adamw_moments(s, gv[j], mv[j], vv[j]);
      pv[j] = adamw_param(s, pv[j], mv[j], sqrtf(vv[j]));
    }
    store_n<4>(p + i, pv);
    store_n<4>(m + i, mv);
    store_n<4>(v + i, vv);
  }
  for (; i < end; ++i) {      // a tensor's last one to three elements, one thread's
    float mv = m[i], vv = v[i];
    adamw_moments(s, load_as_f32(g + i), mv, vv);
    store_from_f32(p + i, adamw_param(s, load_as_f32(p + i), mv, sqrtf(vv)));
    m[i] = mv;
    v[i] = vv;
  }
}

// a / b rounded as the division is, of a reciprocal y of b that is rounded so (the product's
// error, found exactly, corrects it): the codes are the unrounded quotient's.
__device__ __forceinline__ float quotient(float a, float b, float y) {
  const float q = a * y;
  return fmaf(fmaf(-q, b, a), y, q);
}

// sqrt(v) to the last place but for one value in millions; v is 0 or at least 2^-126 (the
// hardware's root takes less for 0), infinite or NaN
__device__ __forceinline__ float root_of(float v) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(v, 0x1p-126f)), s = v * y;
  return v < INFINITY ? fmaf(fmaf(-s, s, v), 0.5f * y, s) : v;
}
__device__ __forceinline__ bool subnormal(float v) { return __builtin_amdgcn_classf(v, 0x80); }
// of any v: a subnormal one's from 2^64 of it
__device__ __forceinline__ float root_of_any(float v) {
  const bool sub = subnormal(v);
  return root_of(sub ? v * 0x1p64f : v) * (sub ? 0x1p-32f : 1.f);
}

// A magnitude a in [0, 448] as the e4m3 value below it and what is left over: `code`, and in
// units of 2^-20 of the step between the two, `at` = the value's place counted from its
// octave's (the subnormals': zero's) first, `rest` over it. kSub: a may be under 2^-6, where
// values are 2^-9 apart as they are from 2^-6 on: the sum's mantissa is both places.
struct E4m3Place {
  uint32_t code, at, rest;
};
template <bool kSub>
__device__ __forceinline__ E4m3Place e4m3_place(float a) {
  const bool sub = kSub && a < 0x1p-6f;
  const uint32_t b = __float_as_uint(sub ? a + 0x1p-6f : a);
  const uint32_t A = (b & 0x7fffffu) | (sub ? 0u : 0x800000u);
  return {(b >> 20) - (sub ? 968u : 960u), A & 0xf00000u, A & 0xfffffu};
}
// The code of a value in byte kByte of c, up with the chance rest / step: where the upper 16
// bits of h, 8 more below them, are under rest. The conversion adds the upper 20 bits that it
// is given to the mantissa and cuts: with their complement it goes up just there (values
// under 2^-6 go by their place). A quotient that rounding put over 448 is a place or two
// over it: no bits are low enough to go up.
template <bool kSub, int kByte>
__device__ __forceinline__ uint32_t e4m3_code(float a, uint32_t h, uint32_t c) {
  if constexpr (kSub) {
    const E4m3Place p = e4m3_place<true>(fabsf(a));
    return c | (p.code + ((h >> 16 << 4 | 8u) < p.rest ? 1u : 0u) |
                (__float_as_uint(a) >> 24 & 0x80u)) << 8 * kByte;
  } else {
    return __builtin_amdgcn_cvt_sr_fp8_f32(a, (h | 0xffffu) ^ 0xffff8fffu, c, kByte);
  }
}
// The code of a root r, up with the chance (r^2 - lo^2) / (hi^2 - lo^2)
// = rest (r + lo) / (hi + lo); odd: (2 q + 1, its reciprocal rounded) for q = 0 .. 15.
template <bool kSub>
__device__ __forceinline__ uint32_t e4m3_root_code(float r, uint32_t u16, const float2* odd) {
#pragma clang fp contract(off)
  const E4m3Place p = e4m3_place<kSub>(r);
  const float2 o = odd[p.at >> 20];
  const float t = quotient((float)(2u * p.at + p.rest), o.x, o.y);
  const float chance = (float)p.rest * t;                       // 2^40 of it
  const float u = fmaf((float)u16, 0x1p+24f, 0x1p+23f);
  const uint32_t c = p.code + (u < chance ? 1u : 0u);
  return kSub ? max(c, min(__float_as_uint(r), 1u)) : c;
}
// The codes of eight moments (m over their scale, r over theirs).
template <bool kSub>
__device__ __forceinline__ void e4m3_codes(const float (&qm)[8], const float (&qr)[8], uint32_t key,
                                           uint32_t step_key, const float2* odd, codes8& m, codes8& r) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t h[4], cm = 0u, cr = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[j] = mix32((key + (uint32_t)(4 * w + j)) ^ step_key);
      cr |= e4m3_root_code<kSub>(qr[4 * w + j], h[j] & 0xffffu, odd) << 8 * j;
    }
    cm = e4m3_code<kSub, 0>(qm[4 * w], h[0], cm);
    cm = e4m3_code<kSub, 1>(qm[4 * w + 1], h[1], cm);
    cm = e4m3_code<kSub, 2>(qm[4 * w + 2], h[2], cm);
    cm = e4m3_code<kSub, 3>(qm[4 * w + 3], h[3], cm);
    m[w] = cm;
    r[w] = cr;
  }
}

// Half a wave takes a block of 256 elements, eight neighbours a lane (a wave with four a lane:
// 52.9 us against 48.6 at 19.3 M when that was measured; the next block read ahead gained nothing there). What
// decides a code is computed as the formulas round it (a step's codes are the next one's
// values), the rest with the hardware's reciprocals: the arithmetic, not the memory, is the
// bound. A moment whose block's scale is under 2^-110 is taken for zero (the reciprocal of
// less overflows).
template <class T>
__global__ __launch_bounds__(kAdamwThreads) void k_adamw8(const AdamwTable a) {
#pragma clang fp contract(off)
  __shared__ float2 odd[16];
  if (threadIdx.x < 16) {
    const float o = (float)(2 * threadIdx.x + 1);
    odd[threadIdx.x] = make_float2(o, 1.f / o);
  }
  __syncthreads();
  const AdamwStep s = adamw_step(a);
  const int64_t n = a.n[s.t];
  constexpr int kEach = 8, kLanes = kAdamwBlock / kEach, kTeams = kAdamwThreads / kLanes;
  // the lanes' part of the work-group's chunk: `count` elements from `first` on, in 32 bits
  const uint32_t lane = threadIdx.x % kLanes, team = threadIdx.x / kLanes;
  const uint32_t all = (uint32_t)(a.chunk < n - s.base ? a.chunk : n - s.base);
  const int64_t first = s.base + team * kAdamwBlock;
  const uint32_t count = all > team * kAdamwBlock ? all - team * kAdamwBlock : 0u;
  T* p = static_cast<T*>(a.p[s.t]) + first;
  const T* g = static_cast<const T*>(a.g[s.t]) + first;
  uint8_t* mq = static_cast<uint8_t*>(a.m[s.t]) + first;
  uint8_t* rq = static_cast<uint8_t*>(a.v[s.t]) + first;
  float* ms = a.ms[s.t] + first / kAdamwBlock;
  float* rs = a.vs[s.t] + first / kAdamwBlock;
  for (uint32_t b = 0, blk = 0; b < count; b += kTeams * kAdamwBlock, blk += kTeams) {
    const uint32_t i = b + kEach * lane;
    const bool whole = i + kEach <= count;
    const int live = i < count ? (int)(count - i) : 0;   // where not whole
    const float sm = ms[blk], sr = rs[blk];
    float pv[kEach] = {}, gv[kEach] = {}, m[kEach], r[kEach];
    codes8 mc = {0u, 0u}, rc = {0u, 0u};
    if (whole) {
      load_n<kEach>(p + i, pv);
      load_n<kEach>(g + i, gv);
      mc = *reinterpret_cast<const codes8*>(mq + i);
      rc = *reinterpret_cast<const codes8*>(rq + i);
    } else {
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (j < live) {
          pv[j] = load_as_f32(p + i + j);
          gv[j] = load_as_f32(g + i + j);
          mc[j / 4] |= (uint32_t)mq[i + j] << 8 * (j % 4);
          rc[j / 4] |= (uint32_t)rq[i + j] << 8 * (j % 4);
        }
    }
#pragma unroll
    for (int j = 0; j < kEach; j += 4) {
      const f32x2_t m01 = __builtin_amdgcn_cvt_pk_f32_fp8(mc[j / 4], false);
      const f32x2_t m23 = __builtin_amdgcn_cvt_pk_f32_fp8(mc[j / 4], true);
      const f32x2_t r01 = __builtin_amdgcn_cvt_pk_f32_fp8(rc[j / 4], false);
      const f32x2_t r23 = __builtin_amdgcn_cvt_pk_f32_fp8(rc[j / 4], true);
      m[j] = m01[0], m[j + 1] = m01[1], m[j + 2] = m23[0], m[j + 3] = m23[1];
      r[j] = r01[0], r[j + 1] = r01[1], r[j + 2] = r23[0], r[j + 3] = r23[1];
    }
    bool sub = false;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      m[j] *= sm;
      r[j] *= sr;
      r[j] *= r[j];
      adamw_moments(s, gv[j], m[j], r[j]);
      sub |= subnormal(r[j]);
    }
    if (__any(sub)) {       // their roots are as large as 2^-63: with an eps of 0 they count
#pragma unroll
      for (int j = 0; j < kEach; ++j) r[j] = root_of_any(r[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kEach; ++j) r[j] = root_of(r[j]);
    }
    // magnitudes as integers: in their order, a NaN above all
    uint32_t am = 0u, ar = 0u;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      pv[j] = fmaf(m[j] * -s.rate, __builtin_amdgcn_rcpf(fmaf(r[j], s.inv_c2, s.eps)), pv[j] * s.keep);
      am = max(am, __float_as_uint(m[j]) & 0x7fffffffu);
      ar = max(ar, __float_as_uint(r[j]) & 0x7fffffffu);
    }
    float nsm = __uint_as_float(lanes_max<kLanes>(am)) * (1.f / kE4m3Max);
    float nsr = __uint_as_float(lanes_max<kLanes>(ar)) * (1.f / kE4m3Max);
    nsm = nsm < 0x1p-110f ? 0.f : nsm;
    nsr = nsr < 0x1p-110f ? 0.f : nsr;
    const float dm = nsm == 0.f ? 1.f : nsm, dr = nsr == 0.f ? 1.f : nsr;
    // reciprocals to half a place, for quotient()
    float im = __builtin_amdgcn_rcpf(dm), ir = __builtin_amdgcn_rcpf(dr);
    im = fmaf(fmaf(-dm, im, 1.f), im, im);
    ir = fmaf(fmaf(-dr, ir, 1.f), ir, ir);
    float least = INFINITY;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      m[j] = quotient(m[j], dm, im);
      r[j] = quotient(r[j], dr, ir);
      least = fminf(least, fminf(fabsf(m[j]), r[j]));
    }
    const uint64_t e = (uint64_t)(first + i);    // the neighbours share its upper half
    const uint32_t key = (a.first + (uint32_t)s.t) * 0x9E3779B9u + (uint32_t)e +
                         (uint32_t)(e >> 32) * 0xC2B2AE35u;
    if (__any(!(least >= 0x1p-6f))) e4m3_codes<true>(m, r, key, s.key, odd, mc, rc);
    else e4m3_codes<false>(m, r, key, s.key, odd, mc, rc);
    if (whole) {
      store_n<kEach>(p + i, pv);
      *reinterpret_cast<codes8*>(mq + i) = mc;
      *reinterpret_cast<codes8*>(rq + i) = rc;
    } else {
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (j < live) {
          store_from_f32(p + i + j, pv[j]);
          mq[i + j] = (uint8_t)(mc[j / 4] >> 8 * (j % 4));
          rq[i + j] = (uint8_t)(rc[j / 4] >> 8 * (j % 4));
        }
    }
    if (lane == 0) {
      ms[blk] = nsm;
      rs[blk] = nsr;
    }
  }
}

}  // namespace dev
}  // namespace tmoe
