// What the routers share: a token's logits in its lanes, and whole numbers in the order of
// floats to select by.
#pragma once

#include "tmoe_elem.hpp"

namespace tmoe {
namespace dev {

constexpr int kRouterTopK = 16;       // slots of a token at most

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

// The largest key below `best`; one exists, or a key of 0 is none.
template <int L, int V>
__device__ __forceinline__ uint32_t key_below(const uint32_t (&key)[V], uint32_t best) {
  uint32_t below[V];
#pragma unroll
  for (int j = 0; j < V; ++j) below[j] = key[j] - best;
  return lanes_max<L>(max_of(below)) + best;
}

}  // namespace dev
}  // namespace tmoe
