// Element types of the device code: bf16 bits and floats, and 16-byte chunks of them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tmoe {
namespace dev {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint16_t f32_to_bf16_bits(float f) {
  return __builtin_bit_cast(uint16_t, (__bf16)f);   // round to nearest even
}
// Two floats to two bf16 (round to nearest even) in one register; as a vector
// conversion this is a single v_cvt_pk_bf16_f32.
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

__device__ __forceinline__ float load_as_f32(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ __forceinline__ float load_as_f32(const float* p) { return *p; }
__device__ __forceinline__ void store_from_f32(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }
__device__ __forceinline__ void store_from_f32(float* p, float v) { *p = v; }

// f over the values of L lanes (a power of two, aligned), the same result in all of them:
// neighbours of a quad, quads of 8, halves of 16 (mirrored: each holds one value by then),
// then the swapped rows of 16 and halves of the wave. Lanes of other groups may be off.
template <int L, int kStep = 1, class F>
__device__ __forceinline__ uint32_t lanes_reduce(uint32_t v, F f) {
  if constexpr (kStep < L) {
    if constexpr (kStep == 1) v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true));
    if constexpr (kStep == 2) v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true));
    if constexpr (kStep == 4) v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true));
    if constexpr (kStep == 8) v = f(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true));
    if constexpr (kStep == 16) {
      const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
      v = f(r[0], r[1]);
    }
    if constexpr (kStep == 32) {
      const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
      v = f(r[0], r[1]);
    }
    return lanes_reduce<L, 2 * kStep>(v, f);
  } else {
    return v;
  }
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  return __uint_as_float(lanes_reduce<L>(__float_as_uint(v), [](uint32_t x, uint32_t y) {
    return __float_as_uint(__uint_as_float(x) + __uint_as_float(y));
  }));
}
template <int L>
__device__ __forceinline__ double lanes_sum64(double v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  return lanes_reduce<L>(v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}
template <int L>
__device__ __forceinline__ uint32_t lanes_min(uint32_t v) {
  return lanes_reduce<L>(v, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
}

}  // namespace dev
}  // namespace tmoe
