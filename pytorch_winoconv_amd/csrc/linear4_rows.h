// What the products of few rows over a weight in 4 bits share (linear4_few.hip, linear4_gradient.hip): eight widened values a lane as an operand.
#pragma once
#include "packed4.h"

namespace wc {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 multiply(const Pack<half_t, 8>& a, const Pack<half_t, 8>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply(const Pack<bf16_t, 8>& a, const Pack<bf16_t, 8>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// what the weight's codes become
template <typename T> struct Widened { using type = T; };
template <> struct Widened<float> { using type = bf16_t; };

// x: eight values of T, times eight of the weight
template <typename T>
__device__ __forceinline__ f32x4 multiply_run(const T (&x)[8], const Pack<typename Widened<T>::type, 8>& w, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
    Pack<bf16_t, 8> part;
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned bits = __float_as_uint(x[e]);
      const float high = __uint_as_float(bits & 0xffff0000u);
      part.v[e] = __builtin_bit_cast(bf16_t, (unsigned short)(bits >> 16));
      // (of an infinity nothing is left; a NaN whose upper half says infinity stays one)
      rest[e] = (bits & 0x7fffffffu) == 0x7f800000u ? 0.f : x[e] - high;
    }
    c = multiply(w, part, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      part.v[e] = static_cast<bf16_t>(rest[e]);
      rest[e] -= static_cast<float>(part.v[e]);
    }
    c = multiply(w, part, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) part.v[e] = static_cast<bf16_t>(rest[e]);
    return multiply(w, part, c);
  } else {
    Pack<T, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v.v[e] = x[e];
    return multiply(w, v, c);
  }
}

}  // namespace wc
