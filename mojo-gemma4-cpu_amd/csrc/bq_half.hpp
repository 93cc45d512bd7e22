// bq_half.hpp -- the two 16-bit floating types of the paged cache: conversions
// (round to nearest even; NaN stays NaN), packing, and their matrix products.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bq_device.hpp"

namespace bq {

typedef float v4f32 __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v4hf __attribute__((ext_vector_type(4)));

struct Bf16 {
  static constexpr float kWeightBits = 0.0f;
  __device__ static float lo(uint32_t w) { return __uint_as_float(w << 16); }
  __device__ static float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  __device__ static uint32_t pack(float a, float b) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
  }
  // D[16, 16] += A[16, 32] B[32, 16]: lane l holds 8 k-values of row / column
  // l % 16 of A / B, and rows 4 (l / 16) + r, column l % 16 of D
  __device__ static v4f32 mfma32(v4u a, v4u b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
  __device__ static v4f32 mfma16(v2u a, v2u b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4s, a),
                                                     __builtin_bit_cast(v4s, b), c, 0, 0, 0);
  }
};

struct F16 {
  // Softmax weights, at most 1, are kept 2^14 times as large: f16 loses bits below
  // 2^-14, and many weights of 2^-17 may add up to what counts.
  static constexpr float kWeightBits = 14.0f;
  __device__ static float lo(uint32_t w) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xFFFFu));
  }
  __device__ static float hi(uint32_t w) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  }
  __device__ static uint32_t pack(float a, float b) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    const v2 r = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
  }
  __device__ static v4f32 mfma32(v4u a, v4u b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8hf, a),
                                                  __builtin_bit_cast(v8hf, b), c, 0, 0, 0);
  }
  __device__ static v4f32 mfma16(v2u a, v2u b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4hf, a),
                                                 __builtin_bit_cast(v4hf, b), c, 0, 0, 0);
  }
};

// eight 16-bit values of one 16-byte word
template <typename T>
__device__ inline void unpack8(v4u w, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = T::lo(w[i]);
    v[2 * i + 1] = T::hi(w[i]);
  }
}
template <typename T>
__device__ inline v4u pack8(const float (&v)[8]) {
  v4u w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = T::pack(v[2 * i], v[2 * i + 1]);
  return w;
}

}  // namespace bq
