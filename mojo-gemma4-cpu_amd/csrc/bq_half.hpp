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

// ---------------------------------------------------------------------------
// Reductions over a wave, the result in every lane: neighbours by DPP (lane ^ 1, ^ 2,
// then halves and rows mirrored, whose lanes hold the same by then), rows of 16 and
// halves of 32 by lane swaps.
// ---------------------------------------------------------------------------
template <int CTRL>
__device__ inline uint32_t dpp32(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}
template <typename T, typename F>
__device__ inline T wave_all(T v, F&& f) {
  constexpr int W = sizeof(T) / 4;
  struct Words {
    uint32_t w[W];
  };
  auto step = [&](auto&& other) {
    Words a = __builtin_bit_cast(Words, v), b;
#pragma unroll
    for (int i = 0; i < W; ++i) b.w[i] = other(a.w[i]);
    v = f(v, __builtin_bit_cast(T, b));
  };
  step([](uint32_t x) { return dpp32<0xB1>(x); });   // quad_perm [1, 0, 3, 2]
  step([](uint32_t x) { return dpp32<0x4E>(x); });   // quad_perm [2, 3, 0, 1]
  step([](uint32_t x) { return dpp32<0x141>(x); });  // row_half_mirror
  step([](uint32_t x) { return dpp32<0x140>(x); });  // row_mirror
  auto swapped = [&](auto&& swap) {
    const Words a = __builtin_bit_cast(Words, v);
    Words lo, hi;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const auto r = swap(a.w[i]);
      lo.w[i] = r[0];
      hi.w[i] = r[1];
    }
    v = f(__builtin_bit_cast(T, lo), __builtin_bit_cast(T, hi));
  };
  swapped([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  swapped([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
  return v;
}
__device__ inline float wave_all_max(float v) {
  return wave_all(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline double wave_all_sum(double v) {
  return wave_all(v, [](double a, double b) { return a + b; });
}

// ---------------------------------------------------------------------------
// Results that another workgroup of the same launch reads: past the caches that are
// not shared by all of the device, both ways.
// ---------------------------------------------------------------------------
typedef float v2f __attribute__((ext_vector_type(2)));
__device__ inline void store_agent(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void store_agent(float* p, float x, float y) {
  store_agent(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v2f{x, y}));
}
__device__ inline uint64_t load_agent(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline v2f load2_agent(const float* p) {
  return __builtin_bit_cast(v2f, load_agent(reinterpret_cast<const uint64_t*>(p)));
}
// the wave's stores so far have arrived
__device__ inline void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Whether this is the last of `count` workgroups that share the marks, each of which
// has waited (stores_done) for what it leaves to the others, in every wave.  Every
// workgroup marks its place with the launch's tag, then looks at all marks: the last
// to mark sees them all (two may, and then both do the same work).  Whoever does takes
// the marks off, for a replay of the launch; what memory held before the first one is
// no tag.  Called by all threads; `said` is LDS.
__device__ inline bool last_of(uint64_t* marks, int64_t stride, int count, int place, uint64_t tag,
                               int* said) {
  __syncthreads();
  if (threadIdx.x < 64) {
    if (threadIdx.x == 0) store_agent(marks + place * stride, tag);
    stores_done();
    bool seen = true;
    for (int i = threadIdx.x; i < count; i += 64) seen &= load_agent(marks + i * stride) == tag;
    seen = __ballot(!seen) == 0;
    if (seen)
      for (int i = threadIdx.x; i < count; i += 64) store_agent(marks + i * stride, 0);
    if (threadIdx.x == 0) *said = seen;
  }
  __syncthreads();
  return *said != 0;
}

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
