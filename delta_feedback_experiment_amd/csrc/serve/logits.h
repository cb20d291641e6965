// Rows of logits as the operators on them read them (gfx950).
#pragma once

#include "pkda_common.h"
#include "serve/pkda_serve_gfx950.h"

namespace pkda {

constexpr float kMaxFloat = 3.402823466e38f;

// A logit as the operator takes it: NaN as -inf (never taken), +inf as the
// largest finite number.
__device__ __forceinline__ float usable(float x) { return x > -INFINITY ? fminf(x, kMaxFloat) : -INFINITY; }

// 16 bytes of a row that begins anywhere.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
template <typename T> struct Logits;
template <> struct Logits<float> {
  static constexpr int N = 4;
  static constexpr uint32_t none = 0xff800000u;  // -inf
  __device__ __forceinline__ static float get(const u32x4& v, int j) { return __uint_as_float(v[j]); }
  __device__ __forceinline__ static void clean(u32x4& v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __float_as_uint(usable(get(v, j)));
  }
};
template <> struct Logits<bf16_t> {
  static constexpr int N = 8;
  static constexpr uint32_t none = 0xff80ff80u;
  __device__ __forceinline__ static float get(const u32x4& v, int j) {
    return __uint_as_float(j & 1 ? v[j / 2] & 0xffff0000u : v[j / 2] << 16);
  }
  // (the largest BF16 for +inf: kMaxFloat has no BF16 of its own)
  __device__ __forceinline__ static void clean(u32x4& v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = __float_as_uint(usable(get(v, 2 * j))), hi = __float_as_uint(usable(get(v, 2 * j + 1)));
      v[j] = (lo >> 16) | (hi & 0xffff0000u);
    }
  }
};

}  // namespace pkda
