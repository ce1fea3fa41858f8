// Scores that are bent before the softmax: capped by a tanh, leaning on distance.
#pragma once

#include "elements.hpp"

namespace certex_amd::attention {

/** y = cap tanh(scale x / cap) - slopes[head] * |p - t| for the query's position p and the key's t. */
struct score_shape {
  float cap           = 0;        // 0: scale x as it is
  const float* slopes = nullptr;  // [heads], or NULL: none
  [[nodiscard]] bool any() const { return cap != 0.0f || slopes != nullptr; }
};

/** Up to this size tanh is a polynomial. (Of a degree less, up to 0.6, it takes prompts as long.) */
constexpr float kNear = 0.8f;

/**
 * tanh(u) for |u| < kNear, within 2 units in the last place: u + u s p(s) with s = u^2, p of degree 5 with the least largest error of
 * s p(s) over [0, 0.64] (fitted: 3.4e-9, coefficients rounded to float32). What is added to u is 0.17 u at most, so that its
 * roundings, four units or less, weigh little.
 */
__device__ __forceinline__ float tanh_near(float u)
{
  const float s = u * u;
  float p = __builtin_fmaf(s, 0.0015930377412587404f, -0.007425214163959026f);
  p       = __builtin_fmaf(s, p, 0.02131400816142559f);
  p       = __builtin_fmaf(s, p, -0.05385585501790047f);
  p       = __builtin_fmaf(s, p, 0.13332270085811615f);
  p       = __builtin_fmaf(s, p, -0.33333298563957214f);
  return __builtin_fmaf(u * s, p, u);
}

/**
 * tanh(u) within 3 units in the last place, NaN where u is, if the exponential and the reciprocal are within one: tanh_near, and beyond
 * 1 - 2 / (e + 1) with e = 2^(2 log2(e) |u|), where roundings of e weigh 2 e / (e + 1)^2, 0.28 at most, those of the quotient 0.34.
 */
__device__ __forceinline__ float tanh_of(float u)
{
  const float a = __builtin_fabsf(u);
  const float e = __builtin_amdgcn_exp2f(a * (2.0f * kLog2e));  // infinite: 2 / (e + 1) is 0
  const float far = __builtin_copysignf(__builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f), u), near = tanh_near(u);
  // by a mask that the compiler does not look into: it makes branches of such conditions, 32 a tile in prompts' kernels, and spills
  uint32_t small = a < kNear ? 0xffffffffu : 0u;
  asm("" : "+v"(small));
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, near) & small) | (__builtin_bit_cast(uint32_t, far) & ~small));
}

/** The bent score of a product x; per_cap = scale / cap. */
__device__ __forceinline__ float bent(float x, float scale, float per_cap, float cap, float slope, float distance)
{
  const float y = cap != 0.0f ? cap * tanh_of(x * per_cap) : x * scale;
  return __builtin_fmaf(-slope, distance, y);
}

}  // namespace certex_amd::attention
