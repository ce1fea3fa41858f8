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

/**
 * tanh(u) within 3 units in the last place, NaN where u is, if the exponential and the reciprocal are within one. With s = u^2, up to
 * 0.6 in size u - u s (315 + 14 s) / (945 + 420 s + 15 s^2), the fifth convergent of its continued fraction less u: it is off by
 * u^10 / (945 * 10395) of it, 6e-10, and what is taken from u is 0.105 u at most, so that its roundings (7.3 halves of a unit) weigh an
 * eighth. Beyond 1 - 2 / (e + 1) with e = 2^(2 log2(e) |u|): roundings of e weigh 2 e / (e + 1)^2, 0.36 at most, those of the
 * quotient 0.46. One reciprocal for both.
 */
__device__ __forceinline__ float tanh_of(float u)
{
  const float a = __builtin_fabsf(u), s = u * u;
  const float e = __builtin_amdgcn_exp2f(a * (2.0f * kLog2e));  // infinite: 2 / (e + 1) is 0
  // by a mask that the compiler does not look into: it makes branches of such conditions, 32 a tile in prompts' kernels, and spills
  uint32_t small = a < 0.6f ? 0xffffffffu : 0u;
  asm("" : "+v"(small));
  const auto pick = [small](float x, float y) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & small) | (__builtin_bit_cast(uint32_t, y) & ~small));
  };
  const float over  = pick(s * __builtin_fmaf(s, 14.0f, 315.0f), 2.0f);
  const float under = pick(__builtin_fmaf(s, __builtin_fmaf(s, 15.0f, 420.0f), 945.0f), e + 1.0f);
  const float whole = pick(u, __builtin_copysignf(1.0f, u));
  return __builtin_fmaf(-whole, over * __builtin_amdgcn_rcpf(under), whole);
}

/** The bent score of a product x; per_cap = scale / cap. */
__device__ __forceinline__ float bent(float x, float scale, float per_cap, float cap, float slope, float distance)
{
  const float y = cap != 0.0f ? cap * tanh_of(x * per_cap) : x * scale;
  return __builtin_fmaf(-slope, distance, y);
}

}  // namespace certex_amd::attention
