// The rotation of a pair of elements by its position.
#pragma once

#include "elements.hpp"

namespace certex_amd::attention {

/** x in the element type, rounded from its float32 value: the compiler would round some float16 results once from the
 *  exact sum of products (v_fma_mixlo_f16) and others twice, so that the vector's width showed in the bits. */
template <typename T>
__device__ __forceinline__ T narrowed(float x)
{
  if constexpr (std::is_same_v<T, f16_t>) { asm("" : "+v"(x)); }
  return T(x);
}

struct sines {
  float c, s;
};

/** Of the angle of position p and a frequency in turns times 2^64: the product's low half is the fraction of a turn,
 *  exactly. Its top 24 bits go to the sine and the cosine, the next 8 turn the result by their small angle. */
__device__ __forceinline__ sines sines_of(int64_t p, uint64_t frequency)
{
  const uint32_t turns = uint32_t((uint64_t(p) * frequency) >> 32);
  float sine, cosine;
  sincospif(float(int32_t(turns & ~255u)) * 0x1p-31f, &sine, &cosine);
  const float rest = float(turns & 255u) * float(M_PI * 0x1p-31);
  return {__builtin_fmaf(sine, -rest, cosine), __builtin_fmaf(cosine, rest, sine)};
}

template <typename T>
__device__ __forceinline__ T turned_first(float f, float g, float c, float s)
{
  return narrowed<T>(__builtin_fmaf(f, c, -(g * s)));
}
template <typename T>
__device__ __forceinline__ T turned_second(float f, float g, float c, float s)
{
  return narrowed<T>(__builtin_fmaf(f, s, g * c));
}

}  // namespace certex_amd::attention
