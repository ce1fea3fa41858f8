// Elements of the attention operators' tensors (float32, float16 and bfloat16, computed in float32), and the weights of a
// softmax.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

namespace certex_amd::attention {

using f16_t  = _Float16;
using bf16_t = __bf16;

/** N elements that one load or store moves. */
template <typename T, int N>
struct alignas(sizeof(T) * N) pack {
  T e[N];
};

template <typename T, int N>
__device__ __forceinline__ pack<T, N> load(const T* p)
{
  return *reinterpret_cast<const pack<T, N>*>(p);
}
/** The same at any address of the elements: the memory takes misaligned vectors. */
template <typename T, int N>
__device__ __forceinline__ pack<T, N> load_loose(const T* p)
{
  pack<T, N> v;
  __builtin_memcpy(&v, __builtin_assume_aligned(p, sizeof(T)), sizeof(v));
  return v;
}
template <typename T, int N>
__device__ __forceinline__ void store_loose(T* p, pack<T, N> const& v)
{
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &v, sizeof(v));
}

/** Elements that the call reads once: not kept in the caches. */
template <typename T, int N>
__device__ __forceinline__ pack<T, N> load_once(const T* p)
{
  if constexpr (sizeof(T) * N >= 4) {
    using words = uint32_t __attribute__((ext_vector_type(sizeof(T) * N / 4)));
    return __builtin_bit_cast(pack<T, N>, __builtin_nontemporal_load(reinterpret_cast<const words*>(p)));
  } else {
    return load<T, N>(p);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, pack<T, N> const& v)
{
  *reinterpret_cast<pack<T, N>*>(p) = v;
}

constexpr float kLog2e = 1.44269504088896340736f;

/**
 * The scale of a softmax's scores: weights are 2^(scale2 (score - top)). Scores are subtracted before they are scaled: what
 * is rounded is their distance from the largest one, however far from 0 they are, and that one weighs 1. They are signed
 * by the scale's sign, so that the largest weighs most.
 */
struct score_scale {
  float sign;    // of the scale
  float scale;   // its magnitude
  float scale2;  // that times log2(e)
};

inline score_scale scale_of(float scale)
{
  const double s = std::abs(double(scale));
  return {scale < 0.0f ? -1.0f : 1.0f, float(s), float(std::min(s * M_LOG2E, double(FLT_MAX)))};
}

/** The weight of a score relative to the finite score `top`; -inf counts nothing, NaN stays. */
__device__ __forceinline__ float weight_of(score_scale const& s, float score, float top)
{
  const float d = score - top;
  // a distance past the largest float: that much, so that a scale of 0 or near it has its say
  return score == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((d < -FLT_MAX ? -FLT_MAX : d) * s.scale2);
}

/** What sums taken relative to the score `part` count relative to `whole` >= part. Where nothing was counted both are
 *  -inf, and the sums are 0, or NaN of NaN scores: they pass as they are. */
__device__ __forceinline__ float factor_of(score_scale const& s, float part, float whole)
{
  return whole == -INFINITY ? 1.0f : weight_of(s, part, whole);
}

/** The logarithm of a sum of weights relative to `top`, 2^lift times themselves. */
__device__ __forceinline__ float lse_of(score_scale const& s, float top, float sum, float lift = 0.0f)
{
  return sum == 0.0f ? -INFINITY : __builtin_fmaf(top, s.scale, (__builtin_log2f(sum) - lift) / kLog2e);
}

}  // namespace certex_amd::attention
