// Elements of the attention operators' tensors: float32, float16 and bfloat16, computed in float32.
#pragma once

#include <hip/hip_runtime.h>

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

/** What sums taken relative to the maximum `part` count relative to `whole` >= part (both in powers of 2). Where nothing
 *  was counted both are -inf, and the sums are 0, or NaN of NaN scores: they pass as they are. */
__device__ __forceinline__ float factor_of(float part, float whole)
{
  return whole == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(part - whole);
}

}  // namespace certex_amd::attention
