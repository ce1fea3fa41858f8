// What the attention kernels share: vectors of words, products on the matrix cores, quotients.
#pragma once

#include "elements.hpp"

namespace certex_amd::attention {

using f32x4  = __attribute__((ext_vector_type(4))) float;
using u32x4  = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2  = __attribute__((ext_vector_type(2))) uint32_t;
using f16x8  = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;

/** A value that all lanes have, in scalar registers. */
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x)
{
  const uint32_t lo = uint32_t(uniform(int(x))), hi = uint32_t(uniform(int(x >> 32)));
  return int64_t(uint64_t(hi) << 32 | lo);
}
template <typename T>
__device__ __forceinline__ const T* uniform(const T* p)
{
  return reinterpret_cast<const T*>(uniform(int64_t(reinterpret_cast<uintptr_t>(p))));
}

/** The LDS byte address of p. */
__device__ __forceinline__ uint32_t lds_address(const void* p)
{
  return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)(const_cast<void*>(p))));
}

/** 16 bytes a lane from base + offset to LDS byte m0 + 16 lane. In assembly, so that the compiler does not order LDS reads
 *  against it: the kernels see to it that what is copied over has been read, and wait for vmcnt before they read the copy.
 *  (It is among the loads that the compiler's own waits pass over in order: those can only wait longer.) Nor does the compiler see
 *  that it reads scalar registers: a vector instruction that writes one (a lane read, as where scalars are spilled) has to be 5 wait
 *  states before, which are here. M0 is an operand, which the compiler writes: named as clobbered it would be undefined. */
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t offset, uint32_t m0)
{
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(uniform(static_cast<const char*>(base))), "{m0}"(m0)
               : "memory");
}
__device__ __forceinline__ void copy_to_lds(const void* from, uint32_t m0)
{
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(m0) : "memory");
}

/** n / d for n < 2^29 by a product: m = ceil(2^(29 + s) / d) with 2^s >= d exceeds 2^(29 + s) / d by less
 *  than 1, so n m / 2^(29 + s) exceeds n / d by less than 1 / d. */
struct divisor {
  uint32_t m, shift, d;
  explicit divisor(uint32_t by) : d(by)
  {
    uint32_t s = 0;
    while ((uint64_t(1) << s) < by) { ++s; }
    shift = 29 + s;
    m     = uint32_t(((uint64_t(1) << shift) + by - 1) / by);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return uint32_t((uint64_t(n) * m) >> shift); }
};

__device__ __forceinline__ f32x4 mfma(f16_t, u32x4 a, u32x4 b, f32x4 c)
{
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16_t, u32x4 a, u32x4 b, f32x4 c)
{
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
  using two = __attribute__((ext_vector_type(2))) T;
  using f32x2 = __attribute__((ext_vector_type(2))) float;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), two));
}

/** The elements of a word. */
template <typename T>
__device__ __forceinline__ float lower(uint32_t w)
{
  using two = __attribute__((ext_vector_type(2))) T;
  return float(__builtin_bit_cast(two, w)[0]);
}
template <typename T>
__device__ __forceinline__ float upper(uint32_t w)
{
  using two = __attribute__((ext_vector_type(2))) T;
  return float(__builtin_bit_cast(two, w)[1]);
}

}  // namespace certex_amd::attention
