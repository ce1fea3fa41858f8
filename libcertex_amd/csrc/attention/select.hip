// Attention over a selected top k: the scores are given (a key cache returns them with the ids), so
// no key is read again. out = sum_j p_j v[id_j] / sum_j p_j with p_j = exp(scale (s_j - max s)).
#include "attention.hpp"
#include "elements.hpp"

#include <algorithm>

namespace certex_amd::attention {
namespace {

constexpr int kThreads = 256;

/** One workgroup per query: its weights in LDS, 256 at a time, one column of values per thread. */
template <typename T>
__global__ __launch_bounds__(kThreads) void select_kernel(select_args a)
{
  __shared__ float s_p[kThreads];
  __shared__ int64_t s_v[kThreads];
  __shared__ float s_part[kThreads / 64];
  const int tid     = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int h       = int(row / a.queries), g = h / (a.heads / a.kv_heads);
  const float* s    = a.scores + row * a.k;
  float top         = -INFINITY;
  for (int64_t j = tid; j < a.k; j += kThreads) {
    const int64_t id = a.ids[row * a.k + j];
    if (id >= 0 && id < a.n) { top = fmaxf(top, s[j] * a.scale); }
  }
  for (int d = 32; d > 0; d /= 2) { top = fmaxf(top, __shfl_xor(top, d)); }
  if (tid % 64 == 0) { s_part[tid / 64] = top; }
  __syncthreads();
  top              = fmaxf(fmaxf(s_part[0], s_part[1]), fmaxf(s_part[2], s_part[3]));
  const float base = top == -INFINITY ? 0.0f : top;
  __syncthreads();
  float total = 0.0f;
  constexpr int kColumns = 16;  // of a thread: up to 4,096 in all
  float acc[kColumns] = {};
  for (int64_t j0 = 0; j0 < a.k; j0 += kThreads) {
    const int64_t j = j0 + tid;
    float p         = 0.0f;
    int64_t at      = -1;
    if (j < a.k) {
      const int64_t id = a.ids[row * a.k + j];
      if (id >= 0 && id < a.n) {
        int64_t page = 0, slot = id;
        if (a.pages.table != nullptr) {
          page = a.pages.table[id / a.pages.page];
          slot = id % a.pages.page;
          if (page >= a.pages.n_pages) { page = -1; }
        }
        if (page >= 0) {
          at = page * a.v_page + slot * a.v_slot + g * a.v_head;
          p  = expf(__builtin_fmaf(s[j], a.scale, -base));
        }
      }
    }
    s_p[tid] = p;
    s_v[tid] = p == 0.0f ? -1 : at;
    __syncthreads();
    for (int i = 0; i < kThreads; ++i) {
      if (s_v[i] < 0) { continue; }
      total += s_p[i];
      const T* v = static_cast<const T*>(a.v) + s_v[i];
#pragma unroll
      for (int c = 0; c < kColumns; ++c) {
        if (tid + c * kThreads < a.vdim) { acc[c] = __builtin_fmaf(s_p[i], float(v[tid + c * kThreads]), acc[c]); }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    const int i = tid + c * kThreads;
    if (i < a.vdim) { static_cast<T*>(a.out)[row * a.vdim + i] = T(total > 0.0f ? acc[c] / total : total); }
  }
  if (tid == 0 && a.lse != nullptr) { a.lse[row] = total == 0.0f ? -INFINITY : top + logf(total); }
}

}  // namespace

size_t select_workspace(elem, select_args const&) { return 0; }

void select(elem type, select_args const& a, hipStream_t stream)
{
  const dim3 grid(uint32_t(a.heads * a.queries));
  switch (type) {
    case elem::f32: select_kernel<float><<<grid, kThreads, 0, stream>>>(a); break;
    case elem::f16: select_kernel<f16_t><<<grid, kThreads, 0, stream>>>(a); break;
    case elem::bf16: select_kernel<bf16_t><<<grid, kThreads, 0, stream>>>(a); break;
  }
}

}  // namespace certex_amd::attention
