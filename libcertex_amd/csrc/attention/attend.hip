// Attention of one new token of every sequence over its pages of keys and values.
//
// out = sum_t p_t v_t / sum_t p_t with p_t = exp(scale q.k_t - m), m the largest exponent, over the
// positions t of [max(0, len - window), len). One pass over the positions keeps m, the sum and the
// output in float32, and scales the last two where m grows.
#include "attention.hpp"
#include "elements.hpp"

#include <algorithm>

namespace certex_amd::attention {
namespace {

constexpr int kThreads = 256;

/** One workgroup per sequence and query head: 256 positions at a time, one per thread. */
template <typename T>
__global__ __launch_bounds__(kThreads) void attend_kernel(attend_args a)
{
  __shared__ float s_q[kMaxHeadDim];
  __shared__ float s_p[kThreads];
  __shared__ int64_t s_v[kThreads];
  __shared__ float s_part[kThreads / 64];
  const int h = blockIdx.x, g = h / (a.heads / a.kv_heads), tid = threadIdx.x;
  const int64_t b = blockIdx.y;
  const T* q      = static_cast<const T*>(a.q) + b * a.q_seq + h * a.q_head;
  for (int i = tid; i < a.dim; i += kThreads) { s_q[i] = float(q[i]); }
  int64_t end         = a.lengths[b];
  end                 = end < 0 ? 0 : min(end, int64_t(a.pages.width) * a.pages.page);
  const int64_t begin = a.window > 0 && end > a.window ? end - a.window : 0;
  float top = -INFINITY, total = 0.0f, acc = 0.0f;
  for (int64_t t0 = begin; t0 < end; t0 += kThreads) {
    const int64_t t = t0 + tid;
    float x         = -INFINITY;
    int64_t v_at    = -1;
    __syncthreads();
    if (t < end) {
      const int32_t page = a.pages.table[b * a.pages.width + t / a.pages.page];
      if (page >= 0 && page < a.pages.n_pages) {
        const int64_t slot = t % a.pages.page;
        const T* k = static_cast<const T*>(a.k) + page * a.k_page + slot * a.k_slot + g * a.k_head;
        v_at       = page * a.v_page + slot * a.v_slot + g * a.v_head;
        float dot  = 0.0f;
        for (int i = 0; i < a.dim; ++i) { dot = __builtin_fmaf(s_q[i], float(k[i]), dot); }
        x = dot * a.scale;
      }
    }
    float m = x;
    for (int d = 32; d > 0; d /= 2) { m = fmaxf(m, __shfl_xor(m, d)); }
    if (tid % 64 == 0) { s_part[tid / 64] = m; }
    __syncthreads();
    m                 = fmaxf(fmaxf(s_part[0], s_part[1]), fmaxf(s_part[2], s_part[3]));
    const float grown = fmaxf(top, m);
    const float base  = grown == -INFINITY ? 0.0f : grown;
    const float keep  = expf(top - base);  // 0 at first
    const float p     = expf(x - base);
    s_p[tid]          = p;
    s_v[tid]          = v_at;
    float sum         = p;
    for (int d = 32; d > 0; d /= 2) { sum += __shfl_xor(sum, d); }
    __syncthreads();
    if (tid % 64 == 0) { s_part[tid / 64] = sum; }
    __syncthreads();
    total = total * keep + ((s_part[0] + s_part[1]) + (s_part[2] + s_part[3]));
    top   = grown;
    if (tid < a.vdim) {
      acc         = acc * keep;
      const int n = int(min(int64_t(kThreads), end - t0));
      for (int i = 0; i < n; ++i) {
        if (s_v[i] >= 0) { acc = __builtin_fmaf(s_p[i], float(static_cast<const T*>(a.v)[s_v[i] + tid]), acc); }
      }
    }
  }
  const int64_t row = b * a.heads + h;
  if (tid < a.vdim) { static_cast<T*>(a.out)[row * a.vdim + tid] = T(total > 0.0f ? acc / total : total); }
  if (tid == 0 && a.lse != nullptr) { a.lse[row] = total == 0.0f ? -INFINITY : top + logf(total); }
}

}  // namespace

size_t attend_workspace(elem, attend_args const&) { return 0; }

void attend(elem type, attend_args const& a, hipStream_t stream)
{
  const dim3 grid(uint32_t(a.heads), uint32_t(a.pages.sequences));
  switch (type) {
    case elem::f32: attend_kernel<float><<<grid, kThreads, 0, stream>>>(a); break;
    case elem::f16: attend_kernel<f16_t><<<grid, kThreads, 0, stream>>>(a); break;
    case elem::bf16: attend_kernel<bf16_t><<<grid, kThreads, 0, stream>>>(a); break;
  }
}

}  // namespace certex_amd::attention
