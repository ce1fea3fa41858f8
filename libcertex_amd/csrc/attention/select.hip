// Attention over a selected top k: the scores are given (a key cache returns them with the ids), so
// no key is read again. out = sum_j p_j v[id_j] / sum_j p_j, p_j = 2^(x_j - m), x_j = scale log2(e) s_j.
//
// What bounds it: gathers of value rows (256 bytes of 128 bfloat16 columns), one multiplication per element read.
// A wave takes 64 ids at a time: each lane the weight and the row of one; then 16 bytes of a row per lane, as many
// rows at once as 64 lanes hold, 16 loads in flight. The running maximum is per wave. Workgroups of few
// queries split a query's ids, and a second launch joins the parts.
#include "../kernels/lanes.hpp"
#include "attention.hpp"
#include "elements.hpp"

#include <algorithm>

namespace certex_amd::attention {
namespace {

constexpr int kWaves   = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kIds     = 64;              // ids of a wave's step
constexpr int kStep    = kIds * kWaves;   // of a workgroup's
constexpr int kFill    = 1024;            // workgroups that fill the chip
constexpr float kLog2e = 1.44269504088896340736f;

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

struct select_plan {
  int32_t splits;   // of a query's ids
  int64_t per;      // ids of a split, a multiple of kStep
  int64_t work;     // queries x splits
  float scale2;     // scale log2(e)
  float* part_out;  // [work][vdim]
  float* part_max;  // [work]
  float* part_sum;
};

template <typename T>
__device__ __forceinline__ float element(u32x4 v, int i)
{
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(float, uint32_t(v[i]));
  } else if constexpr (std::is_same_v<T, bf16_t>) {
    return __builtin_bit_cast(float, i % 2 == 0 ? v[i / 2] << 16 : v[i / 2] & 0xffff0000u);
  } else {
    return float(__builtin_bit_cast(_Float16, uint16_t(v[i / 2] >> (i % 2 * 16))));
  }
}

/** L lanes read a row, 16 bytes each; TINY: rows of fewer than 8 elements, read one by one. */
template <typename T, int L, bool TINY>
__global__ __launch_bounds__(kThreads) void select_kernel(select_args a, select_plan plan)
{
  constexpr int E     = 16 / sizeof(T);  // elements of a lane
  constexpr int kOnce = 64 / L;          // rows that one load reads
  constexpr int kLoads = kIds / kOnce;   // of a step
  constexpr int kBatch = kLoads < 16 ? kLoads : 16;
  __shared__ float s_p[kWaves][kIds];
  __shared__ int64_t s_at[kWaves][kIds];
  __shared__ float s_out[kWaves][L * E];
  __shared__ float s_max[kWaves], s_sum[kWaves];
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  // consecutive workgroups go to the 8 dies in turn: each die takes a range of queries, whose heads
  // share values in its cache
  const int64_t each = (plan.work + 7) / 8, work = int64_t(blockIdx.x % 8) * each + blockIdx.x / 8;
  if (work >= plan.work) { return; }
  const int64_t row = work / plan.splits, first = (work - row * plan.splits) * plan.per;
  const int64_t end = min(a.k, first + plan.per);
  const int g       = int(row / a.queries) / (a.heads / a.kv_heads);
  const T* values   = static_cast<const T*>(a.v) + g * a.v_head;
  const float* s    = a.scores + row * a.k;
  const int col     = lane % L * E;
  const int off     = TINY ? col : min(col, a.vdim - E);

  float top = -INFINITY, total = 0.0f, acc[E] = {};
  for (int64_t j0 = first + wave * kIds; j0 < end; j0 += kStep) {
    const int64_t j = j0 + lane;
    float x         = -INFINITY;
    int64_t at      = 0;
    if (j < end) {
      const int64_t id = a.ids[row * a.k + j];
      const float raw  = s[j];
      if (id >= 0 && id < a.n && raw != -INFINITY) {
        if (a.pages.table == nullptr) {
          at = id * a.v_slot;
          x  = raw * plan.scale2;
        } else {
          const uint32_t e   = uint32_t(id) / uint32_t(a.pages.page);
          const int32_t page = a.pages.table[e];
          if (uint32_t(page) < uint32_t(a.pages.n_pages)) {
            at = page * a.v_page + (id - int64_t(e) * a.pages.page) * a.v_slot;
            x  = raw * plan.scale2;
          }
        }
      }
    }
    const float high  = lanes::max<64>(x);
    const float grown = fmaxf(top, high);
    if (grown > top) {
      const float keep = __builtin_amdgcn_exp2f(top - grown);
      total *= keep;
#pragma unroll
      for (int i = 0; i < E; ++i) { acc[i] *= keep; }
      top = grown;
    }
    const float p       = __builtin_amdgcn_exp2f(x - (top == -INFINITY ? 0.0f : top));
    const uint64_t some = __ballot(p != 0.0f);  // NaN too
    if (some == 0) { continue; }
    total += p;
    // what weighs nothing reads the row of an id that does: its own may hold anything
    const int64_t other = __shfl(at, __builtin_ctzll(some));
    s_p[wave][lane]     = p;
    s_at[wave][lane]    = p != 0.0f ? at : other;
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
    for (int i0 = 0; i0 < kLoads; i0 += kBatch) {
      u32x4 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const T* from = values + s_at[wave][(i0 + i) * kOnce + lane / L] + off;
        if constexpr (TINY) {
          T e[E];
#pragma unroll
          for (int c = 0; c < E; ++c) { e[c] = col + c < a.vdim ? from[c] : T(0.0f); }
          __builtin_memcpy(&v[i], e, 16);
        } else {
          __builtin_memcpy(&v[i], __builtin_assume_aligned(from, sizeof(T)), 16);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float w = s_p[wave][(i0 + i) * kOnce + lane / L];
#pragma unroll
        for (int c = 0; c < E; ++c) { acc[c] = __builtin_fmaf(w, element<T>(v[i], c), acc[c]); }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  total = lanes::sum<64>(total);
  // the row groups of the wave, then the waves
#pragma unroll
  for (int c = 0; c < E; ++c) {
    const auto add = [](float u, float w) { return u + w; };
    if constexpr (L <= 8) { acc[c] = add(acc[c], lanes::exchange<8>(acc[c])); }
    if constexpr (L <= 16) { acc[c] = lanes::fold16(acc[c], add); }
    if constexpr (L <= 32) { acc[c] = lanes::fold32(acc[c], add); }
  }
  if (lane < L) {
#pragma unroll
    for (int c = 0; c < E; ++c) {
      // a piece shifted back to the row's end holds columns of an earlier one again: the same sums
      if (off + c < L * E) { s_out[wave][off + c] = acc[c]; }
    }
  }
  if (lane == 0) {
    s_max[wave] = top;
    s_sum[wave] = total;
  }
  __syncthreads();
  float m = s_max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) { m = fmaxf(m, s_max[w]); }
  float f[kWaves], sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = factor_of(s_max[w], m);
    sum += f[w] * s_sum[w];
  }
  for (int i = tid; i < a.vdim; i += kThreads) {
    float out = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) { out += f[w] * s_out[w][i]; }
    if (plan.splits == 1) {
      static_cast<T*>(a.out)[row * a.vdim + i] = T(sum == 0.0f ? 0.0f : out / sum);
    } else {
      plan.part_out[work * a.vdim + i] = out;
    }
  }
  if (tid == 0) {
    if (plan.splits > 1) {
      plan.part_max[work] = m;
      plan.part_sum[work] = sum;
    } else if (a.lse != nullptr) {
      a.lse[row] = sum == 0.0f ? -INFINITY : (m + __builtin_log2f(sum)) / kLog2e;
    }
  }
}

/** One workgroup per query: joins its splits in order. */
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(select_args a, select_plan plan)
{
  const int64_t row = blockIdx.x, w0 = row * plan.splits;
  float m = -INFINITY;
  for (int w = 0; w < plan.splits; ++w) { m = fmaxf(m, plan.part_max[w0 + w]); }
  for (int i = threadIdx.x; i < a.vdim; i += kThreads) {
    float sum = 0.0f, out = 0.0f;
#pragma unroll 8
    for (int w = 0; w < plan.splits; ++w) {
      const float f = factor_of(plan.part_max[w0 + w], m);
      sum += f * plan.part_sum[w0 + w];
      out += f * plan.part_out[(w0 + w) * a.vdim + i];
    }
    static_cast<T*>(a.out)[row * a.vdim + i] = T(sum == 0.0f ? 0.0f : out / sum);
    if (i == 0 && a.lse != nullptr) { a.lse[row] = sum == 0.0f ? -INFINITY : (m + __builtin_log2f(sum)) / kLog2e; }
  }
}

auto plan_of(select_args const& a) -> select_plan
{
  select_plan p{};
  const int64_t rows = a.heads * a.queries, steps = std::max<int64_t>(1, (a.k + kStep - 1) / kStep);
  // enough workgroups to fill the chip, each of at least one step
  const int64_t splits = std::clamp<int64_t>((kFill + rows - 1) / std::max<int64_t>(1, rows), 1, steps);
  const int64_t each   = (steps + splits - 1) / splits;
  p.splits             = int32_t((steps + each - 1) / each);
  p.per                = each * kStep;
  p.work               = rows * p.splits;
  p.scale2             = a.scale * kLog2e;
  return p;
}

}  // namespace

size_t select_workspace(elem, select_args const& a)
{
  const auto p = plan_of(a);
  return p.splits == 1 ? 0 : sizeof(float) * p.work * (a.vdim + 2);
}

void select(elem type, select_args const& a, hipStream_t stream)
{
  select_plan p = plan_of(a);
  p.part_out    = static_cast<float*>(a.workspace);
  p.part_max    = p.part_out + p.work * a.vdim;
  p.part_sum    = p.part_max + p.work;
  const dim3 grid(uint32_t((p.work + 7) / 8 * 8));
  const auto launched = [&](auto tag) {
    using T         = decltype(tag);
    const int bytes = a.vdim * int(sizeof(T));
    if (a.vdim < 8) {
      select_kernel<T, 8, true><<<grid, kThreads, 0, stream>>>(a, p);
    } else if (bytes <= 128) {
      select_kernel<T, 8, false><<<grid, kThreads, 0, stream>>>(a, p);
    } else if (bytes <= 256) {
      select_kernel<T, 16, false><<<grid, kThreads, 0, stream>>>(a, p);
    } else if (bytes <= 512) {
      select_kernel<T, 32, false><<<grid, kThreads, 0, stream>>>(a, p);
    } else if constexpr (sizeof(T) == 4) {
      select_kernel<T, 64, false><<<grid, kThreads, 0, stream>>>(a, p);
    }
    if (p.splits > 1) { join_kernel<T><<<dim3(uint32_t(a.heads * a.queries)), kThreads, 0, stream>>>(a, p); }
  };
  switch (type) {
    case elem::f32: launched(float{}); break;
    case elem::f16: launched(f16_t{}); break;
    case elem::bf16: launched(bf16_t{}); break;
  }
}

}  // namespace certex_amd::attention
