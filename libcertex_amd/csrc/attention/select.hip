// Attention over a selected top k: the scores are given (a key cache returns them with the ids), so
// no key is read again. out = sum_j p_j v[id_j] / sum_j p_j, p_j = 2^(scale log2(e) (s_j - m)), m the largest score
// (the smallest, where scale < 0). The scores are subtracted before they are scaled: what is rounded is their distance
// from m, however far from 0 they are, and scores of the type's lowest value among themselves stay at distance 0.
//
// What bounds it: gathers of value rows (256 bytes of 128 bfloat16 columns), one multiplication per element read.
// A wave takes 64 ids at a time: each lane the weight and the row of one; then 16 bytes of a row per lane, as many
// rows at once as 64 lanes hold, 16 loads in flight. The running maximum is per wave. Workgroups of few
// queries split a query's ids, and a second launch joins the parts.
//
// Measured (32 query heads, 8 value heads of 131,072 rows of 128 bfloat16, k = 2,048): one query a head, 17 MB: 8.2 us
// and 2.4 us of the join; 16 queries a head 44 us, 268 MB of gathers at 6.1 TB/s; 64 queries a head, taken by
// ranges of rows, 116 us a pass where 1.07 GB of gathers as they come take 154: ids sorted in 25 us, rows gathered in 91
// (11.8 TB/s, 72% of them from the dies' caches; values that fit there are gathered at 18 TB/s), parts added in 5.
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
// Workgroups that fill the chip: fewer queries than this split their ids. Measured, 32 heads, k = 2,048, with 1, 256,
// 1,024 and 4,096: one query a head 35, 10.8, 10.9 and 10.8 us; 8 queries 50, 50, 29 and 31; 32 queries 81 (1,024), 88 (4,096).
constexpr int kFill    = 1024;

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

struct select_plan {
  int32_t splits;   // of a query's ids
  int64_t per;      // ids of a split, a multiple of kStep
  int64_t work;     // queries x splits
  score_scale scale;
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

/** Where an id's row begins (elements from its head's values), or -1. */
__device__ __forceinline__ int64_t row_of(select_args const& a, int64_t id)
{
  if (id < 0 || id >= a.n) { return -1; }
  if (a.pages.table == nullptr) { return id * a.v_slot; }
  const uint32_t e   = uint32_t(id) / uint32_t(a.pages.page);
  const int32_t page = a.pages.table[e];
  if (uint32_t(page) >= uint32_t(a.pages.n_pages)) { return -1; }
  return page * a.v_page + (id - int64_t(e) * a.pages.page) * a.v_slot;
}

/** Consecutive workgroups go to the 8 dies in turn: each die takes a range of queries, whose heads share values in
 *  its cache. */
__device__ __forceinline__ int64_t work_of_block(select_plan const& plan)
{
  return int64_t(blockIdx.x % 8) * ((plan.work + 7) / 8) + blockIdx.x / 8;
}

/** Adds the row groups of a wave and the waves, and writes the query's output or its part. L lanes hold a row, lane l its
 *  elements off..off + E - 1. */
template <typename T, int L, int E>
__device__ __forceinline__ void finish(select_args const& a, select_plan const& plan, int64_t work, int off, float top,
                                       float total, float* acc, float (*s_out)[L * E])
{
  __shared__ float s_max[kWaves], s_sum[kWaves];
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  const int64_t row = work / plan.splits;
  total             = lanes::sum<64>(total);
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
    f[w] = factor_of(plan.scale, s_max[w], m);
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
      a.lse[row] = lse_of(plan.scale, m, sum);
    }
  }
}

/** L lanes read a row, 16 bytes each; TINY: rows of fewer than 8 elements, read one by one. */
template <typename T, int L, bool TINY>
__global__ __launch_bounds__(kThreads) void select_kernel(select_args a, select_plan plan)
{
  constexpr int E      = 16 / sizeof(T);  // elements of a lane
  constexpr int kOnce  = 64 / L;          // rows that one load reads
  constexpr int kLoads = kIds / kOnce;    // of a step
  constexpr int kBatch = kLoads < 16 ? kLoads : 16;
  __shared__ float s_p[kWaves][kIds];
  __shared__ int64_t s_at[kWaves][kIds];
  __shared__ float s_out[kWaves][L * E];
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  const int64_t work = work_of_block(plan);
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
      const float raw = s[j];
      at              = row_of(a, a.ids[row * a.k + j]);
      if (at >= 0 && raw != -INFINITY) { x = raw * plan.scale.sign; }
    }
    const float high  = lanes::max<64>(x);
    const float grown = fmaxf(top, high);
    if (grown > top) {
      const float keep = weight_of(plan.scale, top, grown);
      total *= keep;
#pragma unroll
      for (int i = 0; i < E; ++i) { acc[i] *= keep; }
      top = grown;
    }
    const float p       = weight_of(plan.scale, x, top == -INFINITY ? 0.0f : top);
    const bool counts   = x != -INFINITY;  // however little it weighs
    const uint64_t some = __ballot(counts);
    if (some == 0) { continue; }
    total += p;
    // what does not count reads the row of an id that does: its own may hold anything
    const int64_t other = __shfl(at, __builtin_ctzll(some));
    s_p[wave][lane]     = p;
    s_at[wave][lane]    = counts ? at : other;
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
  finish<T, L, E>(a, plan, work, off, top, total, acc, s_out);
}

// ---- many queries per head ----
//
// Where a head's queries select its rows several times over, the rows' second and later reads should meet the first
// one's in the die's cache. So the ids of every query are put in order of ranges of the head's rows first, their
// weights final (sort_kernel). Then the ranges are taken one after the other: a wave per query and range, dealt to a die
// range by range, so that its waves read from a window of a few ranges (phase_kernel). A query's outputs of the
// ranges are added last (sum_kernel).

constexpr int kMaxRanges = 64;

struct phase_plan {
  int32_t ranges;
  int64_t rows;     // queries of all heads
  float per_n;      // ranges / n
  score_scale scale;
  uint2* list;      // [rows][k]: row offset, weight
  int32_t* starts;  // [rows][ranges + 1]
  float* part;      // [ranges][rows][vdim]
};

/**
 * One workgroup per query: weights p / sum p, and the ids sorted by range: a counting sort, stable, so that the sums' order
 * does not depend on timing. Every wave sorts a quarter of the ids with its own counters.
 */
__global__ __launch_bounds__(kThreads) void sort_kernel(select_args a, phase_plan plan)
{
  constexpr int kBlock = 8;  // ids of a lane that are in flight, and kept when they are all of them
  __shared__ int32_t s_count[kWaves][kMaxRanges];
  __shared__ float s_part[2][kWaves];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const int64_t row = blockIdx.x;
  const float* s    = a.scores + row * a.k;
  const int64_t per = (a.k + kThreads - 1) / kThreads * 64;  // ids of a wave
  const int64_t begin = min(a.k, wave * per), end = min(a.k, begin + per);
  s_count[wave][lane] = 0;

  uint32_t at[kBlock], range[kBlock];
  float x[kBlock];
  const auto take = [&](int64_t j0) {
    int64_t id[kBlock];
#pragma unroll
    for (int i = 0; i < kBlock; ++i) {
      const int64_t j = j0 + i * 64 + lane;
      id[i]           = j < end ? a.ids[row * a.k + j] : -1;
      x[i]            = j < end ? s[j] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kBlock; ++i) {
      const int64_t to = row_of(a, id[i]);
      at[i]            = uint32_t(to);
      range[i]         = min(uint32_t(float(max(id[i], int64_t(0))) * plan.per_n), uint32_t(plan.ranges - 1));
      x[i]             = to >= 0 && x[i] != -INFINITY ? x[i] * plan.scale.sign : -INFINITY;
    }
  };

  float top = -INFINITY, total = 0.0f;
  for (int64_t j0 = begin; j0 < end; j0 += 64 * kBlock) {
    take(j0);
    float grown = top;
#pragma unroll
    for (int i = 0; i < kBlock; ++i) { grown = fmaxf(grown, x[i]); }
    total *= factor_of(plan.scale, top, grown);
    top = grown;
#pragma unroll
    for (int i = 0; i < kBlock; ++i) {
      total += weight_of(plan.scale, x[i], top == -INFINITY ? 0.0f : top);
      if (x[i] != -INFINITY) { atomicAdd(&s_count[wave][range[i]], 1); }
    }
  }
  float high = lanes::max<64>(top);
  if (lane == 0) { s_part[0][wave] = high; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) { high = fmaxf(high, s_part[0][w]); }
  total = lanes::sum<64>(factor_of(plan.scale, top, high) * total);
  if (lane == 0) { s_part[1][wave] = total; }
  // a wave's counters become where its ids of each range begin
  int32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int32_t n = s_count[w][lane];
    before += w < wave ? n : 0;
    all += n;
  }
  const int32_t base = lanes::scan_incl(all) - all;
  __syncthreads();
  s_count[wave][lane] = base + before;
  if (wave == 0) {
    int32_t* starts = plan.starts + row * (plan.ranges + 1);
    if (lane <= plan.ranges) { starts[lane] = base; }
    if (lane == 63 && plan.ranges == kMaxRanges) { starts[kMaxRanges] = base + all; }
  }
  total               = (s_part[1][0] + s_part[1][1]) + (s_part[1][2] + s_part[1][3]);
  const float per_sum = 1.0f / total;
  const float from    = high == -INFINITY ? 0.0f : high;
  if (tid == 0 && a.lse != nullptr) { a.lse[row] = lse_of(plan.scale, high, total); }
  uint2* list = plan.list + row * a.k;
  for (int64_t j0 = begin; j0 < end; j0 += 64 * kBlock) {
    if (end - begin > 64 * kBlock) { take(j0); }
#pragma unroll
    for (int i = 0; i < kBlock; ++i) {
      const bool in = x[i] != -INFINITY;
      uint64_t same = __ballot(in);
#pragma unroll
      for (int bit = 0; bit < 6; ++bit) {
        const bool one     = range[i] >> bit & 1;
        const uint64_t set = __ballot(one);
        same &= one ? set : ~set;
      }
      const uint32_t rank = __builtin_amdgcn_mbcnt_hi(uint32_t(same >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(same), 0u));
      if (in) {
        const int32_t to = s_count[wave][range[i]] + int32_t(rank);
        const float p    = weight_of(plan.scale, x[i], from) * per_sum;
        list[to]         = make_uint2(at[i], __builtin_bit_cast(uint32_t, p));
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (in && rank == 0) { s_count[wave][range[i]] += int32_t(__popcll(same)); }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

/** One wave per query and range, 64 ids at a time: the die's part of the queries, range by range. */
template <typename T, int L>
__global__ __launch_bounds__(kThreads) void phase_kernel(select_args a, phase_plan plan)
{
  constexpr int E      = 16 / sizeof(T);
  constexpr int kOnce  = 64 / L;
  constexpr int kLoads = kIds / kOnce;
  constexpr int kBatch = kLoads < 16 ? kLoads : 16;
  __shared__ uint2 s_list[kWaves][kIds];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int64_t each  = (plan.rows + 8 * kWaves - 1) / (8 * kWaves);  // workgroups of a range on a die
  const int64_t here  = blockIdx.x / 8, range = here / each;
  const int64_t row   = (int64_t(blockIdx.x % 8) * each + here - range * each) * kWaves + wave;
  if (row >= plan.rows) { return; }
  const int g       = int(row / a.queries) / (a.heads / a.kv_heads);
  const int off     = min(lane % L * E, a.vdim - E);
  const T* values   = static_cast<const T*>(a.v) + g * a.v_head + off;
  const int32_t* at = plan.starts + row * (plan.ranges + 1) + range;
  const int32_t begin = at[0], end = at[1];
  const uint2* list   = plan.list + row * a.k;
  float acc[E]        = {};
  uint2 mine          = begin < end ? list[min(begin + lane, end - 1)] : make_uint2(0u, 0u);
  for (int32_t j0 = begin; j0 < end; j0 += kIds) {
    // what is past the range: its last row again, of weight 0
    s_list[wave][lane] = make_uint2(mine.x, j0 + lane < end ? mine.y : 0u);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int loads = min(kLoads, (end - j0 + kOnce - 1) / kOnce);
    mine            = list[min(j0 + kIds + lane, end - 1)];
#pragma unroll
    for (int i0 = 0; i0 < kLoads; i0 += kBatch) {
      if (i0 >= loads) { break; }
      u32x4 v[kBatch];
      float p[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint2 e = s_list[wave][min(i0 + i, loads - 1) * kOnce + lane / L];
        p[i]          = i0 + i < loads ? __builtin_bit_cast(float, e.y) : 0.0f;
        if (i0 + i < loads) { __builtin_memcpy(&v[i], __builtin_assume_aligned(values + e.x, sizeof(T)), 16); }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (i0 + i < loads) {
#pragma unroll
          for (int c = 0; c < E; ++c) { acc[c] = __builtin_fmaf(p[i], element<T>(v[i], c), acc[c]); }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
#pragma unroll
  for (int c = 0; c < E; ++c) {
    const auto add = [](float u, float w) { return u + w; };
    if constexpr (L <= 8) { acc[c] = add(acc[c], lanes::exchange<8>(acc[c])); }
    if constexpr (L <= 16) { acc[c] = lanes::fold16(acc[c], add); }
    if constexpr (L <= 32) { acc[c] = lanes::fold32(acc[c], add); }
  }
  if (lane < L && lane * E < a.vdim) {
    float* to = plan.part + (range * plan.rows + row) * a.vdim + off;
#pragma unroll
    for (int c = 0; c < E; ++c) { to[c] = acc[c]; }
  }
}

/** out = the sum of the ranges' parts, in order; a thread per column. */
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_kernel(select_args a, phase_plan plan)
{
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x, n = plan.rows * a.vdim;
  if (i >= n) { return; }
  float out = 0.0f;
#pragma unroll 16
  for (int r = 0; r < plan.ranges; ++r) { out += plan.part[r * n + i]; }
  static_cast<T*>(a.out)[i] = T(out);
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
      const float f = factor_of(plan.scale, plan.part_max[w0 + w], m);
      sum += f * plan.part_sum[w0 + w];
      out += f * plan.part_out[(w0 + w) * a.vdim + i];
    }
    static_cast<T*>(a.out)[row * a.vdim + i] = T(sum == 0.0f ? 0.0f : out / sum);
    if (i == 0 && a.lse != nullptr) { a.lse[row] = lse_of(plan.scale, m, sum); }
  }
}

constexpr int64_t kDieCache  = int64_t(4) << 20;  // bytes
constexpr int64_t kRangeBytes = int64_t(2) << 20;

/**
 * In how many ranges of rows the ids are taken (0: as they come): where the values that a die's queries read exceed its
 * cache and the queries select them three times over, with enough ids of a query in a range. Measured, as they come
 * and by ranges, 32 heads, 131,072 rows of 128 columns, k = 2,048: 64 queries a head (4 times over) 154 and 117 us, float32
 * 290 and 197 us; 32 queries 75 and 78 us; 16 queries 44 and 51 us. Ranges of 1, 2, 4 and 8 MB: 151, 117, 120 and 141 us
 * (smaller ones write more parts, larger ones leave the cache). Offsets are kept in 32 bits.
 */
int ranges_of(elem type, select_args const& a)
{
  const int64_t bytes    = a.vdim * elem_bytes(type), rows = a.heads * a.queries;
  const int64_t farthest = a.pages.table != nullptr
                             ? (a.pages.n_pages - 1) * a.v_page + (a.pages.page - 1) * a.v_slot
                             : (a.n - 1) * a.v_slot;
  const int64_t die      = std::max(1, a.kv_heads / 8) * a.n * bytes;
  const int64_t ranges   = std::min<int64_t>(kMaxRanges, (die + kRangeBytes - 1) / kRangeBytes);
  const bool fits        = a.vdim >= 8 && bytes <= 512 && farthest < (int64_t(1) << 32) && rows <= (int64_t(1) << 18) &&
                    rows * a.k <= (int64_t(1) << 28);
  const bool pays = die > kDieCache && rows >= 256 && a.k * (rows / a.kv_heads) >= 3 * a.n && a.k >= 32 * ranges;
  return fits && pays ? int(ranges) : 0;
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
  p.scale              = scale_of(a.scale);
  return p;
}

}  // namespace

size_t select_workspace(elem type, select_args const& a)
{
  if (const int ranges = ranges_of(type, a)) {
    const int64_t rows = a.heads * a.queries;
    return sizeof(uint2) * rows * a.k + sizeof(int32_t) * rows * (ranges + 1) + sizeof(float) * ranges * rows * a.vdim;
  }
  const auto p = plan_of(a);
  return p.splits == 1 ? 0 : sizeof(float) * p.work * (a.vdim + 2);
}

void select(elem type, select_args const& a, hipStream_t stream)
{
  if (const int ranges = ranges_of(type, a)) {
    phase_plan p{};
    p.ranges = ranges;
    p.rows   = a.heads * a.queries;
    p.per_n  = float(ranges) / float(a.n);
    p.scale  = scale_of(a.scale);
    p.list   = static_cast<uint2*>(a.workspace);
    p.starts = reinterpret_cast<int32_t*>(p.list + p.rows * a.k);
    p.part   = reinterpret_cast<float*>(p.starts + p.rows * (ranges + 1));
    const int64_t each = (p.rows + 8 * kWaves - 1) / (8 * kWaves);
    const dim3 phases(uint32_t(each * 8 * ranges)), sums(uint32_t((p.rows * a.vdim + kThreads - 1) / kThreads));
    sort_kernel<<<dim3(uint32_t(p.rows)), kThreads, 0, stream>>>(a, p);
    const auto launched = [&](auto tag) {
      using T         = decltype(tag);
      const int bytes = a.vdim * int(sizeof(T));
      if (bytes <= 128) {
        phase_kernel<T, 8><<<phases, kThreads, 0, stream>>>(a, p);
      } else if (bytes <= 256) {
        phase_kernel<T, 16><<<phases, kThreads, 0, stream>>>(a, p);
      } else {
        phase_kernel<T, 32><<<phases, kThreads, 0, stream>>>(a, p);
      }
      sum_kernel<T><<<sums, kThreads, 0, stream>>>(a, p);
    };
    switch (type) {
      case elem::f32: launched(float{}); break;
      case elem::f16: launched(f16_t{}); break;
      case elem::bf16: launched(bf16_t{}); break;
    }
    return;
  }
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
