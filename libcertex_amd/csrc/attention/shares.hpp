// How the attention of one new token per sequence is dealt: the tiles of all sequences, one after the other, in equal shares
// of workgroups, computed on the device from the lengths; and the join of sequences that shares cut.
#pragma once

#include "../kernels/lanes.hpp"
#include "attention.hpp"
#include "elements.hpp"
#include "tiles.hpp"

#include <algorithm>

namespace certex_amd::attention {
namespace {  // its kernels belong to each source that launches them

constexpr int kWaves   = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows    = 16;   // query heads of a product
constexpr int kUnits   = 256;  // compute units
constexpr int kMaxShares = 2 * kUnits;

struct attend_plan {
  divisor page_groups;  // lane groups' positions per page
  int32_t row_tiles;    // products of 16 query heads per key head
  int32_t group;        // query heads per key head
  int32_t tables;       // key heads x row_tiles: table t is key head t % kv_heads, product t / kv_heads
  int32_t shares;       // of a table's tiles, at most
  int32_t halve;        // half as many shares where each of those has this many tiles or more (0: never)
  bool one_die;         // the tables of a share run on one die
  score_scale scale;
  float lift;           // sums are 2^lift times themselves
  float slack;          // kSlack in scores
  float* part_out;      // [tables][2 shares][kRows][vdim]
  float* part_max;      // [tables][2 shares][kRows]
  float* part_sum;
};

/** Positions [begin, end) of a sequence, and its tiles of TILE from begin rounded down to 8. */
struct span {
  int32_t begin, end, tiles;
};

template <int TILE>
__device__ __forceinline__ span span_of(attend_args const& a, int64_t b)
{
  int64_t end = a.lengths[b];
  end         = end < 0 ? 0 : min(end, int64_t(a.pages.width) * a.pages.page);
  if (a.pages.n_pages == 0) { end = 0; }
  const int64_t begin = a.window > 0 && end > a.window ? end - a.window : 0;
  return {int32_t(begin), int32_t(end), int32_t((end - (begin & ~int64_t(7)) + TILE - 1) / TILE)};
}

/** The shares of a table: share w takes the tiles [w tiles / n, (w + 1) tiles / n) of all sequences'. */
struct shares {
  int64_t tiles, n;
  __device__ __forceinline__ int64_t first(int64_t w) const { return w * tiles / n; }
  __device__ __forceinline__ int64_t of(int64_t tile) const { return ((tile + 1) * n - 1) / tiles; }
};

__device__ __forceinline__ shares split(attend_plan const& p, int64_t tiles)
{
  const int64_t half = p.shares / 2;
  return {tiles, p.halve > 0 && half > 0 && tiles >= half * p.halve ? half : min(int64_t(p.shares), tiles)};
}

template <int TILE>
__device__ __forceinline__ shares shares_of(attend_args const& a, attend_plan const& p)
{
  int64_t mine = 0;
  for (int64_t b = threadIdx.x % 64; b < a.pages.sequences; b += 64) { mine += span_of<TILE>(a, b).tiles; }
  return split(p, lanes::sum<64>(mine));
}

/**
 * One workgroup per sequence and query head: joins the partials of a sequence that shares cut. Their
 * factors first, in LDS; then a thread per column and part of the partials.
 */
template <typename T, int THREADS, int TILE>
__global__ __launch_bounds__(THREADS) void join_kernel(attend_args a, attend_plan plan)
{
  __shared__ float s_factor[kMaxShares];
  __shared__ float s_out[THREADS];
  __shared__ float s_part[THREADS / 64];
  const int h = blockIdx.x, tid = threadIdx.x;
  const int64_t b = blockIdx.y;
  const int kv = h / plan.group, in_group = h - kv * plan.group;
  const int table = in_group / kRows * a.kv_heads + kv, row = in_group % kRows;
  const int tiles = span_of<TILE>(a, b).tiles;
  int64_t before = 0, all = 0;
  for (int64_t i = tid % 64; i < a.pages.sequences; i += 64) {
    const int n = span_of<TILE>(a, i).tiles;
    before += i < b ? n : 0;
    all += n;
  }
  before = lanes::sum<64>(before);
  all    = lanes::sum<64>(all);
  if (tiles == 0) { return; }
  const shares sh = split(plan, all);
  const int64_t w0 = sh.of(before), w1 = sh.of(before + tiles - 1);
  if (w0 == w1) { return; }
  const int n = int(w1 - w0) + 1;
  // the later shares begin inside the sequence: their first slot
  const int64_t slot0 = 2 * w0 + (sh.first(w0) == before ? 0 : 1);
  const auto slot     = [&](int i) {
    return (int64_t(table) * plan.shares * 2 + (i == 0 ? slot0 : 2 * (w0 + i))) * kRows + row;
  };

  float m = -INFINITY;
  for (int i = tid; i < n; i += THREADS) {
    s_factor[i] = plan.part_max[slot(i)];
    m           = fmaxf(m, s_factor[i]);
  }
  m = lanes::max<64>(m);
  if (tid % 64 == 0) { s_part[tid / 64] = m; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) { m = fmaxf(m, s_part[w]); }
  __syncthreads();
  float sum = 0.0f;
  for (int i = tid; i < n; i += THREADS) {
    s_factor[i] = factor_of(plan.scale, s_factor[i], m);
    sum += s_factor[i] * plan.part_sum[slot(i)];
  }
  sum = lanes::sum<64>(sum);
  if (tid % 64 == 0) { s_part[tid / 64] = sum; }
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) { sum += s_part[w]; }

  const int64_t at = b * a.heads + h;
  const int cols = min(THREADS, a.vdim <= 64 ? 64 : a.vdim <= 128 ? 128 : 256);
  const int part = tid / cols, parts = THREADS / cols;
  for (int col0 = 0; col0 < a.vdim; col0 += cols) {  // more than once only with one part
    const int col = col0 + tid % cols;
    float acc     = 0.0f;
    if (col < a.vdim) {
#pragma unroll 8
      for (int i = part; i < n; i += parts) { acc = __builtin_fmaf(s_factor[i], plan.part_out[slot(i) * a.vdim + col], acc); }
    }
    if (parts > 1) {
      s_out[tid] = acc;
      __syncthreads();
    }
    if (part == 0 && col < a.vdim) {
      for (int i = 1; i < parts; ++i) { acc += s_out[i * cols + tid]; }
      static_cast<T*>(a.out)[at * a.vdim + col] = T(sum == 0.0f ? 0.0f : acc / sum);
    }
  }
  if (tid == 0 && a.lse != nullptr) {
    a.lse[at] = lse_of(plan.scale, m, sum, plan.lift);
  }
}

int row_tiles_of(attend_args const& a) { return (a.heads / a.kv_heads + kRows - 1) / kRows; }

/** Most positions of a sequence, from begin rounded down to 8. */
int64_t longest_of(attend_args const& a)
{
  const int64_t most = int64_t(a.pages.width) * a.pages.page;
  return a.window > 0 && a.window < most ? std::min(most, a.window + 7) : most;
}

/** Shares of a table: one workgroup per place on the chip over all tables, two rounds where that would leave places
 *  empty; no more than there can be tiles. */
int shares_for(attend_args const& a, int tile, int per_unit)
{
  const int64_t places = int64_t(kUnits) * per_unit, tables = int64_t(a.kv_heads) * row_tiles_of(a);
  int64_t n = std::max<int64_t>(1, places / tables);
  if (n * tables * 4 < places * 3) { n = (2 * places + tables - 1) / tables; }
  return int(std::min({n, int64_t(kMaxShares), std::max<int64_t>(1, a.pages.sequences * ((longest_of(a) + tile - 1) / tile))}));
}

}  // namespace
}  // namespace certex_amd::attention
