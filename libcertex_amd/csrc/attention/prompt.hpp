// Attention of the new tokens of every sequence over its pages of keys and values: prompts, and pieces of prompts.
//
// Row (i, h) of a sequence with n new tokens and `length` positions in the cache is its query at position
// p = length - n + i of query head h. It sees the positions t < length with t <= p or t < prefix, and p - t < window:
// out = sum_t w_t v_t / sum_t w_t, w_t = 2^(log2(e) (y_t - m)), y_t the score scale q.k_t or its bent form. One pass over
// the positions keeps a reference m per row, the sum and the output in float32.
//
// What bounds it: two products of 2 dim operations per row and position it sees, and about five vector
// operations per score, of which the exponential takes a quarter of the vector rate. The rows of a key head are taken
// together: the tokens' query heads that share it, 128 rows a workgroup, 32 a wave. So K and V pass from memory to
// LDS once per 128 rows, and each wave reads them from there.
// - S^T = K Q^T in products of 32 positions x 32 rows: a row is a lane's column, so that the reference, the sum and the
//   scaling are per lane; the products begin at -m, so that they end as distances from the reference.
// - The rows of S^T that a lane holds are the positions that it feeds to O^T = V^T P^T: the weights never move.
//   V is turned on its way into LDS, in the order of positions of these rows.
// - Weights of 16-bit types enter the second product as two elements, the nearest and what it leaves (bfloat16 2^-16, float16
//   2^-22 of them off at most); their sum is not rounded. One element would be 2^-8 and 2^-11 off, as much again as the output is
//   rounded, for half as many products less: 8,192 tokens 670 us where 830 is.
// - Tiles of positions are in two buffers: the next one's loads are in flight during the products.
//
// Work is dealt without reading the lengths back: the host launches as many tiles of rows as there may be, the
// kernel finds the sequence of each. The last rows of a prompt see most and go first. Where tiles are too few to
// fill the chip their positions are split over workgroups, which leave partials (m, sum, output) for join_kernel. The kernels count
// what the tiles see for that: rows of a page table that have no new tokens take no part of the chip, and no workspace.
//
// Measured (bfloat16, 32 heads on 8 of 128; products alone reach 1,227 TFLOP/s): a prompt of 8,192 tokens 815 to 840 us,
// 655 to 675 TFLOP/s, and half as many products more for the weights (one at a time, traced: 896); the matrix units are busy 41
// percent of the time, the vector units 43. 512 capped tokens behind 65,536 positions 1,125 to 1,140 with 12 for the join: matrix
// units 28 percent, vector units 54. Seven prompts of up to 2,000 tokens, 16 leaning heads of
// 64 of float16, 125 to 131 us. Single precision (products alone: 154 TFLOP/s) 4,000 tokens of 12 heads of 128 on 4, 815 us, 60
// TFLOP/s, on 0.7 of the chip's places. The same in bfloat16 by head size: 128 148 us, 192 217, 256 318; rows of odd sizes, which no
// copy into LDS takes, 111 466 us. With weights of one element: values loaded only after the first products 1,009 us where 831 was
// then; pages looked up by branches within the loads 966.
#pragma once

#include "../kernels/lanes.hpp"
#include "attention.hpp"
#include "elements.hpp"
#include "tiles.hpp"

#include <algorithm>
#include <cfloat>

namespace certex_amd::attention {
namespace {

constexpr int kWaves   = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows    = 32 * kWaves;  // of a tile
constexpr int kUnits   = 256;          // compute units
constexpr int kMaxSplits = 64;
/** Fewest tiles of positions of a split. */
constexpr int kLeast = 4;

using f32x16 = __attribute__((ext_vector_type(16))) float;

struct prompt_plan {
  divisor page_groups;  // groups of 8 positions per page
  divisor group;        // query heads per key head
  int32_t tiles;        // of rows, at most, over all sequences
  int32_t splits;       // of a tile's positions, at most
  int32_t places;       // workgroups that the chip holds
  bool near;            // strides of pages and of 8 slots fit 32 bits
  score_scale scale;
  float slack;          // kSlack in scores
  // (a split's side by side: workgroups that write within one cache line wait for each other)
  float* part_out;      // [splits][tokens][heads][vdim]
  float* part_max;      // [splits][tokens][heads]
  float* part_sum;
};

/** A tile of rows: its sequence, the first of its rows there, and what those see. */
struct row_tile {
  int32_t sequence;
  int32_t row0, rows;   // rows of the sequence (token major): the tile's first, and all
  int64_t token0;       // of the sequence
  int32_t past;         // position of the sequence's first token
  int32_t length;
  int32_t prefix;
  int32_t begin, tiles; // positions from begin on, in tiles of TILE
};

__device__ __forceinline__ int64_t clamped(int64_t x, int64_t hi) { return x < 0 ? 0 : x > hi ? hi : x; }

/** A piece of a tile's positions: which, and of how many at most. */
struct piece_of {
  int32_t split, splits;
};

/** Splits of `tiles` equal tiles per key head, which are to fill the chip once. */
__device__ __forceinline__ int splits_alone(prompt_args const& a, prompt_plan const& plan, int tiles)
{
  const int64_t blocks = int64_t(max(1, tiles)) * a.kv_heads;
  return 2 * blocks > plan.places ? 1 : min(plan.splits, plan.places / int(blocks));
}

/**
 * The tile at a place of the launch, and its piece (WHOLE: all of it, of the tiles that are split); false where there is none.
 * - One sequence: from the last tile on, a tile's pieces side by side.
 * - Several, where something may be split (few tokens): pieces of equal length, of which the chip holds one each. The positions that
 *   the tiles see are counted (a sequence's tiles as its last one); a sequence's tiles are split as often as its length is a multiple
 *   of that share, to the nearest. (Split alike: one piece of 128 tokens behind 20,000 positions beside 63 sequences of one token and
 *   2,000 positions, 32 heads on 8 of 128, 719 us for 224.) Up to 64 sequences a lane counts one's pieces, else a thread some.
 * - 2 to 64, whole: those that see most first, by the number of row tiles that end no later (a tile's rows, and those of the
 *   sequence before them). Measured, seven prompts of up to 2,000 tokens, 16 heads of 64: 161 us by sequence, 127 by length.
 * - More, whole: from the last tile on; sequence s has the indexes from floor(first[s] group / kRows) + min(s, first[s]) on, of which
 *   the first ceil(rows / kRows) are its tiles and the next sequence's begin behind them.
 */
template <int TILE, bool WHOLE>
__device__ __forceinline__ bool find_tile(prompt_args const& a, prompt_plan const& plan, int64_t place, row_tile* out, piece_of* as)
{
  const int64_t sequences = a.pages.sequences;
  if (sequences == 0) { return false; }  // first has one entry, the lengths none
  const int lane        = threadIdx.x % 64;
  const int64_t group   = plan.group.d;
  const auto token      = [&](int64_t s) { return clamped(a.first[s], a.tokens); };
  const auto tiles_for  = [&](int64_t tokens) { return int((tokens * group + kRows - 1) / kRows); };
  const int64_t longest = a.pages.n_pages > 0 ? int64_t(a.pages.width) * a.pages.page : 0;
  int64_t lo = 0, t0, t1, length, at;
  if (sequences == 1) {
    t0 = token(0), t1 = token(1);
    const int tiles  = tiles_for(max(int64_t(0), t1 - t0));
    const int splits = uniform(splits_alone(a, plan, tiles));
    const int index  = int(uint32_t(place) / uint32_t(WHOLE ? 1 : splits));
    *as              = {uniform(int(place) - index * (WHOLE ? 1 : splits)), splits};
    at               = tiles - 1 - uniform(index);
    length           = clamped(a.lengths[0], longest);
  } else if (plan.splits > 1) {
    const auto tiles_of = [&](int f0, int f1) { return int((uint32_t(max(0, f1 - f0)) * uint32_t(group) + kRows - 1) / kRows); };
    const auto seen_by  = [&](int length) {  // tiles of positions, by a sequence's last tile
      return int((uint32_t(a.window > 0 ? min(int64_t(length), a.window + kRows) : length) + TILE - 1) / TILE);
    };
    const auto splits_for = [&](int tiles, int seen, int64_t all_work) {
      if (seen > 0 && int64_t(tiles) * seen == all_work) { return splits_alone(a, plan, tiles); }  // as without the others
      const float share = float(plan.places) / (float(max(all_work, int64_t(1))) * float(a.kv_heads));  // places per position
      return min(plan.splits, max(1, int(float(seen) * share + 0.5f)));
    };
    constexpr int kMost = 1 << 22;  // pieces; no more unless first falls
    // the pieces of tiles that are split go first: the others are shorter
    bool of_split;
    int left;  // of this lane's or thread's pieces of that kind, the place's number, if it has that one
    const auto find = [&](int split, int split_before, int all_split, int single, int single_before, int all) {
      of_split = place < all_split;
      left     = int(place) - (of_split ? split_before : all_split + single_before);
      return place < all && left >= 0 && left < (of_split ? split : single);
    };
    int tile, splits;
    if (sequences <= 64) {  // a lane's sequence
      const int64_t s  = min(int64_t(lane), sequences - 1);
      const int f0 = int(token(s)), f1 = int(token(s + 1)), n = int(clamped(a.lengths[s], longest));
      const int tiles = lane < sequences ? tiles_of(f0, f1) : 0, seen = seen_by(n);
      splits              = splits_for(tiles, seen, lanes::sum<64>(int64_t(tiles) * seen));
      const int pieces    = min(WHOLE ? tiles : tiles * splits, kMost);
      const int split     = splits > 1 ? pieces : 0, single = splits > 1 || WHOLE ? 0 : pieces;
      const int split_up  = lanes::scan_incl(split), single_up = lanes::scan_incl(single);
      const int all_split = __builtin_amdgcn_readlane(split_up, 63), all = all_split + __builtin_amdgcn_readlane(single_up, 63);
      const uint64_t mine = __ballot(find(split, split_up - split, all_split, single, single_up - single, all));
      if (mine == 0) { return false; }
      const int from   = __builtin_ctzll(mine);
      const auto taken = [&](int x) { return __builtin_amdgcn_readlane(x, from); };
      lo = from, t0 = taken(f0), t1 = taken(f1), length = taken(n);
      splits = taken(splits), tile = taken(tiles), left = taken(left);
    } else {
      // A thread's sequences, which follow one another. (Loops that are not unrolled: the code is run once by each workgroup, so that
      // fetching it is what counts. Unrolled by 4, 64 sequences of one token and 2,000 positions took 151 us for 130.)
      __shared__ int64_t s_work[kWaves];
      __shared__ int s_pieces[2][kWaves], s_found[7];
      const int wave     = threadIdx.x / 64;
      const int64_t each = (sequences + kThreads - 1) / kThreads, s0 = min(sequences, threadIdx.x * each);
      const int64_t s1   = min(sequences, s0 + each);
      int64_t busy       = s1;  // the first of them that has tokens
      // f(sequence, its first token and the next one's, its length) of those that have tokens, until that is true
      const auto each_of = [&](int64_t from, auto f) {
        int f0 = int(token(from));
#pragma unroll 1
        for (int64_t s = from; s < s1; ++s) {
          const int f1 = int(token(s + 1));
          if (f1 > f0) {
            busy = min(busy, s);
            if (f(s, f0, f1, int(clamped(a.lengths[s], longest)))) { return; }
          }
          f0 = f1;
        }
      };
      int64_t work = 0;
      each_of(s0, [&](int64_t, int f0, int f1, int n) {
        work += int64_t(tiles_of(f0, f1)) * seen_by(n);
        return false;
      });
      work = lanes::sum<64>(work);
      if (lane == 0) { s_work[wave] = work; }
      __syncthreads();
      int64_t all_work = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) { all_work += s_work[w]; }
      int split = 0, single = 0;
      each_of(busy, [&](int64_t, int f0, int f1, int n) {
        const int tiles = tiles_of(f0, f1), many = splits_for(tiles, seen_by(n), all_work);
        (many > 1 ? split : single) += WHOLE ? tiles : tiles * many;
        return false;
      });
      split              = min(max(0, split), kMost);
      single             = WHOLE ? 0 : min(max(0, single), kMost);
      const int split_up = lanes::scan_incl(split), single_up = lanes::scan_incl(single);
      if (lane == 63) {
        s_pieces[0][wave] = split_up;
        s_pieces[1][wave] = single_up;
      }
      __syncthreads();
      int split_before = split_up - split, single_before = single_up - single, all_split = 0, all = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        split_before += w < wave ? s_pieces[0][w] : 0;
        single_before += w < wave ? s_pieces[1][w] : 0;
        all_split += s_pieces[0][w];
        all += s_pieces[0][w] + s_pieces[1][w];
      }
      if (place >= uniform(all)) { return false; }
      if (find(split, split_before, all_split, single, single_before, all)) {
        each_of(busy, [&](int64_t s, int f0, int f1, int n) {
          const int tiles = tiles_of(f0, f1), many = splits_for(tiles, seen_by(n), all_work), pieces = WHOLE ? tiles : tiles * many;
          if ((many > 1) != of_split) { return false; }
          if (left >= pieces) {
            left -= pieces;
            return false;
          }
          s_found[0] = int(s);
          s_found[1] = left;
          s_found[2] = many;
          s_found[3] = tiles;
          s_found[4] = f0;
          s_found[5] = f1;
          s_found[6] = n;
          return true;
        });
      }
      __syncthreads();
      lo = uniform(s_found[0]), left = uniform(s_found[1]), splits = uniform(s_found[2]), tile = uniform(s_found[3]);
      t0 = uniform(s_found[4]), t1 = uniform(s_found[5]), length = uniform(s_found[6]);
    }
    const int index = WHOLE ? left : int(uint32_t(left) / uint32_t(splits));
    *as             = {WHOLE ? 0 : uniform(left - index * splits), uniform(splits)};
    at              = tile - 1 - uniform(index);
  } else if (sequences > 1 && sequences <= 64) {
    // this lane's sequence: `tiles` row tiles, of the costs behind + 1 to behind + tiles
    const int64_t s  = min(int64_t(lane), sequences - 1);
    const int64_t f0 = token(s), f1 = max(f0, token(s + 1)), n = clamped(a.lengths[s], longest);
    const int tiles  = lane < sequences ? tiles_for(f1 - f0) : 0;
    const int behind = int(min(max(int64_t(0), n - (f1 - f0)) * group / kRows, int64_t(1) << 28));  // beyond, all alike
    *as              = {0, 1};
    const int64_t index = place;
    // the largest cost that more than `index` tiles have or exceed
    const auto reach = [&](int cost) { return lanes::sum<64>(min(max(behind + tiles - cost + 1, 0), tiles)); };
    int some = 0, none = uniform(lanes::max<64>(behind + tiles)) + 1;  // 1 and more, if any has
    while (none - some > 1) {
      const int cost = some + (none - some) / 2;
      if (uniform(reach(cost)) > index) {
        some = cost;
      } else {
        none = cost;
      }
    }
    if (some == 0) { return false; }
    const int rank       = int(index) - uniform(reach(some + 1));
    const uint64_t equal = __ballot(some > behind && some <= behind + tiles);
    const int before     = __builtin_amdgcn_mbcnt_hi(uint32_t(equal >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(equal), 0));
    const uint64_t mine  = __ballot((equal >> lane & 1u) != 0 && before == rank);
    if (mine == 0) { return false; }
    const int from  = __builtin_ctzll(mine);
    const auto take = [&](int64_t x) {
      const uint32_t low = __builtin_amdgcn_readlane(int(x), from), high = __builtin_amdgcn_readlane(int(x >> 32), from);
      return int64_t(uint64_t(high) << 32 | low);
    };
    lo = from, t0 = take(f0), t1 = take(f1), length = take(n);
    at = some - __builtin_amdgcn_readlane(behind, from) - 1;
  } else {
    *as                 = {0, 1};
    const int64_t index = plan.tiles - 1 - place;
    const auto begins   = [&](int64_t s) {
      const int64_t f = token(s);
      return f * group / kRows + min(s, f);
    };
    // the last sequence that begins at or before the index, 64 at a time
    for (int64_t n = sequences; n > 0;) {
      const int64_t step = (n + 63) / 64, s = lo + lane * step;
      const bool before  = s < lo + n && begins(s) <= index;
      const int count    = __builtin_popcountll(__ballot(before));
      if (count == 0) { return false; }
      lo += (count - 1) * step;
      n = step == 1 ? 0 : min(step, sequences - lo);
    }
    t0 = token(lo), t1 = token(lo + 1);
    at     = index - begins(lo);
    length = clamped(a.lengths[lo], longest);
  }
  const int64_t rows = (t1 - t0) * group;
  if (at < 0 || at * kRows >= rows) { return false; }  // at < 0: first does not rise
  const int64_t past = length - (t1 - t0);
  const int64_t prefix = a.prefix.p != nullptr ? clamped(a.prefix[lo], length) : 0;
  // the positions that any row sees
  const int row0   = int(at * kRows);
  const int64_t i0 = plan.group(uint32_t(row0)), i1 = plan.group(uint32_t(min(rows, int64_t(row0) + kRows) - 1));
  const int64_t end   = max(min(past + i1 + 1, length), prefix);
  const int64_t begin = a.window > 0 ? max(int64_t(0), past + i0 + 1 - a.window) & ~int64_t(7) : 0;
  *out = {uniform(int(lo)),     uniform(row0),        uniform(int(rows)),   uniform(t0),
          uniform(int(past)),   uniform(int(length)), uniform(int(prefix)), uniform(int(begin)),
          uniform(int(end > begin ? (end - begin + TILE - 1) / TILE : 0))};
  return true;
}

/** The splits of a tile. */
__device__ __forceinline__ int splits_of(piece_of const& as, int tiles) { return max(1, min(as.splits, tiles / kLeast)); }

__device__ __forceinline__ f32x16 mfma32(f16_t, u32x4 a, u32x4 b, f32x16 c)
{
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(bf16_t, u32x4 a, u32x4 b, f32x16 c)
{
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(float, u32x4 a, u32x4 b, f32x16 c)
{
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, uint32_t(a[i])),
                                             __builtin_bit_cast(float, uint32_t(b[i])), c, 0, 0, 0);
  }
  return c;
}

/** N elements as words. */
template <typename T, int N>
struct words {
  uint32_t w[N * sizeof(T) / 4];
};

/** Elements [off, off + N) of a row of n, which begin at `from`; what is past its end is 0: the last piece is read so that it
 *  ends with the row, and moved. (Element by element a prompt of 4,000 tokens, heads of 111 bfloat16, took 353 us.) */
template <bool FULL, int N, typename T>
__device__ __forceinline__ words<T, N> row_piece(const T* from, int off, int n)
{
  constexpr int W = N * sizeof(T) / 4;
  words<T, N> v{};
  if (FULL) {
    __builtin_memcpy(&v, __builtin_assume_aligned(from, sizeof(T)), sizeof(v));
  } else if (n >= N) {
    const int past = max(0, off + N - n);
    __builtin_memcpy(&v, __builtin_assume_aligned(from - past, sizeof(T)), sizeof(v));
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < W; ++i) { v.w[i] = __builtin_amdgcn_alignbyte(i + 1 < W ? v.w[i + 1] : 0u, v.w[i], 2 * (past & 1)); }
    }
    const int by = past * int(sizeof(T)) / 4;
#pragma unroll
    for (int step = 1; step < W; step *= 2) {
#pragma unroll
      for (int i = 0; i < W; ++i) { v.w[i] = (by & step) != 0 ? (i + step < W ? v.w[i + step] : 0u) : v.w[i]; }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) { v.w[i] = by < W ? v.w[i] : 0u; }
  } else if (off < n) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) { e[i] = off + i < n ? from[i] : T(0.0f); }
    __builtin_memcpy(&v, e, sizeof(v));
  }
  return v;
}

/** The elements of a word that are infinite or NaN, as 0; whether there are any. */
template <typename T>
__device__ __forceinline__ bool drop_unbounded(uint32_t& w)
{
  if constexpr (sizeof(T) == 4) {
    if ((w & 0x7f800000u) != 0x7f800000u) { return false; }
    w = 0;
    return true;
  }
  constexpr uint32_t kExponent = std::is_same_v<T, f16_t> ? 0x7c00u : 0x7f80u;
  bool any = false;
  if ((w & kExponent) == kExponent) {
    w &= 0xffff0000u;
    any = true;
  }
  if ((w >> 16 & kExponent) == kExponent) {
    w &= 0x0000ffffu;
    any = true;
  }
  return any;
}

/** The weights' reference may lag the largest exponent by this much, and weights are multiplied by 2^kLift: float16 weights
 *  reach 2^15 and keep their precision down to 2^-27 of the largest. */
template <typename T>
constexpr float kSlack = 8.0f;
template <>
constexpr float kSlack<f16_t> = 1.0f;
template <typename T>
constexpr float kLift = 0.0f;
template <>
constexpr float kLift<f16_t> = 13.0f;

/** Positions of a tile: 128 bytes of a turned row. */
template <typename T>
constexpr int kTile = 128 / sizeof(T);

/** Workgroups per compute unit, by registers and LDS. */
template <typename T, int D>
constexpr int kPerUnit = D <= 64 ? 3 : D <= 128 ? 2 : 1;

/** Columns of V of a workgroup: half of 256, though both halves take the scores. Queries and all outputs leave no registers for
 *  the rest: 4,000 tokens, 12 heads on 4 of 256, took 377 us in bfloat16 and 3,580 in float32, where halves take 288 and 1,700. */
template <typename T, int D>
constexpr int kColumns = D > 192 ? D / 2 : D;

constexpr int power_of_two(int n) { return n <= 1 ? 1 : 2 * power_of_two((n + 1) / 2); }

/** Rows of D elements; of whole pieces, the keys at multiples of 16 bytes; of any length and alignment. */
enum class fit : int { full, whole, ragged };

template <typename T, int D, fit FIT, bool BENT>
__global__ __launch_bounds__(kThreads, (kPerUnit<T, D>)) void prompt_kernel(prompt_args a, prompt_plan plan)
{
  constexpr bool FULL   = FIT == fit::full;
  constexpr bool COPIED = FIT != fit::ragged;   // keys go to LDS as they lie
  constexpr bool WIDE   = sizeof(T) == 4;
  constexpr int TILE    = kTile<T>;
  constexpr int kPiece  = 16 / sizeof(T);       // elements of 16 bytes
  constexpr int kChunks = D / (2 * kPiece);     // products along a row, of a piece per half wave
  constexpr int kBlocks = TILE / 32;            // products along the positions
  constexpr int VD      = kColumns<T, D>;
  constexpr int kCols   = VD / 32;              // products along the columns of V
  constexpr int kGroups = TILE / 8;             // groups of 8 positions, which lie in one page
  // threads of a key row, rows at a time
  constexpr int kPieces = D / kPiece, kAcross = power_of_two(kPieces), kDown = kThreads / kAcross, kPasses = TILE / kDown;
  // Key rows in LDS. Copied there as the lanes are, 16 bytes each; a row's pieces are exchanged by its number, so that 8
  // rows' same pieces are in 8 places. Else stored from registers, 16 bytes apart.
  constexpr int kRowBytes = COPIED ? kAcross * 16 : D * sizeof(T) + 16;
  // columns of a thread in V's turn, the positions of its slot
  constexpr int kTurn = std::max(power_of_two(VD / 32), 2), kSlot = kPiece;
  __shared__ __attribute__((aligned(16))) uint8_t s_k[2][TILE * kRowBytes];
  __shared__ __attribute__((aligned(16))) uint8_t s_v[2][VD * 128];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const int column = lane % 32, half = lane / 32;

  const int kv = blockIdx.x % a.kv_heads;

  // rows of no sequence
  {
    const int64_t t0 = clamped(a.first[0], a.tokens), t1 = clamped(a.first[a.pages.sequences], a.tokens);
    for (int64_t i = blockIdx.x; i < t0 + a.tokens - max(t0, t1); i += gridDim.x) {
      const int64_t token = i < t0 ? i : max(t0, t1) + i - t0;
      T* out              = static_cast<T*>(a.out) + token * a.heads * a.vdim;
      for (int j = tid; j < a.heads * a.vdim; j += kThreads) { out[j] = T(0.0f); }
      if (a.lse != nullptr) {
        for (int j = tid; j < a.heads; j += kThreads) { a.lse[token * a.heads + j] = -INFINITY; }
      }
    }
  }
  row_tile rt;
  piece_of as;
  if (!find_tile<TILE, false>(a, plan, blockIdx.x / a.kv_heads, &rt, &as)) { return; }
  const int splits = splits_of(as, rt.tiles), split = as.split;
  if (split >= splits) { return; }
  const int tile0 = int(int64_t(split) * rt.tiles / splits), tile1 = int(int64_t(split + 1) * rt.tiles / splits);

  // this lane's row: its token and head, and the positions [lo, hi) that it sees
  const int row     = rt.row0 + wave * 32 + column;
  const bool exists = row < rt.rows;
  const uint32_t i  = plan.group(uint32_t(exists ? row : rt.row0));
  const int head    = kv * int(plan.group.d) + (exists ? row : rt.row0) - int(i * plan.group.d);
  const int p       = rt.past + int(i);
  const int hi      = exists ? max(min(p + 1, rt.length), rt.prefix) : 0;
  const int lo      = a.window > 0 ? int(max(int64_t(0), int64_t(p) + 1 - a.window)) : 0;
  const int first_col = VD < D ? blockIdx.y * VD : 0;
  const int dim = FULL ? D : a.dim, vdim = FULL ? VD : min(VD, a.vdim - first_col);

  u32x4 q[kChunks];
  {
    const T* from       = static_cast<const T*>(a.q) + (rt.token0 + i) * a.q_token + head * a.q_head;
    const uint32_t flip = plan.scale.sign < 0.0f ? (WIDE ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int off = (c * 2 + half) * kPiece;
      const auto v  = row_piece<FULL, kPiece>(from + off, off, dim);
#pragma unroll
      for (int w = 0; w < 4; ++w) { q[c][w] = exists ? v.w[w] ^ flip : 0u; }
    }
  }
  const float slope   = BENT && a.shape.slopes != nullptr ? a.shape.slopes[head] : 0.0f;
  const float per_cap = BENT && a.shape.cap != 0.0f ? a.scale / a.shape.cap : 0.0f;

  // where the groups of a tile begin in the pools: lane l has group l % kGroups
  struct places {
    int64_t k, v;    // elements behind the head's first
    uint32_t there;  // bit per group: the sequence has its page
  };
  const T* k_head      = static_cast<const T*>(a.k) + kv * a.k_head;
  const T* v_head      = static_cast<const T*>(a.v) + kv * a.v_head + first_col;
  const int32_t* table = a.pages.table + int64_t(rt.sequence) * a.pages.width;
  const int final      = max(0, rt.length - 1) / 8;
  const auto look_up   = [&](int tile) {
    const int g = min(rt.begin / 8 + tile * kGroups + lane % kGroups, final);
    const int e = int(plan.page_groups(uint32_t(g)));
    const int32_t found = table[e];
    const bool there    = uint32_t(found) < uint32_t(a.pages.n_pages);
    const uint32_t page = there ? found : 0, group = g - e * int(plan.page_groups.d);
    places at;
    if (plan.near) {
      at.k = int64_t(uint64_t(page) * uint32_t(a.k_page) + uint64_t(group) * uint32_t(8 * a.k_slot));
      at.v = int64_t(uint64_t(page) * uint32_t(a.v_page) + uint64_t(group) * uint32_t(8 * a.v_slot));
    } else {
      at.k = int64_t(page) * a.k_page + int64_t(group) * 8 * a.k_slot;
      at.v = int64_t(page) * a.v_page + int64_t(group) * 8 * a.v_slot;
    }
    at.there = uint32_t(__ballot(there)) & ((1u << kGroups) - 1u);
    return at;
  };
  const auto of_group = [](int64_t at, int g) {
    const uint32_t lo = __builtin_amdgcn_readlane(int(at), g), hi = __builtin_amdgcn_readlane(int(at >> 32), g);
    return int64_t(uint64_t(hi) << 32 | lo);
  };
  const int k_piece = tid % kAcross;
  const int v_col   = column * kTurn;
  // rows of a thread within a group
  constexpr int kStep  = std::min(8, kDown);
  // (rows of a thread are 8 apart, or 4: then the second is exchanged otherwise)
  const int64_t k_lane = int64_t(tid / kAcross % kStep) * a.k_slot;
  const auto key_piece = [&](int n) { return COPIED ? k_piece ^ ((n * kDown + tid / kAcross) % 8) : k_piece; };
  const int64_t v_lane = 4 * half * a.v_slot + v_col;

  words<T, kPiece> k_next[COPIED ? 1 : kPasses];
  words<T, kTurn> v_next[kSlot];
  // whether this thread turns columns of V (whole ones, or some that the row has not)
  const bool turns = (FULL && VD % (32 * kTurn) == 0) || v_col < (COPIED ? vdim : VD);
  const auto load_tile = [&](places const& at, int buffer) {
#pragma unroll
    for (int n = 0; n < kPasses; ++n) {
      // a wave's rows of a pass are in one group
      const int first = n * kDown + wave * (kDown / kWaves);
      const T* from   = k_head + of_group(at.k, first / 8) + int64_t(n * kDown % 8) * a.k_slot;
      const int piece = key_piece(n);
      if ((FULL && kPieces == kAcross) || piece < (COPIED ? dim / kPiece : kPieces)) {
        if constexpr (COPIED) {
          copy_to_lds(from + k_lane + piece * kPiece, lds_address(&s_k[buffer][first * kRowBytes]));
        } else {
          k_next[n] = row_piece<false, kPiece>(from + k_lane + piece * kPiece, piece * kPiece, dim);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kSlot; ++j) {
      const T* from = v_head + of_group(at.v, WIDE ? wave : 2 * wave + j / 4) + int64_t(j % 4) * a.v_slot;
      if (turns) { v_next[j] = row_piece<COPIED, kTurn>(from + v_lane, v_col, vdim); }
    }
  };
  /** Into LDS: keys as they lie, V turned. At an edge values that no row sees are 0 and unbounded ones are left out; true
   *  if there are any. */
  const auto store_tile = [&](int buffer, int tile, places const& at, bool edge) {
    bool unbounded = false;
    if (edge && turns) {
#pragma unroll
      for (int j = 0; j < kSlot; ++j) {
        const int g    = WIDE ? wave : 2 * wave + j / 4;
        const bool use = (at.there >> g & 1u) != 0 && rt.begin + tile * TILE + g * 8 + 4 * half + j % 4 < rt.length;
#pragma unroll
        for (uint32_t& w : v_next[j].w) {
          if (!use) { w = 0; }
          unbounded |= drop_unbounded<T>(w);
        }
      }
    }
    if constexpr (!COPIED) {
#pragma unroll
      for (int n = 0; n < kPasses; ++n) {
        const int r = n * kDown + tid / kAcross;
        if (kPieces == kAcross || k_piece < kPieces) {
          *reinterpret_cast<u32x4*>(&s_k[buffer][r * kRowBytes + k_piece * 16]) = __builtin_bit_cast(u32x4, k_next[n]);
        }
      }
    }
    if (turns) {
#pragma unroll
      for (int e = 0; e < kTurn; ++e) {
        u32x4 t;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (WIDE) {
            t[w] = v_next[w].w[e];
          } else {
            t[w] = __builtin_amdgcn_perm(v_next[2 * w + 1].w[e / 2], v_next[2 * w].w[e / 2],
                                         e % 2 == 0 ? 0x05040100u : 0x07060302u);
          }
        }
        const int col = v_col + e, slot = (2 * wave + half) ^ ((col / 4 + 2 * (col % 4)) % 8);
        *reinterpret_cast<u32x4*>(&s_v[buffer][col * 128 + slot * 16]) = t;
      }
    }
    if constexpr (COPIED) { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }  // the keys' copies
    return unbounded;
  };
  // whether some row does not see all of a tile
  const int first_hi = max(min(rt.past + int(plan.group(uint32_t(rt.row0))) + 1, rt.length), rt.prefix);
  const int last_row = min(rt.row0 + kRows, rt.rows) - 1;
  const int last_lo =
    a.window > 0 ? int(max(int64_t(0), int64_t(rt.past) + plan.group(uint32_t(last_row)) + 1 - a.window)) : 0;
  const auto at_edge = [&](int tile, places const& at) {
    const int t = rt.begin + tile * TILE;
    return at.there != (1u << kGroups) - 1u || t < last_lo || t + TILE > first_hi;
  };

  f32x16 o[kCols];
#pragma unroll
  for (int n = 0; n < kCols; ++n) { o[n] = f32x16{}; }
  float base = 0.0f, limit = -INFINITY, total = 0.0f;

  if constexpr (FIT == fit::whole) {
    // pieces that no row has, which meet the query's 0
    for (int at = tid * 16; at < int(sizeof(s_k)); at += kThreads * 16) { *reinterpret_cast<u32x4*>(&s_k[0][0] + at) = u32x4{}; }
    __syncthreads();
  }
  if (tile0 < tile1) {
    places here = look_up(tile0), next = tile0 + 1 < tile1 ? look_up(tile0 + 1) : here;
    load_tile(here, 0);
    bool edge      = at_edge(tile0, here);
    bool unbounded = store_tile(0, tile0, here, edge);
    unbounded      = edge ? __syncthreads_or(unbounded) != 0 : (__syncthreads(), false);
    for (int tile = tile0; tile < tile1; ++tile) {
      const int buffer = (tile - tile0) % 2;
      const bool more  = tile + 1 < tile1;
      places ahead     = next;
      if (more) {
        if (tile + 2 < tile1) { ahead = look_up(tile + 2); }
        load_tile(next, 1 - buffer);
      }
      const int t0    = rt.begin + tile * TILE;
      const bool some = t0 < hi && t0 + TILE > lo;
      if (__any(some)) {
        f32x16 s[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
          for (int e = 0; e < 16; ++e) { s[b][e] = BENT ? 0.0f : -base; }
        }
        // operands are read four products ahead, and no further: registers are what is short
        const auto key_at = [&](int c, int b) {
          const int piece = COPIED ? (c * 2 + half) ^ (column % 8) : c * 2 + half;
          return *reinterpret_cast<const u32x4*>(&s_k[buffer][(b * 32 + column) * kRowBytes + piece * 16]);
        };
        constexpr int kAhead = 4;
        u32x4 k[kAhead];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) { k[i] = key_at(i / kBlocks, i % kBlocks); }
#pragma unroll
        for (int i = 0; i < kChunks * kBlocks; ++i) {
          s[i % kBlocks] = mfma32(T{}, k[i % kAhead], q[i / kBlocks], s[i % kBlocks]);
          if (i + kAhead < kChunks * kBlocks) { k[i % kAhead] = key_at((i + kAhead) / kBlocks, i % kBlocks); }
          if (i % kAhead == kAhead - 1) { __builtin_amdgcn_sched_barrier(0); }
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (BENT) {
          // less base, which is the last operation's other term
          const float ahead_of = float(p - t0 - 4 * half);
          if (a.shape.cap != 0.0f) {
            // where all of the wave's scores are small beside the cap, tanh_of's polynomial alone: the same numbers. (512 tokens behind
            // 65,536 positions 1,125 us, 1,373 with tanh_of alone; 1 - 2 / (e^2u + 1), 2^-22 cap off however small u is, 1,040.)
            float most = 0.0f;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
              for (int e = 0; e < 16; ++e) { most = fmaxf(most, __builtin_fabsf(s[b][e])); }
            }
            if (__all(most * __builtin_fabsf(per_cap) < kNear)) {
#pragma unroll
              for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int e = 0; e < 16; ++e) { s[b][e] = __builtin_fmaf(a.shape.cap, tanh_near(s[b][e] * per_cap), -base); }
              }
            } else {
#pragma unroll
              for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  float x = s[b][e];
                  asm("" : "+v"(x));  // or the polynomial is taken ahead of the branch, into registers that are not there
                  s[b][e] = __builtin_fmaf(a.shape.cap, tanh_of(x * per_cap), -base);
                }
              }
            }
            if (a.shape.slopes != nullptr) {
#pragma unroll
              for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  s[b][e] = __builtin_fmaf(-slope, __builtin_fabsf(ahead_of - float(b * 32 + 8 * (e / 4) + e % 4)), s[b][e]);
                }
              }
            }
          } else {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float lean = __builtin_fabsf(ahead_of - float(b * 32 + 8 * (e / 4) + e % 4));
                s[b][e]          = __builtin_fmaf(s[b][e], a.scale, __builtin_fmaf(-slope, lean, -base));
              }
            }
          }
        }
        const bool masked = edge && !(here.there == (1u << kGroups) - 1u && __all(!exists || (t0 >= lo && t0 + TILE <= hi)));
        if (masked) {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int t   = t0 + b * 32 + 8 * (e / 4) + 4 * half + e % 4;
              const bool in = t >= lo && t < hi && (here.there >> (b * 4 + e / 4) & 1u) != 0;
              s[b][e]       = in ? s[b][e] : -INFINITY;
            }
          }
        }
        float high = s[0][0];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
          for (int e = 0; e < 16; ++e) { high = fmaxf(high, s[b][e]); }
        }
        if (__any(high > limit)) {
          high = lanes::fold32(high, [](float u, float w) { return fmaxf(u, w); });
          // relative to base: where something was counted before, base itself is 0
          const float up = limit == -INFINITY ? high : fmaxf(high, 0.0f);
          const bool set = up > -INFINITY;
          // with a scale of 0 all weigh alike, wherever the scores are
          const float grown = !set || plan.scale.scale2 == 0.0f ? base : base + up;
          const float moved = grown - base;
          const float keep  = limit == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-moved * plan.scale.scale2);
          total *= keep;
#pragma unroll
          for (int n = 0; n < kCols; ++n) { o[n] *= keep; }
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) { s[b][e] -= moved; }
          }
          base  = grown;
          limit = set ? (plan.scale.scale2 == 0.0f ? INFINITY : plan.slack) : limit;
        }
        if (masked && plan.scale.scale2 == 0.0f) {  // -inf times 0
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) { s[b][e] = s[b][e] == -INFINITY ? -INFINITY : s[b][e] * 0.0f; }
          }
        }
        const float scale2 = masked && plan.scale.scale2 == 0.0f ? 1.0f : plan.scale.scale2;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], scale2, kLift<T>));
          }
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
          for (int e = 0; e < 16; e += 4) { total += (s[b][e] + s[b][e + 1]) + (s[b][e + 2] + s[b][e + 3]); }
        }
        constexpr int kSteps = TILE / (2 * kSlot);  // products along the positions, of a slot per half wave
        const auto value_at  = [&](int m, int n) {
          const int col = n * 32 + column, slot = (2 * m + half) ^ ((col / 4 + 2 * (col % 4)) % 8);
          return *reinterpret_cast<const u32x4*>(&s_v[buffer][col * 128 + slot * 16]);
        };
        u32x4 v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) { v[i] = value_at(i / kCols, i % kCols); }
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
          u32x4 w, rest;  // the weights, and what rounding them to 16 bits leaves
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (WIDE) {
              w[e] = __builtin_bit_cast(uint32_t, float(s[0][4 * m + e]));
            } else {
              const float even = s[m / 2][8 * (m % 2) + 2 * e], odd = s[m / 2][8 * (m % 2) + 2 * e + 1];
              w[e]             = pack2<T>(even, odd);
              rest[e]          = pack2<T>(even - lower<T>(w[e]), odd - upper<T>(w[e]));
            }
          }
#pragma unroll
          for (int n = 0; n < kCols; ++n) {
            const int i = m * kCols + n;
            o[n]        = mfma32(T{}, v[i % kAhead], w, o[n]);
            if constexpr (!WIDE) { o[n] = mfma32(T{}, v[i % kAhead], rest, o[n]); }
            if (i + kAhead < kSteps * kCols) { v[i % kAhead] = value_at((i + kAhead) / kCols, (i + kAhead) % kCols); }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (unbounded) {
          // values that are infinite or NaN show in the rows that see them, and in no other: each by itself
          for (int j = 0; j < TILE; ++j) {
            const int t = t0 + j, g = j / 8;
            if (t >= rt.length || (here.there >> g & 1u) == 0) { continue; }
            const T* from = v_head + of_group(here.v, g) + int64_t(j % 8) * a.v_slot;
            const bool in = t >= lo && t < hi;
#pragma unroll
            for (int n = 0; n < kCols; ++n) {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const int col = n * 32 + 8 * (e / 4) + 4 * half + e % 4;
                const float v = in && col < vdim ? float(from[col]) : 0.0f;
                o[n][e] += __builtin_fabsf(v) < INFINITY ? 0.0f : v;
              }
            }
          }
        }
      }
      if (more) {
        edge      = at_edge(tile + 1, next);
        unbounded = store_tile(1 - buffer, tile + 1, next, edge);
        unbounded = edge ? __syncthreads_or(unbounded) != 0 : (__syncthreads(), false);
      }
      here = next;
      next = ahead;
    }
  }

  total = lanes::fold32(total, [](float u, float w) { return u + w; });
  if (!exists) { return; }
  const bool counted = limit != -INFINITY;
  if (splits == 1) {
    const int64_t at  = (rt.token0 + i) * a.heads + head;
    const float scale = total == 0.0f ? 0.0f : 1.0f / total;
    T* out            = static_cast<T*>(a.out) + at * a.vdim + first_col;
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = n * 32 + 8 * (e / 4) + 4 * half + e % 4;
        if (col < vdim) { out[col] = T(total == 0.0f ? 0.0f : o[n][e] * scale); }
      }
    }
    if (half == 0 && first_col == 0 && a.lse != nullptr) { a.lse[at] = lse_of(plan.scale, base, total, kLift<T>); }
  } else {
    const int64_t at = (split * a.tokens + rt.token0 + i) * a.heads + head;
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = n * 32 + 8 * (e / 4) + 4 * half + e % 4;
        if (col < vdim) { plan.part_out[at * a.vdim + first_col + col] = o[n][e]; }
      }
    }
    if (half == 0 && first_col == 0) {
      plan.part_max[at] = counted ? base : -INFINITY;
      plan.part_sum[at] = total;
    }
  }
}

/** Rows of a workgroup that joins: fewer, so that there are more. (32 rows: 24 us where 18 was.) */
constexpr int kJoinRows = kThreads / 32;

/** Rows of a tile that was split, 32 threads each: joins their partials in order of position. */
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(prompt_args a, prompt_plan plan)
{
  __shared__ float s_factor[kJoinRows][kMaxSplits], s_sum[kJoinRows][kMaxSplits];
  const int kv = blockIdx.x % a.kv_heads, r = threadIdx.x / 32, lane = threadIdx.x % 32;
  row_tile rt;
  piece_of as;
  if (!find_tile<kTile<T>, true>(a, plan, blockIdx.x / a.kv_heads, &rt, &as)) { return; }
  const int n   = splits_of(as, rt.tiles);
  const int row = rt.row0 + blockIdx.y * kJoinRows + r;
  if (n == 1 || row - r >= rt.rows) { return; }
  const uint32_t token = plan.group(uint32_t(min(row, rt.rows - 1)));
  const int64_t at     = (rt.token0 + token) * a.heads + kv * int(plan.group.d) + min(row, rt.rows - 1) - int(token * plan.group.d);
  const int64_t next   = a.tokens * a.heads;  // from a split's partials to those of the next
  // a thread per split (or two) reads them, then all take them in order
  float m = -INFINITY;
  for (int s = lane; s < n; s += 32) {
    s_factor[r][s] = plan.part_max[at + s * next];
    s_sum[r][s]    = plan.part_sum[at + s * next];
    m              = fmaxf(m, s_factor[r][s]);
  }
  m = lanes::max<32>(m);
  for (int s = lane; s < n; s += 32) { s_factor[r][s] = factor_of(plan.scale, s_factor[r][s], m); }
  __syncthreads();
  if (row >= rt.rows) { return; }
  float sum = 0.0f;
  for (int s = 0; s < n; ++s) { sum += s_factor[r][s] * s_sum[r][s]; }
  for (int col = lane; col < a.vdim; col += 32) {
    float acc = 0.0f;
#pragma unroll 4
    for (int s = 0; s < n; ++s) { acc = __builtin_fmaf(s_factor[r][s], plan.part_out[(at + s * next) * a.vdim + col], acc); }
    static_cast<T*>(a.out)[at * a.vdim + col] = T(sum == 0.0f ? 0.0f : acc / sum);
  }
  if (lane == 0 && a.lse != nullptr) { a.lse[at] = lse_of(plan.scale, m, sum, kLift<T>); }
}

/** Tiles of rows over all sequences, at most: a last one of each that has tokens, and whole ones. One where there is none, for the
 *  tokens' zeros. */
int64_t tiles_of(prompt_args const& a)
{
  return std::max<int64_t>(1, a.tokens * (a.heads / a.kv_heads) / kRows + std::min(a.tokens, a.pages.sequences));
}

/** Splits of a tile's positions, at most: those of one sequence that has all tokens. The kernels count what the tiles see, and take
 *  as many splits as the chip holds at once (find_tile). One more, which takes a second
 *  round, costs most: bfloat16, 32 heads on 8 of 128, 1,500 tokens 80 us where 65 is now. Long prompts whose rows see unequally much and
 *  that fill some three quarters of the places would have less: 4,000 tokens, 12 heads on 4 of 128, 125 us for 148, of 111 275 for
 *  466, float32 526 for 815. 64 sequences of one token behind 16,383 positions, 813 us, took 1,074 where splits went by the tokens
 *  alone; 16 tokens behind 16,000 in a table of 64 rows, 60, took 213 where a row counted as a tile. */
int splits_for(prompt_args const& a, int tile, int per_unit)
{
  const int64_t most   = int64_t(a.pages.width) * a.pages.page;
  const int64_t seen   = a.window > 0 ? std::min(most, a.window + kRows) : most;
  const int64_t blocks = std::max<int64_t>(1, (a.tokens * (a.heads / a.kv_heads) + kRows - 1) / kRows * a.kv_heads);
  const int64_t wanted = int64_t(kUnits) * per_unit / blocks;
  return int(std::max<int64_t>(1, std::min({wanted, int64_t(kMaxSplits), seen / tile / kLeast})));
}

template <typename T>
size_t workspace_for(prompt_args const& a)
{
  // the most splits that any variant takes
  const int splits = std::max(splits_for(a, kTile<T>, 1), splits_for(a, kTile<T>, 3));
  return splits == 1 ? 0 : sizeof(float) * size_t(a.tokens) * a.heads * splits * (a.vdim + 2);
}

template <typename T>
void launch(prompt_args const& a, hipStream_t stream)
{
  const auto launched = [&](auto bucket, auto how) {
    constexpr int D = decltype(bucket)::value;
    prompt_plan plan{divisor(uint32_t(a.pages.page / 8)), divisor(uint32_t(a.heads / a.kv_heads))};
    plan.tiles  = int32_t(tiles_of(a));
    plan.splits = splits_for(a, kTile<T>, kPerUnit<T, D>);
    plan.near   = std::max({a.k_page, a.v_page, 8 * a.k_slot, 8 * a.v_slot}) < (int64_t(1) << 32);
    plan.scale  = scale_of(a.shape.any() ? 1.0f : a.scale);
    plan.slack  = float(std::min(double(kSlack<T>) / double(plan.scale.scale2), double(FLT_MAX)));
    plan.places         = kUnits * kPerUnit<T, D>;
    const int64_t slots = a.tokens * a.heads * plan.splits;
    plan.part_out       = static_cast<float*>(a.workspace);
    plan.part_max       = plan.part_out + slots * a.vdim;
    plan.part_sum       = plan.part_max + slots;
    // a workgroup per piece: to the nearest, they are as many as the chip's places and the tiles at most
    const int64_t blocks = int64_t(plan.tiles) * a.kv_heads;
    const dim3 grid(uint32_t(std::min(blocks * plan.splits, blocks + plan.places)), (a.vdim + kColumns<T, D> - 1) / kColumns<T, D>);
    if (a.shape.any()) {
      prompt_kernel<T, D, decltype(how)::value, true><<<grid, kThreads, 0, stream>>>(a, plan);
    } else {
      prompt_kernel<T, D, decltype(how)::value, false><<<grid, kThreads, 0, stream>>>(a, plan);
    }
    if (plan.splits > 1) {
      // tiles that are split see 1.5 places' share of the positions at least
      const int64_t split = std::min<int64_t>(plan.tiles, plan.places * 2 / (3 * a.kv_heads) + 1);
      join_kernel<T><<<dim3(uint32_t(split) * a.kv_heads, kRows / kJoinRows), kThreads, 0, stream>>>(a, plan);
    }
  };
  const auto aligned = [](int64_t elements) { return elements * sizeof(T) % 16 == 0; };
  const bool whole   = reinterpret_cast<uintptr_t>(a.k) % 16 == 0 && aligned(a.k_page) && aligned(a.k_slot) &&
                     aligned(a.k_head) && aligned(a.dim) && a.vdim % 8 == 0;
  const auto bucket = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (whole && a.dim == D && a.vdim == D) {
      launched(d, std::integral_constant<fit, fit::full>{});
    } else if (whole) {
      launched(d, std::integral_constant<fit, fit::whole>{});
    } else {
      launched(d, std::integral_constant<fit, fit::ragged>{});
    }
  };
  const int dim = std::max(a.dim, a.vdim);
  if (dim <= 64) {
    bucket(std::integral_constant<int, 64>{});
  } else if (dim <= 96) {
    bucket(std::integral_constant<int, 96>{});
  } else if (dim <= 128) {
    bucket(std::integral_constant<int, 128>{});
  } else if (dim <= 192) {
    bucket(std::integral_constant<int, 192>{});
  } else {
    bucket(std::integral_constant<int, 256>{});
  }
}

}  // namespace
}  // namespace certex_amd::attention
