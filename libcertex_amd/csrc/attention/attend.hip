// Attention of one new token of every sequence over its pages of keys and values.
//
// out = sum_t p_t v_t / sum_t p_t with p_t = 2^(scale log2(e) (x_t - m)), x_t = q.k_t, over the positions t
// of [max(0, len - window), len). One pass over the positions keeps a reference m, the sum and the
// output in float32, and scales the last two where m grows. A negative scale turns q's sign.
//
// What bounds it: every key and value is read once and used by the heads / kv_heads query heads that share
// it, a few operations per byte, so the rate at which memory is read. The kernel keeps the two products
// off the critical path by giving them to the matrix cores in a form that needs no exchange between lanes
// and no LDS:
// - a wave takes 32 positions (float32: 16); S^T = K Q^T has the positions as rows and up to 16 query heads
//   as columns, so that K rows go from memory to the operand registers as they lie (16 bytes per lane);
// - the rows of the two 16-position products are permuted such that a lane's 8 results are the 8
//   consecutive positions that it holds as k-slots of O^T = V^T P^T: the weights never move (16-bit types take them
//   whole, as three elements, and so this product three times);
// - V^T is formed in registers: a lane loads 8 positions x 8 columns (16 bytes of a row each, whole rows
//   per 16 lanes) and swaps halfwords (v_perm), 32 instructions per 32 x 128 values (float32: as it lies);
// - m, the sum and the scaling are per query head, that is per lane.
// The loads of the next keys and of this tile's values are in flight during both products.
//
// Work is dealt on the device, from the lengths: the tiles of all sequences, one after the other, in
// equal shares, each share to one workgroup per key head. So any mix of lengths fills the chip and the
// host reads nothing back, and the heads of a position are read at about the same time (they are
// neighbours in memory where a slot holds all heads). A share that cuts a sequence leaves a partial
// (m, sum, output) in the workspace, and a second launch joins them in order of position.
//
// Measured (8 key heads of 128 bfloat16, 32 query heads; reading alone reaches 6.4 TB/s): 64 sequences up
// to 8,192, 0.94 GB of keys and values: 158 us with the 6 us of the join, 5.9 TB/s; one sequence of
// 131,072, 0.54 GB: 88 us, 6.1 TB/s; four of up to 131,072: 6.3 TB/s. Heads of 64: 5.4 TB/s where a slot holds
// all heads (128 bytes of a line pair each), 6.2 with the heads first; of 256 6.2, and 5.8 in float32; of 160, and of 192
// with values of 128, which run as 256, 4.4. More workgroups or waves per
// compute unit read slower (three: 193 us for the 64 sequences): the memory prefers fewer streams.
//
// Bent scores (BENT) are taken between the products, some 20 operations each in the shade of the reads: the 64
// sequences with a cap 159 us; three of up to 3,001 float16 positions of heads of 64 with slopes 7.1 us and 5 for the join.
#include "scores.hpp"
#include "shares.hpp"
#include "tiles.hpp"

namespace certex_amd::attention {
namespace {

/** Positions of a lane group in a step: its rows of the 16-position products (two of 16 bits, one of float32). */
template <typename T>
constexpr int kGroup = sizeof(T) == 4 ? 4 : 8;
/** Positions of a workgroup's step: a tile. */
template <typename T>
constexpr int kTile = 4 * kGroup<T> * kWaves;

/** The elements of a lane's piece: 16 bytes of a row at any alignment of the elements (the memory takes
 *  misaligned vector loads); TINY rows are shorter than a piece and read element by element. */
template <int BYTES, typename T>
__device__ __forceinline__ auto piece(const T* p)
{
  if constexpr (BYTES == 16) {
    u32x4 v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, sizeof(T)), 16);
    return v;
  } else {
    u32x2 v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, sizeof(T)), 8);
    return v;
  }
}

/** A value piece: read once by the call, so it is not kept in the caches. Measured: 64 sequences up to 8,192
 *  184 -> 168 us, one of 131,072 103 -> 92 us. (Key pieces are half lines, whose other half is the next
 *  load's: reading them past the caches 184 -> 181 us alone, 176 us together.) */
template <int BYTES, typename T>
__device__ __forceinline__ auto passing_piece(const T* p)
{
  using words = std::conditional_t<BYTES == 16, u32x4, u32x2>;
  using loose = words __attribute__((aligned(sizeof(T))));
  return words(__builtin_nontemporal_load(reinterpret_cast<const loose*>(p)));
}

/** Keys, queries and values of a wave's step for elements T, head dimensions up to D. */
template <typename T, int D>
struct geometry {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr int kPiece  = kWide ? 4 : 8;           // elements of a key piece (16 bytes)
  static constexpr int kChunk  = 4 * kPiece;              // dimensions of a product's four lane groups
  static constexpr int kChunks = D / kChunk;
  static constexpr int kCols   = kWide || D <= 64 ? 4 : 8;  // columns of a value piece
  static constexpr int kBlocks = (D + 16 * kCols - 1) / (16 * kCols);  // pieces of a lane per value row
  static constexpr bool kWhole = D % (16 * kCols) == 0;                // no piece of a full row is past its end
  static constexpr int kHalves = kGroup<T> / 4;             // 16-position products of a step
  using value = std::conditional_t<kCols * sizeof(T) == 16, u32x4, u32x2>;
};

/** The weights' reference may lag the largest exponent by this much (twice as much where large scores round it) before the
 *  sums are rescaled, and weights are multiplied by 2^kLift: float16 weights reach 2^15 and keep their precision down to
 *  2^-27 of the largest. */
template <typename T>
constexpr float kSlack = 8.0f;
template <>
constexpr float kSlack<f16_t> = 1.0f;
template <typename T>
constexpr float kLift = 0.0f;
template <>
constexpr float kLift<f16_t> = 13.0f;

/** Rows that fill the D elements of their tiles; shorter ones; rows of fewer than 8 elements. */
enum class fit : int { full, part, tiny };

/** Workgroups per compute unit: a wave holds the keys and values of a step in registers. */
template <typename T, int D>
constexpr int kPerUnit = D <= 128 ? 2 : 1;

/** What of word w of a key or query piece counts when its first `skip` elements do not. */
template <typename T>
__device__ __forceinline__ uint32_t counted(int skip, int w)
{
  if constexpr (sizeof(T) == 4) { return skip > w ? 0u : 0xffffffffu; }
  return skip > 2 * w + 1 ? 0u : skip > 2 * w ? 0xffff0000u : 0xffffffffu;
}

template <typename T, int D, fit FIT, bool BENT>
__global__ __launch_bounds__(kThreads, (kPerUnit<T, D>)) void attend_kernel(attend_args a, attend_plan plan)
{
  constexpr bool TINY    = FIT == fit::tiny;
  constexpr bool FULL    = FIT == fit::full;
  using G                = geometry<T, D>;
  constexpr int kChunks  = G::kChunks, kPiece = G::kPiece, kCols = G::kCols, kBlocks = G::kBlocks;
  constexpr int kOut     = kBlocks * kCols;  // accumulators of 16 columns
  constexpr int kGrp     = kGroup<T>, kHalves = G::kHalves, kTiles = kTile<T>;
  __shared__ float s_out[kWaves][kRows][D];
  __shared__ float s_max[kWaves][kRows], s_sum[kWaves][kRows];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, g = lane / 16;
  // consecutive workgroups go to the 8 dies in turn: a share's tables to all of them, or to one
  const int turn      = plan.one_die ? blockIdx.x / 8 : blockIdx.x;
  const int table     = turn % plan.tables;
  const int64_t share = plan.one_die ? int64_t(turn / plan.tables) * 8 + blockIdx.x % 8 : turn / plan.tables;

  const shares sh = shares_of<kTiles>(a, plan);
  // rows without a position
  for (int64_t b = blockIdx.x; b < a.pages.sequences; b += gridDim.x) {
    if (span_of<kTiles>(a, b).tiles == 0) {
      T* out = static_cast<T*>(a.out) + b * a.heads * a.vdim;
      for (int i = tid; i < a.heads * a.vdim; i += kThreads) { out[i] = T(0.0f); }
      if (a.lse != nullptr) {
        for (int i = tid; i < a.heads; i += kThreads) { a.lse[b * a.heads + i] = -INFINITY; }
      }
    }
  }
  if (share >= sh.n) { return; }
  int64_t tile       = sh.first(share);
  const int64_t last = sh.first(share + 1);

  // the sequence of the first tile
  int64_t b = 0, before = 0;  // tiles of the sequences below b
  for (int64_t b0 = 0;; b0 += 64) {
    const int mine    = b0 + lane < a.pages.sequences ? span_of<kTiles>(a, b0 + lane).tiles : 0;
    const int incl    = lanes::scan_incl(mine);
    const uint64_t up = __ballot(before + incl > tile);
    if (up != 0) {
      const int at = __builtin_ctzll(up);
      b            = b0 + at;
      before += __builtin_amdgcn_readlane(incl - mine, at);
      break;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }

  const int key_off   = TINY ? 0 : FULL ? D : a.dim - kPiece;  // of the last whole piece of a row
  const int value_off = TINY ? 0 : (FULL ? D : a.vdim) - kCols;
  const int dim = FULL ? D : a.dim, vdim = FULL ? D : a.vdim;
  const int kv = table % a.kv_heads, row0 = table / a.kv_heads * kRows;
  const int rows = min(kRows, plan.group - row0), h0 = kv * plan.group + row0;
  // bent scores take the scale with its sign before the softmax, which then has a scale of 1
  const float slope   = BENT && a.shape.slopes != nullptr ? a.shape.slopes[h0 + min(r, rows - 1)] : 0.0f;
  const float per_cap = BENT && a.shape.cap != 0.0f ? a.scale / a.shape.cap : 0.0f;
  const uint32_t flip = plan.scale.sign < 0.0f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;  // of a word of q
  const T* k_head = static_cast<const T*>(a.k) + kv * a.k_head;
  const T* v_head = static_cast<const T*>(a.v) + kv * a.v_head;

  // the page of a group's positions, and the first one's slot
  struct place {
    int32_t page, slot;
  };
  span sp{};
  int t0 = 0, t1 = 0, group = 0, stop = 0, final = 0;
  const int32_t* pages = nullptr;
  place v_at{};
  u32x4 q[kChunks], k[kHalves][kChunks];
  const auto entry = [&](int group) {
    const int at = min(group, final);
    const int e  = int(plan.page_groups(uint32_t(at)));
    return place{pages[e], (at - e * int(plan.page_groups.d)) * kGrp};
  };
  const auto load_keys = [&](place at) {
    const int page  = uint32_t(at.page) < uint32_t(a.pages.n_pages) ? at.page : 0;
    const T* k_page = k_head + int64_t(page) * a.k_page;
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {
      const T* row = k_page + int64_t(at.slot + half * 4 + r % 4) * a.k_slot;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int dim0 = (c * 4 + g) * kPiece;
        if constexpr (TINY) {
          T e[kPiece];
#pragma unroll
          for (int j = 0; j < kPiece; ++j) { e[j] = dim0 + j < dim ? row[dim0 + j] : T(0.0f); }
          __builtin_memcpy(&k[half][c], e, 16);
        } else {
          // the piece that a row ends in is taken from the row's end: dimensions that an earlier piece holds come again
          k[half][c] = piece<16>(row + (FULL ? dim0 : min(dim0, key_off)));
        }
      }
    }
  };
  // the share's tiles of sequence b (or of the next that has any): their range, and the first step's loads
  const auto begin = [&] {
    for (sp = span_of<kTiles>(a, b); sp.tiles == 0; sp = span_of<kTiles>(a, b)) { ++b; }
    t0              = int(tile - before);
    t1              = int(min(int64_t(sp.tiles), t0 + last - tile));
    pages           = a.pages.table + b * a.pages.width;
    const int start = sp.begin / 8 * (8 / kGrp);  // in lane groups' positions
    final           = (sp.end - 1) / kGrp;
    // a wave's steps: one in every tile that reaches it
    group = start + (t0 * kWaves + wave) * 4;
    stop  = min(start + t1 * kWaves * 4, final + 1);
    place k_at{};
    if (group < stop) {
      k_at = entry(group + r / 4);
      v_at = entry(group + g);
    }
    // the queries: column r, pieces of the dimensions that this lane's group holds
    const T* q_row = static_cast<const T*>(a.q) + b * a.q_seq + (h0 + min(r, rows - 1)) * a.q_head;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int dim0 = (c * 4 + g) * kPiece;
      if constexpr (TINY) {
        T e[kPiece];
#pragma unroll
        for (int j = 0; j < kPiece; ++j) { e[j] = dim0 + j < dim ? q_row[dim0 + j] : T(0.0f); }
        __builtin_memcpy(&q[c], e, 16);
      } else {
        q[c] = piece<16>(q_row + (FULL ? dim0 : min(dim0, key_off)));
      }
    }
    if (group < stop) { load_keys(k_at); }
  };

  begin();
  for (bool first = true;; first = false) {
    // query heads that there are not, dimensions that come twice: 0
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int dim0 = (c * 4 + g) * kPiece;
      const int skip = FIT == fit::part ? dim0 - min(dim0, key_off) : 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) { q[c][w] = r < rows ? (q[c][w] & counted<T>(skip, w)) ^ flip : 0u; }
    }
    f32x4 o[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i) { o[i] = f32x4{0, 0, 0, 0}; }
    float top = -INFINITY, limit = -INFINITY, base = 0.0f, total = 0.0f;

    while (group < stop) {
      const int next = group + kWaves * 4;
      // values of this step: positions (group + g) * kGrp + 0..kGrp - 1
      const bool have = uint32_t(v_at.page) < uint32_t(a.pages.n_pages);
      const T* v_page = v_head + int64_t(have ? v_at.page : 0) * a.v_page;
      typename G::value v[kGrp][kBlocks];
#pragma unroll
      for (int j = 0; j < kGrp; ++j) {
        const T* row = v_page + int64_t(v_at.slot + j) * a.v_slot;
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
          const int col = (n * 16 + r) * kCols;
          if constexpr (TINY) {
            T e[kCols];
#pragma unroll
            for (int i = 0; i < kCols; ++i) { e[i] = col + i < vdim ? row[col + i] : T(0.0f); }
            __builtin_memcpy(&v[j][n], e, sizeof(e));
          } else {
            v[j][n] = passing_piece<sizeof(T) * kCols>(row + (FULL && G::kWhole ? col : min(col, value_off)));
          }
        }
      }
      if (FIT == fit::part && dim < D) {
        // dimensions past the row, or held by an earlier piece: 0 (an infinity there would meet the query's 0)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int dim0 = (c * 4 + g) * kPiece;
          const int skip = dim0 - min(dim0, key_off);  // leading elements of the piece that do not count
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t mask = counted<T>(skip, w);
#pragma unroll
            for (int half = 0; half < kHalves; ++half) { k[half][c][w] &= mask; }
          }
        }
      }
      f32x4 s[kHalves];
#pragma unroll
      for (int half = 0; half < kHalves; ++half) { s[half] = f32x4{0, 0, 0, 0}; }
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
          if constexpr (G::kWide) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              s[half] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, uint32_t(k[half][c][w])),
                                                             __builtin_bit_cast(float, uint32_t(q[c][w])), s[half], 0, 0, 0);
            }
          } else {
            s[half] = mfma(T{}, k[half][c], q[c], s[half]);
          }
        }
      }
      // the next step's pages and keys
      if (next < stop) {
        const place k_at = entry(next + r / 4);
        v_at             = entry(next + g);
        load_keys(k_at);
      }
      // weights: lane group g holds the positions t + 0..kGrp - 1 of query r
      float x[kGrp];
#pragma unroll
      for (int j = 0; j < kGrp; ++j) { x[j] = s[j / 4][j % 4]; }
      const uint32_t t = uint32_t(group + g) * kGrp;  // past the end it may pass 2^31
      if constexpr (BENT) {
#pragma unroll
        for (int j = 0; j < kGrp; ++j) {
          x[j] = bent(x[j], a.scale, per_cap, a.shape.cap, slope, float(uint32_t(sp.end) - 1u - (t + j)));
        }
      }
      const uint32_t t_begin = uint32_t(sp.begin), t_end = uint32_t(sp.end);
      const bool whole  = have && t >= t_begin && t + kGrp <= t_end;
      const bool masked = !__all(whole);
      if (masked) {
#pragma unroll
        for (int j = 0; j < kGrp; ++j) {
          const bool in = have && t + j >= t_begin && t + j < t_end;
          x[j]          = in ? x[j] : -INFINITY;
#pragma unroll
          for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
            for (int w = 0; w < int(sizeof(v[j][n]) / 4); ++w) { v[j][n][w] = in ? v[j][n][w] : 0u; }
          }
        }
      }
      float high = x[0];
#pragma unroll
      for (int j = 1; j < kGrp; ++j) { high = fmaxf(high, x[j]); }
      if (__any(high > limit)) {
        const auto larger = [](float u, float w) { return fmaxf(u, w); };
        high              = lanes::fold16(lanes::fold32(high, larger), larger);
        const float grown = fmaxf(top, high);
        const float keep  = grown == -INFINITY ? 0.0f : weight_of(plan.scale, top, grown);
        total *= keep;
#pragma unroll
        for (int i = 0; i < kOut; ++i) { o[i] *= keep; }
        top   = grown;
        limit = grown + plan.slack;
        // with a scale of 0 all weigh alike, wherever the scores are
        base = grown == -INFINITY || plan.scale.scale2 == 0.0f ? 0.0f : grown;
      }
      float p[kGrp];
#pragma unroll
      for (int j = 0; j < kGrp; ++j) {
        // what is rounded is the distance from the reference
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j] - base, plan.scale.scale2, kLift<T>));
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < kGrp; ++j) { p[j] = x[j] == -INFINITY ? 0.0f : p[j]; }
      }
#pragma unroll
      for (int j = 0; j < kGrp; j += 4) { total += (p[j] + p[j + 1]) + (p[j + 2] + p[j + 3]); }

      if constexpr (G::kWide) {
#pragma unroll
        for (int j = 0; j < kGrp; ++j) {
#pragma unroll
          for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
            for (int e = 0; e < kCols; ++e) {
              o[n * kCols + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, uint32_t(v[j][n][e])), p[j],
                                                                     o[n * kCols + e], 0, 0, 0);
            }
          }
        }
      } else {
        // the weights enter with all 24 bits, as three elements of 8 or 11 bits each: the value, its remainder, and what that
        // leaves. The matrix cores wait for memory, so the third costs little (two and three, us: 64 sequences up to 8,192 157.5
        // and 158.5, one of 131,072 89 and 89; 32 query heads on one key head 112 and 115).
        u32x4 part[3];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float even = p[2 * w], odd = p[2 * w + 1];
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            part[i][w] = pack2<T>(even, odd);
            even -= float(T(even));
            odd -= float(T(odd));
          }
        }
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
          for (int e = 0; e < kCols; ++e) {
            u32x4 vt;  // column (n 16 + r) kCols + e of the 8 positions
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              vt[w] = __builtin_amdgcn_perm(v[2 * w + 1][n][e / 2], v[2 * w][n][e / 2], e % 2 == 0 ? 0x05040100u : 0x07060302u);
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) { o[n * kCols + e] = mfma(T{}, vt, part[i], o[n * kCols + e]); }
          }
        }
      }
      group = next;
    }

    // join the waves, while the next sequence's first loads are in flight
    total = lanes::fold32(total, [](float u, float w) { return u + w; });
    total = lanes::fold16(total, [](float u, float w) { return u + w; });
    __syncthreads();
    if (r < rows) {
      if (g == 0) {
        s_max[wave][r] = top;
        s_sum[wave][r] = total;
      }
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = (n * 16 + g * 4 + i) * kCols;
          if (col < vdim) {
            const int at = FIT != fit::part ? col : min(col, value_off);
#pragma unroll
            for (int e = 0; e < kCols; ++e) { s_out[wave][r][at + e] = o[n * kCols + e][i]; }
          }
        }
      }
    }
    const bool done    = t0 == 0 && t1 == sp.tiles;
    const int64_t out0 = b * a.heads + h0;
    tile += t1 - t0;
    const bool more = tile < last;
    if (t1 == sp.tiles) {
      before += sp.tiles;
      ++b;
    }
    if (more) { begin(); }
    __syncthreads();
    const int64_t slot = (int64_t(table) * plan.shares + share) * 2 + (first ? 0 : 1);
    constexpr int kOnce = kThreads / D;  // rows at a time
    const int col       = tid % D;
    for (int row = tid < kOnce * D ? tid / D : rows; row < rows; row += kOnce) {
      float m = s_max[0][row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) { m = fmaxf(m, s_max[w][row]); }
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = factor_of(plan.scale, s_max[w][row], m);
        sum += f * s_sum[w][row];
        acc += f * s_out[w][row][col];
      }
      if (done) {
        const int64_t at = out0 + row;
        if (col < vdim) { static_cast<T*>(a.out)[at * vdim + col] = T(sum == 0.0f ? 0.0f : acc / sum); }
        if (col == 0 && a.lse != nullptr) {
          a.lse[at] = lse_of(plan.scale, m, sum, kLift<T>);
        }
      } else {
        if (col < vdim) { plan.part_out[(slot * kRows + row) * vdim + col] = acc; }
        if (col == 0) {
          plan.part_max[slot * kRows + row] = m;
          plan.part_sum[slot * kRows + row] = sum;
        }
      }
    }
    if (!more) { break; }
  }
}

/** Whether tables read the same cache lines, so that one die's cache should serve them: several products of
 *  query heads of a key head, or rows of heads that begin within a line. Measured, over all dies and on one: 32
 *  query heads of one key head 147 and 114 us, heads of 80 145 and 131 us; of 128 168 and 174 us. */
bool shares_lines(attend_args const& a, int bytes)
{
  return row_tiles_of(a) > 1 || (a.kv_heads > 1 && (a.k_head * bytes % 128 != 0 || a.v_head * bytes % 128 != 0));
}

}  // namespace

size_t attend_workspace(elem type, attend_args const& a)
{
  const int tile = type == elem::f32 ? kTile<float> : kTile<f16_t>;
  if (longest_of(a) <= tile) { return 0; }  // nothing to cut
  // the most shares that any variant takes
  const size_t slots = size_t(2) * a.kv_heads * row_tiles_of(a) * std::max(shares_for(a, tile, 1), shares_for(a, tile, 2));
  return sizeof(float) * slots * kRows * (a.vdim + 2);
}

void attend(elem type, attend_args const& a, hipStream_t stream)
{
  const int dim       = std::max(a.dim, a.vdim);
  const auto launched = [&](auto tag, auto bucket, auto how) {
    using T         = decltype(tag);
    constexpr int D = decltype(bucket)::value;
    attend_plan plan{divisor(uint32_t(a.pages.page / kGroup<T>))};
    plan.row_tiles  = row_tiles_of(a);
    plan.group      = a.heads / a.kv_heads;
    plan.tables     = a.kv_heads * plan.row_tiles;
    plan.scale      = scale_of(a.shape.any() ? 1.0f : a.scale);
    plan.lift       = kLift<T>;
    plan.slack      = float(std::min(double(kSlack<T>) / double(plan.scale.scale2), double(FLT_MAX)));
    plan.shares     = shares_for(a, kTile<T>, kPerUnit<T, D>);
    // Long shares of 16-bit heads of 128 keep the memory busy with one workgroup per compute unit, and
    // fewer streams are read faster: 64 sequences up to 8,192 168 -> 159 us, one of 131,072 91.6 -> 89.6 us.
    // Short ones need the other workgroup while they begin and end (128 sequences up to 1,000: 57 and 65 us),
    // as do smaller steps (heads of 64: 177 and 200 us; float32: 156 and 182 us).
    plan.halve          = sizeof(T) == 2 && D == 128 && plan.row_tiles == 1 ? 32 : 0;
    const int64_t slots = int64_t(2) * plan.tables * plan.shares * kRows;
    plan.part_out   = static_cast<float*>(a.workspace);
    plan.part_max   = plan.part_out + slots * a.vdim;
    plan.part_sum   = plan.part_max + slots;
    plan.one_die        = shares_lines(a, sizeof(T)) && plan.shares >= 8;
    const int blocks    = (plan.one_die ? (plan.shares + 7) / 8 * 8 : plan.shares) * plan.tables;
    if (a.shape.any()) {
      attend_kernel<T, D, decltype(how)::value, true><<<dim3(uint32_t(blocks)), kThreads, 0, stream>>>(a, plan);
    } else {
      attend_kernel<T, D, decltype(how)::value, false><<<dim3(uint32_t(blocks)), kThreads, 0, stream>>>(a, plan);
    }
    if (longest_of(a) > kTile<T>) {
      const dim3 grid(uint32_t(a.heads), uint32_t(a.pages.sequences));
      // a few partials per sequence, or many (64 sequences: 13 us with 512 threads, 6 with 128)
      if (plan.shares <= 8 * a.pages.sequences) {
        join_kernel<T, 128, kTile<T>><<<grid, 128, 0, stream>>>(a, plan);
      } else {
        join_kernel<T, 512, kTile<T>><<<grid, 512, 0, stream>>>(a, plan);
      }
    }
  };
  const auto sized = [&](auto tag) {
    using full = std::integral_constant<fit, fit::full>;
    using part = std::integral_constant<fit, fit::part>;
    using tiny = std::integral_constant<fit, fit::tiny>;
    const auto bucket = [&](auto d) {
      constexpr int D = decltype(d)::value;
      a.dim == D && a.vdim == D ? launched(tag, d, full{}) : launched(tag, d, part{});
    };
    if (std::min(a.dim, a.vdim) < 8) {
      dim <= 64 ? launched(tag, std::integral_constant<int, 64>{}, tiny{}) : launched(tag, std::integral_constant<int, 256>{}, tiny{});
    } else if (dim <= 64) {
      bucket(std::integral_constant<int, 64>{});
    } else if (dim <= 96) {
      bucket(std::integral_constant<int, 96>{});
    } else if (dim <= 128) {
      bucket(std::integral_constant<int, 128>{});
    } else {
      bucket(std::integral_constant<int, 256>{});
    }
  };
  switch (type) {
    case elem::f32: sized(float{}); break;
    case elem::f16: sized(f16_t{}); break;
    case elem::bf16: sized(bf16_t{}); break;
  }
}

}  // namespace certex_amd::attention
