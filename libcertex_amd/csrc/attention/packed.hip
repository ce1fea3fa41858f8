// Attention of one new token of every sequence over its 4-bit pages (their layout: packed_pages).
//
// out = sum_t p_t v_t / sum_t p_t with p_t = 2^(log2(e) (x_t - m)); with scales s, offsets o and codes n per group of 64 dimensions
//   q.k_t = sum_group s_t (sum_d q_d n_td) + o_t (sum_d q_d),    sum_t p_t v_td = sum_t (p_t s_t) n_td + sum_t p_t o_t.
// The sums over codes go to the matrix cores as float16 products: a code n in bits 4 to 7 of a halfword is the subnormal
// float16 n 2^-20. So two codes become operands by an AND (and three of four a shift), nothing is converted, and the power of two is
// taken back where sums are used.
//
// What bounds it: 144 bytes of a position and head of 128 (codes 128, scales and offsets 16), read once. In the kernel as it is
// no unit is full: for 32 positions a wave has some 420 vector instructions (float32 queries 620), which take 54 percent of the vector
// units' time (57), the matrix units are busy 13 percent (15), memory is read at 0.62 of its rate. The 3 waves of a SIMD (2) wait 33
// percent of theirs (30) for LDS and memory, and registers hold no more.
//
// The shape of the products is that of attend.hip: a wave takes 32 positions, 8 to a lane group, and holds of each product's result
// the positions that it feeds to the next. A record holds 8 positions of a head, so that a lane group's codes, scales and
// offsets are one piece of memory.
// - Queries enter as float16, scaled by a power of two that brings a row's largest to [2^13, 2^14): 16-bit types whole
//   (what is 2^-28 of the largest loses bits, none that float32 sums would keep), float32 as three elements of 11 bits.
// - p_t s_t enters as two elements of 11 bits, the nearest float16 and what it leaves: 2^-21 of it off at most. (One element
//   would be 2^-11 off, as much as float16 outputs are rounded; 64 sequences 57 us instead of 63.) p's reference is
//   kept such that the largest is below 2^15. Their sum is not rounded. The elements reach down to 2^-24: positions and
//   groups lose bits, one for each power of 2, whose p_t s_t are below 2^-16 of what the largest scale so far makes the largest.
// - Products of subnormal numbers keep fewer of their low bits beside large sums, the fewer the smaller they are: codes in bits 0 to
//   3, as n 2^-24, were 2e-6 to 5e-6 of the values off (64 sequences 63 us instead of 65). float32 takes other
//   codes: less 8, as normal numbers (two operations more each), whose sums stay small; and joins steps outside the products.
// Work is dealt as in attend.hip (shares.hpp). A wave copies its next step to LDS while it works on one, by itself: what it
// copies it alone reads, so that steps need no barrier.
//
// Measured (8 key heads of 128, 32 query heads): 64 sequences up to 8,192 of bfloat16 queries, 0.26 GB of records: 65 us
// and 6 for the join, 4.0 TB/s; a call 73 us, capped 85, leaning 75;
// one sequence of 131,072, float32 queries, 0.15 GB: 53 us and 6, 7e-7 off; 77 positions
// 8.7 us, launch and five dependent loads.
#include "scores.hpp"
#include "shares.hpp"
#include "tiles.hpp"

namespace certex_amd::attention {
namespace {

constexpr int kTile = 32 * kWaves;  // positions of a workgroup's step

using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using u16x2 = __attribute__((ext_vector_type(2))) uint16_t;

/** The reference may lag the largest exponent by this much. */
constexpr float kSlack = 1.0f;
/** Products p s stay below 2^kRoom times 2^kSlack. */
constexpr int kRoom = 13;

struct packed_plan {
  attend_plan at;
  elem type;
};

/** Workgroups per compute unit: as many as registers and LDS hold without spilling. (One more at 4 chunks spills: 64 sequences
 *  66 us instead of 61.) */
constexpr int per_unit(int chunks, bool full, int parts)
{
  return chunks <= 2 ? 4 : chunks == 3 ? (full ? 3 : 2) : chunks == 4 ? (full && parts == 1 ? 3 : 2) : full && parts == 1 ? 2 : 1;
}

/** Bytes of a record of C chunks of dimensions on both sides: the most that a kernel's records take. */
template <int C>
constexpr int kRecord = 256 * C + 64 * ((C + 1) / 2);

/** A wave's steps in LDS: one that is worked on, one that is on its way. */
constexpr int kBuffers = 2;

typedef const __attribute__((address_space(4))) int32_t* constant_ints;

/** Waits until at most n of this wave's copies are on their way (n as they are issued: 0, or those of one step). */
__device__ __forceinline__ void landed(int n)
{
  switch (n) {
    case 0: asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); break;
    case 1: asm volatile("s_waitcnt vmcnt(1)" ::: "memory"); break;
    case 2: asm volatile("s_waitcnt vmcnt(2)" ::: "memory"); break;
    case 3: asm volatile("s_waitcnt vmcnt(3)" ::: "memory"); break;
    case 4: asm volatile("s_waitcnt vmcnt(4)" ::: "memory"); break;
    case 5: asm volatile("s_waitcnt vmcnt(5)" ::: "memory"); break;
    case 6: asm volatile("s_waitcnt vmcnt(6)" ::: "memory"); break;
    case 7: asm volatile("s_waitcnt vmcnt(7)" ::: "memory"); break;
    case 8: asm volatile("s_waitcnt vmcnt(8)" ::: "memory"); break;
    default: asm volatile("s_waitcnt vmcnt(9)" ::: "memory"); break;  // and any larger number
  }
}

/** N words of LDS, which begin at a multiple of ALIGN words. */
template <int N, int ALIGN>
__device__ __forceinline__ void read_words(uint32_t* to, const uint8_t* from)
{
  __builtin_memcpy(to, __builtin_assume_aligned(from, 4 * ALIGN), 4 * N);
}

__device__ __forceinline__ float half_of(uint32_t w, int i)
{
  return float(__builtin_bit_cast(f16x2, w)[i]);
}

/** The codes in bits 4 to 7 of a word's halves as float16 of kCode each, subnormal: no conversion. */
constexpr float kCode = 0x1p-20f;
__device__ __forceinline__ uint32_t opened(uint32_t w) { return w & 0x00f000f0u; }

/** The codes in the low 4 bits of a word's halves, less 8, as float16: 1024 + code is the number with the code in its last bits. */
__device__ __forceinline__ uint32_t less_eight(uint32_t w)
{
  const f16x2 far = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x64006400u);
  return __builtin_bit_cast(uint32_t, far - f16x2{1032.0f, 1032.0f});
}

/** Elements [d, d + 8) of a query of dim elements, in float32. */
__device__ __forceinline__ void load_query(elem type, const void* q, int64_t at, int d, int dim, float* out)
{
#pragma unroll
  for (int i = 0; i < 8; ++i) { out[i] = 0.0f; }
  if (d >= dim) { return; }
  const auto load = [&](auto tag) {
    using T      = decltype(tag);
    const T* row = static_cast<const T*>(q) + at;
    if (d + 8 <= dim) {
      T e[8];
      __builtin_memcpy(e, __builtin_assume_aligned(row + d, sizeof(T)), sizeof(e));
#pragma unroll
      for (int i = 0; i < 8; ++i) { out[i] = float(e[i]); }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) { out[i] = d + i < dim ? float(row[d + i]) : 0.0f; }
    }
  };
  switch (type) {
    case elem::f32: load(float{}); break;
    case elem::f16: load(f16_t{}); break;
    case elem::bf16: load(bf16_t{}); break;
  }
}

/** C chunks of 32 dimensions; FULL: of keys and of values alike, else at most. P: elements that a query enters as. */
template <int C, bool FULL, int P>
__global__ __launch_bounds__(kThreads, per_unit(C, FULL, P)) void packed_kernel(packed_args args, packed_plan pp)
{
  constexpr int G = (C + 1) / 2;  // groups
  constexpr int D = 32 * C;
  constexpr bool FINE = P > 1;  // float32: more of the products' low bits
  // the waves' steps, then their outputs
  __shared__ __attribute__((aligned(16))) uint8_t s_steps[kWaves][kBuffers][4 * kRecord<C>];
  static_assert(sizeof(float) * kRows * D <= sizeof(s_steps[0]));
  __shared__ float s_max[kWaves][kRows], s_sum[kWaves][kRows];
  attend_args const& a    = args.a;
  attend_plan const& plan = pp.at;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, g = lane / 16;
  // consecutive workgroups go to the 8 dies in turn: a share's tables to all of them, or to one
  const int turn      = plan.one_die ? blockIdx.x / 8 : blockIdx.x;
  const int table     = turn % plan.tables;
  const int64_t share = plan.one_die ? int64_t(turn / plan.tables) * 8 + blockIdx.x % 8 : turn / plan.tables;

  const auto put = [&](int64_t at, float x) {
    switch (pp.type) {
      case elem::f32: static_cast<float*>(a.out)[at] = x; break;
      case elem::f16: static_cast<f16_t*>(a.out)[at] = f16_t(x); break;
      case elem::bf16: static_cast<bf16_t*>(a.out)[at] = bf16_t(x); break;
    }
  };
  const shares sh = shares_of<kTile>(a, plan);
  // rows without a position
  for (int64_t b = blockIdx.x; b < a.pages.sequences; b += gridDim.x) {
    if (span_of<kTile>(a, b).tiles == 0) {
      for (int i = tid; i < a.heads * a.vdim; i += kThreads) { put(b * a.heads * a.vdim + i, 0.0f); }
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
    const int mine    = b0 + lane < a.pages.sequences ? span_of<kTile>(a, b0 + lane).tiles : 0;
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

  const int dim = FULL ? D : a.dim, vdim = FULL ? D : a.vdim;
  const int k_chunks = FULL ? C : packed_chunks(dim), v_chunks = FULL ? C : packed_chunks(vdim);
  const int k_groups = (k_chunks + 1) / 2, v_groups = (v_chunks + 1) / 2;
  const int k_bytes  = 128 * k_chunks + 32 * k_groups, record = k_bytes + 128 * v_chunks + 32 * v_groups;
  const int kv = table % a.kv_heads, row0 = table / a.kv_heads * kRows;
  const int rows = min(kRows, plan.group - row0), h0 = kv * plan.group + row0;
  const float slope    = a.shape.slopes != nullptr ? a.shape.slopes[h0 + min(r, rows - 1)] : 0.0f;
  const float per_cap  = a.shape.cap != 0.0f ? a.scale / a.shape.cap : 0.0f;
  const bool bends     = a.shape.cap != 0.0f || a.shape.slopes != nullptr;
  const int per_page   = int(plan.page_groups.d);  // records
  const int64_t head   = int64_t(record) * per_page, page_bytes = head * a.kv_heads;
  const uint8_t* pool  = args.pages.p + kv * head;

  span sp{};
  int t0 = 0, t1 = 0, group = 0, stop = 0, final = 0;
  constant_ints pages = nullptr;
  // where a step's 4 records begin; bit per record: the sequence has its page
  struct place {
    const uint8_t* p[4];
    uint32_t there;
  };
  // the records of a step follow one another if pages hold whole steps and the sequence's first step begins one
  bool follow = false;
  const auto entry = [&](int at, const uint8_t** p) {
    at             = min(at, final);
    const int e    = int(plan.page_groups(uint32_t(at)));
    const int page = pages[e];
    const bool there = uint32_t(page) < uint32_t(a.pages.n_pages);
    *p = pool + (there ? page : 0) * page_bytes + int64_t(at - e * per_page) * record;
    return there;
  };
  const auto look_up = [&](int group) {
    place at{};
    if (follow) {
      at.there = entry(group, &at.p[0]) ? 15u : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) { at.there |= uint32_t(entry(group + i, &at.p[i])) << i; }
    }
    return at;
  };
  /** The copies of a step, and how many they are. */
  const auto copy = [&](place const& at, int buffer) {
    const uint32_t to = lds_address(&s_steps[wave][buffer][0]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what was read there has arrived
    int n = 0;
    if (follow) {
      for (int from = 0; from < 4 * record; from += 1024, ++n) {
        if (from + lane * 16 < 4 * record) { copy_to_lds(at.p[0] + from, lane * 16, to + from); }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        for (int from = 0; from < record; from += 1024, ++n) {
          if (from + lane * 16 < record) { copy_to_lds(at.p[i] + from, lane * 16, to + i * record + from); }
        }
      }
    }
    return n;
  };
  place here{}, next_at{};
  // the share's tiles of sequence b (or of the next that has any): their range, and the first step's copies
  const auto begin = [&] {
    for (sp = span_of<kTile>(a, b); sp.tiles == 0; sp = span_of<kTile>(a, b)) { ++b; }
    sp     = {uniform(sp.begin), uniform(sp.end), uniform(sp.tiles)};
    t0     = uniform(int(tile - before));
    t1     = uniform(int(min(int64_t(sp.tiles), t0 + last - tile)));
    pages  = (constant_ints)uniform(a.pages.table + b * a.pages.width);
    final  = (sp.end - 1) / 8;
    group  = sp.begin / 8 + (t0 * kWaves + wave) * 4;
    stop   = min(sp.begin / 8 + t1 * kWaves * 4, final + 1);
    follow = per_page % 4 == 0 && sp.begin / 8 % 4 == 0;
    if (group < stop) {
      here = look_up(group);
      copy(here, 0);
      if (group + kWaves * 4 < stop) { next_at = look_up(group + kWaves * 4); }
    }
  };

  begin();
  for (bool first = true;; first = false) {
    // the queries: column r, the dimensions 32 c + 8 g + 0..7, scaled by a power of two
    u32x4 q[C][P];
    float q_sum[G];  // of a group's elements, in units of a product
    int exponent;
    {
      float e[C][8];
      float largest = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        load_query(pp.type, a.q, b * a.q_seq + (h0 + min(r, rows - 1)) * a.q_head, c * 32 + g * 8, dim, e[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) { largest = fmaxf(largest, __builtin_fabsf(e[c][i])); }
      }
      const auto larger = [](float u, float w) { return fmaxf(u, w); };
      largest  = lanes::fold16(lanes::fold32(largest, larger), larger);
      exponent = largest > 0.0f && largest < INFINITY ? __builtin_amdgcn_frexp_expf(largest) - 14 : 0;
#pragma unroll
      for (int n = 0; n < G; ++n) { q_sum[n] = 0.0f; }
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[c][i] = r < rows ? __builtin_amdgcn_ldexpf(plan.scale.sign * e[c][i], -exponent) : 0.0f;
          q_sum[c / 2] += e[c][i];
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float lo = e[c][2 * w], hi = e[c][2 * w + 1];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            q[c][i][w] = pack2<f16_t>(lo, hi);
            lo -= float(f16_t(lo));
            hi -= float(f16_t(hi));
          }
        }
      }
      const auto plus = [](float u, float w) { return u + w; };
#pragma unroll
      for (int n = 0; n < G; ++n) { q_sum[n] = lanes::fold16(lanes::fold32(q_sum[n], plus), plus) * (FINE ? 1.0f : kCode); }
      exponent += FINE ? 0 : 20;  // what kCode takes
    }
    f32x4 o[C][2];   // tiles of 16 columns: chunk c of V's units, even and odd dimensions of a pair
    float shift[G];  // sum of p times the offsets, of this lane's positions
#pragma unroll
    for (int c = 0; c < C; ++c) { o[c][0] = o[c][1] = f32x4{0, 0, 0, 0}; }
#pragma unroll
    for (int n = 0; n < G; ++n) { shift[n] = 0.0f; }
    float top = -INFINITY, limit = -INFINITY, base = 0.0f, total = 0.0f;
    // p is taken 2^lift times; scales so far are below 2^(kRoom - lift)
    int lift          = kRoom + 23;
    float scale_limit = __builtin_amdgcn_ldexpf(1.0f, kRoom - lift);

    int buffer = 0;
    while (group < stop) {
      const int next = group + kWaves * 4;
      const uint32_t there = here.there;
      int coming = 0;
      if (next < stop) {
        coming = copy(next_at, 1 - buffer);
        here   = next_at;
        if (next + kWaves * 4 < stop) { next_at = look_up(next + kWaves * 4); }
      }
      landed(coming);
      const bool have       = (there >> g & 1u) != 0;
      const uint8_t* rows_  = &s_steps[wave][buffer][r / 4 * record];  // of the product's row
      const uint8_t* mine   = &s_steps[wave][buffer][g * record];      // of the positions that this lane weighs
      const uint8_t* values = mine + k_bytes;
      f32x4 s[2][G];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int n = 0; n < G; ++n) { s[half][n] = f32x4{0, 0, 0, 0}; }
        uint32_t k[C];
        read_words<C, packed_key_align(C, FULL)>(
          k, FULL ? rows_ + (half * 4 + r % 4) * 16 * C + g * 4 * C : rows_ + (half * 4 + r % 4) * 16 * k_chunks + g * 4 * k_chunks);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const uint32_t w = k[c];
          const u32x4 codes = FINE ? u32x4{less_eight(w), less_eight(w >> 4), less_eight(w >> 8), less_eight(w >> 12)}
                                   : u32x4{opened(w << 4), opened(w), opened(w >> 4), opened(w >> 8)};
#pragma unroll
          for (int i = P - 1; i >= 0; --i) { s[half][c / 2] = mfma(f16_t{}, codes, q[c][i], s[half][c / 2]); }
        }
      }
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) { x[j] = 0.0f; }
#pragma unroll
      for (int n = 0; n < G; ++n) {
        if (!FULL && n >= k_groups) { break; }
        uint32_t scales[4], offsets[4];
        read_words<4, 4>(scales, mine + 128 * k_chunks + n * 32);
        read_words<4, 4>(offsets, mine + 128 * k_chunks + n * 32 + 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float scale = half_of(scales[j / 2], j % 2), sum = s[j / 4][n][j % 4];
          x[j] = __builtin_fmaf(scale, FINE ? __builtin_fmaf(8.0f, q_sum[n], sum) : sum,
                                __builtin_fmaf(half_of(offsets[j / 2], j % 2), q_sum[n], x[j]));
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) { x[j] = __builtin_amdgcn_ldexpf(x[j], exponent); }
      uint32_t vs[G][4], vo[G][4];
#pragma unroll
      for (int n = 0; n < G; ++n) {
#pragma unroll
        for (int w = 0; w < 4; ++w) { vs[n][w] = vo[n][w] = 0; }
        if (FULL || n < v_groups) {
          read_words<4, 4>(vs[n], values + 128 * v_chunks + n * 32);
          read_words<4, 4>(vo[n], values + 128 * v_chunks + n * 32 + 16);
        }
      }
      const uint32_t t = uint32_t(group + g) * 8;  // past the end it may pass 2^31
      const uint32_t t_begin = uint32_t(sp.begin), t_end = uint32_t(sp.end);
      if (bends) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = bent(x[j], a.scale, per_cap, a.shape.cap, slope, float(t_end - 1u - (t + j)));
        }
      }
      const bool masked = !__all(have && t >= t_begin && t + 8 <= t_end);
      if (masked) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = have && t + j >= t_begin && t + j < t_end;
          x[j]          = in ? x[j] : -INFINITY;
          const uint32_t keep = in ? 0xffffffffu : j % 2 == 0 ? 0xffff0000u : 0x0000ffffu;
#pragma unroll
          for (int n = 0; n < G; ++n) {
            vs[n][j / 2] &= keep;
            vo[n][j / 2] &= keep;
          }
        }
      }
      float high = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) { high = fmaxf(high, x[j]); }
      // the largest of the scales, which are not negative: as whole numbers, of which NaN is the largest
      u16x2 most = __builtin_bit_cast(u16x2, vs[0][0]);
#pragma unroll
      for (int n = 0; n < G; ++n) {
#pragma unroll
        for (int w = n == 0 ? 1 : 0; w < 4; ++w) { most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, vs[n][w])); }
      }
      const float even = half_of(__builtin_bit_cast(uint32_t, most), 0), odd = half_of(__builtin_bit_cast(uint32_t, most), 1);
      const bool hidden = __builtin_isunordered(even, odd);  // scales below a NaN, which is no steeper than any
      float steep       = fmaxf(even, odd);
      if (__any(high > limit || steep >= scale_limit || hidden)) {
        if (hidden) {
#pragma unroll
          for (int n = 0; n < G; ++n) {
#pragma unroll
            for (int w = 0; w < 4; ++w) { steep = fmaxf(steep, fmaxf(half_of(vs[n][w], 0), half_of(vs[n][w], 1))); }
          }
        }
        const auto larger = [](float u, float w) { return fmaxf(u, w); };
        high              = lanes::fold16(lanes::fold32(high, larger), larger);
        const float grown = fmaxf(top, high);
        float keep        = grown == -INFINITY ? 0.0f : weight_of(plan.scale, top, grown);
        const float widest = lanes::fold16(lanes::fold32(steep, larger), larger);
        if (widest >= scale_limit) {
          const int less = widest < INFINITY ? kRoom - __builtin_amdgcn_frexp_expf(widest) : kRoom - 17;
          keep           = __builtin_amdgcn_ldexpf(keep, less - lift);
          lift           = less;
          scale_limit    = widest < INFINITY ? __builtin_amdgcn_ldexpf(1.0f, kRoom - lift) : INFINITY;
        }
        total *= keep;
#pragma unroll
        for (int c = 0; c < C; ++c) { o[c][0] *= keep, o[c][1] *= keep; }
#pragma unroll
        for (int n = 0; n < G; ++n) { shift[n] *= keep; }
        top   = grown;
        limit = grown + plan.slack;
        // with a scale of 0 all weigh alike, wherever the scores are
        base = grown == -INFINITY || plan.scale.scale2 == 0.0f ? 0.0f : grown;
      }
      float p[8];
      if (masked && plan.scale.scale2 == 0.0f) {  // what is masked is no number times 0
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = x[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(x[j] - base, 0.0f, float(lift)));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j] - base, plan.scale.scale2, float(lift)));
        }
      }
#pragma unroll
      for (int j = 0; j < 8; j += 4) { total += (p[j] + p[j + 1]) + (p[j + 2] + p[j + 3]); }
#pragma unroll
      for (int n = 0; n < G; ++n) {
        if (!FULL && n >= v_groups) { break; }
        // p s of the group in the order of the codes' words (0, 2), (1, 3), (4, 6), (5, 7): the nearest, and what it leaves
        u32x4 part[2];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int j = w / 2 * 4 + w % 2;
          float lo = __builtin_fmaf(p[j], half_of(vs[n][j / 2], j % 2), 0.0f);
          float hi = __builtin_fmaf(p[j + 2], half_of(vs[n][j / 2 + 1], j % 2), 0.0f);
          // offsets of codes that are less 8
          if (FINE) { shift[n] = __builtin_fmaf(8.0f, hi, __builtin_fmaf(8.0f, lo, shift[n])); }
          shift[n] = __builtin_fmaf(p[j], half_of(vo[n][j / 2], j % 2), shift[n]);
          shift[n] = __builtin_fmaf(p[j + 2], half_of(vo[n][j / 2 + 1], j % 2), shift[n]);
          part[0][w] = pack2<f16_t>(lo, hi);
          lo         = __builtin_fmaf(half_of(part[0][w], 0), -1.0f, lo);
          hi         = __builtin_fmaf(half_of(part[0][w], 1), -1.0f, hi);
          part[1][w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
        }
        uint32_t v[4] = {0, 0, 0, 0};
        const bool pair = 2 * n + 1 < C && (FULL || 2 * n + 1 < v_chunks);  // a unit of 64 dimensions, else of 32
        if (pair) {
          read_words<4, 4>(v, values + n * 256 + r * 16);
        } else {
          read_words<2, 2>(v, values + n * 256 + r * 8);
        }
#pragma unroll
        for (int c = 2 * n; c < 2 * n + 2 && c < C; ++c) {
          const uint32_t w0 = v[c % 2 * 2], w1 = v[c % 2 * 2 + 1];
          if (FINE) {
            const u32x4 even{less_eight(w0), less_eight(w0 >> 8), less_eight(w1), less_eight(w1 >> 8)};
            const u32x4 odd{less_eight(w0 >> 4), less_eight(w0 >> 12), less_eight(w1 >> 4), less_eight(w1 >> 12)};
            const f32x4 zero{0, 0, 0, 0};
            o[c][0] += mfma(f16_t{}, even, part[0], mfma(f16_t{}, even, part[1], zero));
            o[c][1] += mfma(f16_t{}, odd, part[0], mfma(f16_t{}, odd, part[1], zero));
          } else {
            const u32x4 even{opened(w0 << 4), opened(w0 >> 4), opened(w1 << 4), opened(w1 >> 4)};
            const u32x4 odd{opened(w0), opened(w0 >> 8), opened(w1), opened(w1 >> 8)};
            o[c][0] = mfma(f16_t{}, even, part[0], mfma(f16_t{}, even, part[1], o[c][0]));
            o[c][1] = mfma(f16_t{}, odd, part[0], mfma(f16_t{}, odd, part[1], o[c][1]));
          }
        }
      }
      group  = next;
      buffer = 1 - buffer;
    }

    // join the waves; their outputs take the place of their steps
    const auto plus = [](float u, float w) { return u + w; };
    total = __builtin_amdgcn_ldexpf(lanes::fold16(lanes::fold32(total, plus), plus), -lift);
#pragma unroll
    for (int n = 0; n < G; ++n) { shift[n] = __builtin_amdgcn_ldexpf(lanes::fold16(lanes::fold32(shift[n], plus), plus), -lift); }
    if (r < rows) {
      float* out = reinterpret_cast<float*>(&s_steps[wave][0][0]);
      if (g == 0) {
        s_max[wave][r] = top;
        s_sum[wave][r] = total;
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int unit  = c / 2;
        const bool pair = 2 * unit + 1 < C && (FULL || 2 * unit + 1 < v_chunks);  // a unit of 64 dimensions, else of 32
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = g * 4 + i, col = unit * 64 + (pair ? row * 4 + c % 2 * 2 : row * 2) + e;
            if ((pair || c % 2 == 0) && col < vdim) {
              out[r * D + col] = __builtin_amdgcn_ldexpf(o[c][e][i], (FINE ? 0 : 20) - lift) + shift[unit];
            }
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
    __syncthreads();
    const int64_t slot = (int64_t(table) * plan.shares + share) * 2 + (first ? 0 : 1);
    for (int at = tid; at < rows * vdim; at += kThreads) {
      const int row = at / vdim, col = at - row * vdim;
      float m = s_max[0][row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) { m = fmaxf(m, s_max[w][row]); }
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = factor_of(plan.scale, s_max[w][row], m);
        sum += f * s_sum[w][row];
        acc += f * reinterpret_cast<const float*>(&s_steps[w][0][0])[row * D + col];
      }
      if (done) {
        put((out0 + row) * vdim + col, sum == 0.0f ? 0.0f : acc / sum);
        if (col == 0 && a.lse != nullptr) { a.lse[out0 + row] = lse_of(plan.scale, m, sum); }
      } else {
        plan.part_out[(slot * kRows + row) * vdim + col] = acc;
        if (col == 0) {
          plan.part_max[slot * kRows + row] = m;
          plan.part_sum[slot * kRows + row] = sum;
        }
      }
    }
    if (!more) { break; }
    __syncthreads();
    begin();
  }
}

int per_unit_of(elem type, attend_args const& a)
{
  const int chunks = packed_chunks(std::max(a.dim, a.vdim));
  return per_unit(chunks, a.dim == 32 * chunks && a.vdim == 32 * chunks, type == elem::f32 ? 3 : 1);
}

}  // namespace

size_t packed_workspace(elem type, packed_args const& args)
{
  attend_args const& a = args.a;
  if (longest_of(a) <= kTile) { return 0; }  // nothing to cut
  const size_t slots = size_t(2) * a.kv_heads * row_tiles_of(a) * shares_for(a, kTile, per_unit_of(type, a));
  return sizeof(float) * slots * kRows * (a.vdim + 2);
}

void packed_attend(elem type, packed_args const& args, hipStream_t stream)
{
  attend_args const& a = args.a;
  const auto launched  = [&](auto chunks, auto full, auto parts) {
    constexpr int C = decltype(chunks)::value;
    packed_plan pp{{divisor(uint32_t(a.pages.page / 8))}, type};
    attend_plan& plan   = pp.at;
    plan.row_tiles      = row_tiles_of(a);
    plan.group          = a.heads / a.kv_heads;
    plan.tables         = a.kv_heads * plan.row_tiles;
    plan.scale          = scale_of(a.shape.any() ? 1.0f : a.scale);
    plan.lift           = 0.0f;
    plan.slack          = float(std::min(double(kSlack) / double(plan.scale.scale2), double(FLT_MAX)));
    plan.shares         = shares_for(a, kTile, per_unit_of(type, a));
    plan.halve          = 0;
    const int64_t slots = int64_t(2) * plan.tables * plan.shares * kRows;
    plan.part_out       = static_cast<float*>(a.workspace);
    plan.part_max       = plan.part_out + slots * a.vdim;
    plan.part_sum       = plan.part_max + slots;
    plan.one_die        = plan.row_tiles > 1 && plan.shares >= 8;
    const int blocks    = (plan.one_die ? (plan.shares + 7) / 8 * 8 : plan.shares) * plan.tables;
    packed_kernel<C, decltype(full)::value, decltype(parts)::value><<<dim3(uint32_t(blocks)), kThreads, 0, stream>>>(args, pp);
    if (longest_of(a) > kTile) {
      const dim3 grid(uint32_t(a.heads), uint32_t(a.pages.sequences));
      const auto join = [&](auto tag) {
        using T = decltype(tag);
        // a few partials per sequence, or many
        if (plan.shares <= 8 * a.pages.sequences) {
          join_kernel<T, 128, kTile><<<grid, 128, 0, stream>>>(a, plan);
        } else {
          join_kernel<T, 512, kTile><<<grid, 512, 0, stream>>>(a, plan);
        }
      };
      switch (type) {
        case elem::f32: join(float{}); break;
        case elem::f16: join(f16_t{}); break;
        case elem::bf16: join(bf16_t{}); break;
      }
    }
  };
  const auto filled = [&](auto chunks, auto full) {
    type == elem::f32 ? launched(chunks, full, std::integral_constant<int, 3>{})
                      : launched(chunks, full, std::integral_constant<int, 1>{});
  };
  const auto sized = [&](auto chunks) {
    constexpr int C = decltype(chunks)::value;
    a.dim == 32 * C && a.vdim == 32 * C ? filled(chunks, std::true_type{}) : filled(chunks, std::false_type{});
  };
  switch (packed_chunks(std::max(a.dim, a.vdim))) {
    case 2: sized(std::integral_constant<int, 2>{}); break;
    case 3: sized(std::integral_constant<int, 3>{}); break;
    case 4: sized(std::integral_constant<int, 4>{}); break;
    case 6: sized(std::integral_constant<int, 6>{}); break;
    default: sized(std::integral_constant<int, 8>{}); break;
  }
}

}  // namespace certex_amd::attention
