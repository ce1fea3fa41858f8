// Rotation by position, and its fusion with the append to a paged cache.
//
// Position p turns pair i of a head by the angle p f_i: (a, b) -> m (a cos - b sin, a sin + b cos).
// The frequencies are kept in turns as 64-bit fixed point, so p f_i modulo one turn is the low half
// of one integer product: exact for every position, where a float32 product loses the angle (at
// position 131,072 it is 0.008 radians off), and nothing is read from a table. The top 24 bits of
// the fraction go to sin and cos of half turns as they are, the next 8 turn the result by their small angle, so that the
// angle costs the sines less than their own rounding.
//
// What bounds it: every element is read and written once. A thread takes one vector of a row over several heads of a token,
// so that sines are computed once for up to 8 heads. Measured, the kernel alone: 131,072 tokens x 8 heads of 128 bfloat16,
// 0.54 GB: 82 us, 6.5 TB/s (with fresh outputs in turn 96 us a pass, where torch's clone of as much takes 99); prompts of
// 15,443 tokens appended with their queries, 190 MB: 33 us, 5.7 TB/s; 64 queries of a step 4.8 us, their append 5.2 us:
// launch and three dependent loads.
#include "attention.hpp"
#include "elements.hpp"
#include "turn.hpp"

#include <algorithm>
#include <numeric>
#include <stdexcept>

namespace certex_amd::attention {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch   = 4;

/**
 * One thread: one vector of V elements of a row (of both halves in the half layout), over
 * heads_per_thread heads of one token. Blocks are dealt to the jobs in order. LOOSE: rows of any
 * length and alignment; what is turned and what is copied each end in a vector that is moved back to fit and
 * writes some elements a second time, as they were written the first.
 */
template <typename T, int V, bool INTERLEAVED, bool LOOSE>
__global__ __launch_bounds__(kThreads) void turn_kernel(turn_args a)
{
  int64_t block = blockIdx.x;
  int j         = 0;
  while (j + 1 < a.jobs && block >= a.job[j].blocks) { block -= a.job[j++].blocks; }
  const turn_job& b = a.job[j];
  const uint64_t at = uint64_t(block) * kThreads + threadIdx.x;
  uint32_t item, group;
  uint64_t token;
  if (b.blocks < (int64_t(1) << 23)) {  // 32-bit quotients
    const uint32_t row = uint32_t(at) / uint32_t(b.items);
    item               = uint32_t(at) - row * uint32_t(b.items);
    token              = row / uint32_t(b.groups);
    group              = row - uint32_t(token) * uint32_t(b.groups);
  } else {
    const uint64_t row = at / uint64_t(b.items);
    item               = uint32_t(at - row * uint64_t(b.items));
    token              = row / uint64_t(b.groups);
    group              = uint32_t(row - token * uint64_t(b.groups));
  }
  if (token >= uint64_t(a.tokens)) { return; }
  const uint64_t outer = a.inner == a.tokens ? 0 : token / uint64_t(a.inner);
  const uint64_t inner = token - outer * uint64_t(a.inner);
  const int64_t p      = a.positions[int64_t(token)];

  const T* src = static_cast<const T*>(b.src) + int64_t(outer) * b.src_outer + int64_t(inner) * b.src_token;
  T* dst       = static_cast<T*>(b.dst);
  if (b.paged) {
    const int64_t s = a.sequences.p != nullptr ? a.sequences[int64_t(token)] : int64_t(token);
    if (s < 0 || s >= a.pages.sequences || p < 0 || p >= int64_t(a.pages.width) * a.pages.page) { return; }
    const uint32_t entry = uint32_t(p) / uint32_t(a.pages.page);
    const uint32_t slot  = uint32_t(p) - entry * uint32_t(a.pages.page);
    const int32_t page   = a.pages.table[s * a.pages.width + entry];
    if (page < 0 || page >= a.pages.n_pages) { return; }
    dst += int64_t(page) * b.dst_outer + int64_t(slot) * b.dst_token;
  } else {
    dst += int64_t(outer) * b.dst_outer + int64_t(inner) * b.dst_token;
  }
  const int h0 = int(group) * a.heads_per_thread;
  const int h1 = min(h0 + a.heads_per_thread, b.heads);

  constexpr bool kAdjacent = INTERLEAVED && V > 1;   // pairs within a vector; else two vectors
  constexpr int P          = kAdjacent ? V / 2 : V;  // pairs of a thread
  const bool turned        = item < uint32_t(b.turned);  // else a vector that is copied
  const int second         = INTERLEAVED ? 1 : b.rotary / 2;  // from the first
  int first                = turned ? int(item) * (INTERLEAVED && V == 1 ? 2 : V) : int(item - uint32_t(b.turned)) * V;
  if constexpr (LOOSE) { first = min(first, (turned ? (INTERLEAVED ? b.rotary : b.rotary / 2) : b.dim - b.rotary) - V); }
  const int pair = INTERLEAVED ? first / 2 : first;
  if (!turned) { first += b.rotary; }
  src += first;
  dst += first;
  // the rows of kBatch heads are in flight together
  pack<T, V> x[kBatch], y[kBatch];
  const auto take = [&](int h, auto one) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const T* row = src + min(h + i, h1 - 1) * b.src_head;
      x[i]         = one(row);
      if (!kAdjacent && turned) { y[i] = one(row + second); }
    }
  };
  const auto take_heads = [&](int h) {
    if constexpr (LOOSE) {
      take(h, [](const T* p) { return load_loose<T, V>(p); });
    } else if (b.lines) {
      take(h, [](const T* p) { return load_once<T, V>(p); });
    } else {
      take(h, [](const T* p) { return load<T, V>(p); });
    }
  };
  take_heads(h0);  // in flight while the sines are computed
  float c[P], s[P];
  if (turned) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const sines at = sines_of(p, a.frequencies[pair + i]);
      c[i]           = at.c * a.magnitude;
      s[i]           = at.s * (a.transpose ? -a.magnitude : a.magnitude);
    }
  }
  const auto put = [](T* p, pack<T, V> const& v) {
    if constexpr (LOOSE) {
      store_loose<T, V>(p, v);
    } else {
      store<T, V>(p, v);
    }
  };
  for (int h = h0;;) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (h + i >= h1) { break; }
      T* row = dst + (h + i) * b.dst_head;
      if (turned) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
          T& u          = kAdjacent ? x[i].e[2 * j] : x[i].e[j];
          T& w          = kAdjacent ? x[i].e[2 * j + 1] : y[i].e[j];
          const float f = float(u), g = float(w);
          u = turned_first<T>(f, g, c[j], s[j]);
          w = turned_second<T>(f, g, c[j], s[j]);
        }
        if constexpr (!kAdjacent) { put(row + second, y[i]); }
      }
      put(row, x[i]);
    }
    h += kBatch;
    if (h >= h1) { break; }
    take_heads(h);
  }
}

template <typename T, int V, bool INTERLEAVED, bool LOOSE>
void launch(turn_args& a, hipStream_t stream)
{
  int64_t blocks = 0, threads = 0;
  for (int j = 0; j < a.jobs; ++j) {
    turn_job& b = a.job[j];
    // pairs of a thread: V of the half layout, V / 2 interleaved ones (V = 1: one pair)
    const auto vectors = [](int n) { return (n + V - 1) / V; };
    b.turned           = vectors(INTERLEAVED && V > 1 ? b.rotary : b.rotary / 2);
    b.items            = b.turned + vectors(b.dim - b.rotary);
    threads += a.tokens * b.heads * b.items;
    // what one load of a row reads begins and ends on lines: read past the caches. (Half a line would be
    // fetched twice: heads of 64 with 32 turned 125 -> 177 us; whole lines: 131,072 x 8 x 128 keys 100 -> 83 us.)
    const auto whole = [](int64_t elements) { return elements * int64_t(sizeof(T)) % 128 == 0; };
    b.lines = whole(INTERLEAVED ? b.dim : b.rotary / 2) && whole(b.dim) && whole(b.src_token) && whole(b.src_head) &&
              whole(b.src_outer) && reinterpret_cast<uintptr_t>(b.src) % 128 == 0;
  }
  // one thread computes its sines and cosines once for up to 8 heads, unless that would leave
  // fewer threads than the chip holds
  a.heads_per_thread = int32_t(std::clamp<int64_t>(threads / (256 * 2048), 1, 8));
  for (int j = 0; j < a.jobs; ++j) {
    turn_job& b = a.job[j];
    b.groups    = (b.heads + a.heads_per_thread - 1) / a.heads_per_thread;
    b.blocks    = (a.tokens * b.groups * b.items + kThreads - 1) / kThreads;
    blocks += b.blocks;
  }
  if (blocks >= (int64_t(1) << 24)) { throw std::invalid_argument("certex: too many elements to rotate in one call"); }
  if (blocks > 0) { turn_kernel<T, V, INTERLEAVED, LOOSE><<<dim3(uint32_t(blocks)), kThreads, 0, stream>>>(a); }
}

template <typename T, int V, bool LOOSE = false>
void launch(turn_args& a, hipStream_t stream)
{
  a.interleaved ? launch<T, V, true, LOOSE>(a, stream) : launch<T, V, false, LOOSE>(a, stream);
}

/** Whether rows of vectors of v elements can end in one that is moved back: the vector fits what is turned and what is
 *  copied, and no element is read after it may have been written. */
bool can_move_back(turn_args const& a, int v, int size)
{
  for (int j = 0; j < a.jobs; ++j) {
    turn_job const& b = a.job[j];
    const int turned = a.interleaved ? b.rotary : b.rotary / 2, copied = b.dim - b.rotary;
    if ((turned > 0 && turned < v) || (copied > 0 && copied < v)) { return false; }
    const int64_t outer = a.inner > 0 ? a.tokens / a.inner : 1;
    const auto last     = [&](int64_t o, int64_t so, int64_t t, int64_t st, int64_t sh) {
      return ((o - 1) * so + (t - 1) * st + (b.heads - 1) * sh + b.dim) * size;
    };
    const auto src = reinterpret_cast<uintptr_t>(b.src), dst = reinterpret_cast<uintptr_t>(b.dst);
    const auto src_end = src + last(outer, b.src_outer, a.inner, b.src_token, b.src_head);
    const auto dst_end = dst + (b.paged ? last(a.pages.n_pages, b.dst_outer, a.pages.page, b.dst_token, b.dst_head)
                                        : last(outer, b.dst_outer, a.inner, b.dst_token, b.dst_head));
    if (src < dst_end && dst < src_end) { return false; }
  }
  return true;
}

}  // namespace

void turn(elem type, turn_args a, hipStream_t stream)
{
  // the widest vectors that every row, stride and base address is a multiple of; 16 bytes at any alignment where
  // those are narrower
  const int size = elem_bytes(type);
  int64_t g      = 16 / size;
  for (int j = 0; j < a.jobs; ++j) {
    turn_job const& b = a.job[j];
    for (int64_t x : {b.src_outer, b.src_token, b.src_head, b.dst_outer, b.dst_token, b.dst_head, int64_t(b.dim),
                      a.interleaved ? int64_t(b.rotary) : int64_t(b.rotary / 2),
                      int64_t(reinterpret_cast<uintptr_t>(b.src) / size),
                      int64_t(reinterpret_cast<uintptr_t>(b.dst) / size)}) {
      g = std::gcd(g, x);
    }
  }
  const int full      = 16 / size;
  // Measured, narrow vectors and moved ones, us: halves of 33 of 130 (bfloat16) 96 and 84, of 51 of 128 163 and 140, of 20
  // of 80 113 and 98; interleaved, whose narrow vectors of a row follow one another, 102 of 128 109 and 120, 66 of 130 equal.
  const bool loose    = g < (a.interleaved ? 2 : full) && can_move_back(a, full, size);
  const auto by_width = [&](auto tag) {
    using T = decltype(tag);
    if (loose) {
      launch<T, 16 / sizeof(T), true>(a, stream);
    } else if (g == 8) {
      if constexpr (sizeof(T) == 2) { launch<T, 8>(a, stream); }
    } else if (g == 4) {
      launch<T, 4>(a, stream);
    } else if (g == 2) {
      launch<T, 2>(a, stream);
    } else {
      launch<T, 1>(a, stream);
    }
  };
  switch (type) {
    case elem::f32: by_width(float{}); break;
    case elem::f16: by_width(f16_t{}); break;
    case elem::bf16: by_width(bf16_t{}); break;
  }
}

}  // namespace certex_amd::attention
