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
// so that sines are computed once for up to 8 heads. Measured: 131,072 tokens x 8 heads of 128 bfloat16, 0.54 GB: 84 us
// a pass, 6.4 TB/s (a copy of 2 GiB: 4.9); prompts of 15,443 tokens appended with their queries, 190 MB: 35 us,
// 5.4 TB/s; 64 queries of a step 4.6 us, their append 5.3 us: launch and three dependent loads.
#include "attention.hpp"
#include "elements.hpp"

#include <algorithm>
#include <numeric>
#include <stdexcept>

namespace certex_amd::attention {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch   = 4;

/**
 * One thread: one vector of V elements of a row (of both halves in the half layout), over
 * heads_per_thread heads of one token. Blocks are dealt to the jobs in order.
 */
template <typename T, int V, bool INTERLEAVED>
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
  const int first  = !turned ? b.rotary + int(item - uint32_t(b.turned)) * V : int(item) * (INTERLEAVED && V == 1 ? 2 : V);
  const int second = INTERLEAVED ? 1 : b.rotary / 2;  // from the first
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
    if (b.lines) {
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
      const uint32_t turns = uint32_t((uint64_t(p) * a.frequencies[int(item) * P + i]) >> 32);
      float sine, cosine;
      sincospif(float(int32_t(turns & ~255u)) * 0x1p-31f, &sine, &cosine);
      const float rest = float(turns & 255u) * float(M_PI * 0x1p-31);
      s[i]             = __builtin_fmaf(cosine, rest, sine);
      c[i]             = __builtin_fmaf(sine, -rest, cosine);
      c[i] *= a.magnitude;
      s[i] *= a.transpose ? -a.magnitude : a.magnitude;
    }
  }
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
          u = T(__builtin_fmaf(f, c[j], -(g * s[j])));
          w = T(__builtin_fmaf(f, s[j], g * c[j]));
        }
        if constexpr (!kAdjacent) { store<T, V>(row + second, y[i]); }
      }
      store<T, V>(row, x[i]);
    }
    h += kBatch;
    if (h >= h1) { break; }
    take_heads(h);
  }
}

template <typename T, int V, bool INTERLEAVED>
void launch(turn_args& a, hipStream_t stream)
{
  int64_t blocks = 0, threads = 0;
  for (int j = 0; j < a.jobs; ++j) {
    turn_job& b = a.job[j];
    // pairs of a thread: V of the half layout, V / 2 interleaved ones (V = 1: one pair)
    b.turned = INTERLEAVED && V > 1 ? b.rotary / V : b.rotary / 2 / V;
    b.items  = b.turned + (b.dim - b.rotary) / V;
    threads += a.tokens * b.heads * b.items;
    // what one load of a row reads begins and ends on lines: read past the caches. (Half a line would be fetched
    // twice: heads of 64 with 32 turned 125 -> 177 us; whole lines: 131,072 x 8 x 128 keys 100 -> 83 us.)
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
  if (blocks > 0) { turn_kernel<T, V, INTERLEAVED><<<dim3(uint32_t(blocks)), kThreads, 0, stream>>>(a); }
}

template <typename T, int V>
void launch(turn_args& a, hipStream_t stream)
{
  a.interleaved ? launch<T, V, true>(a, stream) : launch<T, V, false>(a, stream);
}

}  // namespace

void turn(elem type, turn_args a, hipStream_t stream)
{
  // the widest vectors that every row, stride and base address is a multiple of
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
  const auto by_width = [&](auto tag) {
    using T = decltype(tag);
    if (g == 8) {
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
