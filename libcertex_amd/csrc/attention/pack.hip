// Keys and values of new tokens into 4-bit pages, the keys turned on the way, and back from them.
//
// Of every 64 elements x of a head: offset o = float16(min x), scale s = float16((max x - o) * (1 / 15 as float32)), and codes
// c = round((x - o) / s) in 0..15, so that o + s c is x within s / 2 (and what o and s are rounded by). Which of two codes is
// nearer is decided in 64 bits: the distance x - o and what it is rounded by together are exact, and so is the rounded distance's
// remainder x - o - s c, which only at half a step the rounding tells apart.
//
// 16 lanes take a group, 4 elements each, and a wave the groups
// of 4 heads, so that the group's minimum and maximum are 4 exchanges away. The 64-bit distance is taken only where an element of the
// wave is so close to the middle of two codes that float32 might err.
//
// What bounds it: every element is read once, and its half byte written; memory alone would take 8 us for the prompts below. In the
// kernels as they are instructions: a wave, a token's group of 8 heads, has 430 vector and 400 scalar ones where it packs, 170 and 290
// where it reads, of which finding its token, group and page by 64-bit divisions is most of the scalar ones; the vector units are busy
// 64 and 33 percent of the time. A record's bytes are moved by 8 waves in pieces of 1 to 4 bytes.
//
// Measured: 15,443 tokens of 8 heads of 64 float16 (32 MB of elements, 9 of records), appended 43 us, 56 with the rotation, whose
// sines every wave takes for its pairs, and read back 30; a token each of 64 sequences, 8 heads of 128 bfloat16, 5.0 (a call with the
// rotation 6.4) and 3.7 us, launch and dependent loads.
#include "../kernels/lanes.hpp"
#include "attention.hpp"
#include "elements.hpp"
#include "turn.hpp"

#include <algorithm>
#include <stdexcept>

namespace certex_amd::attention {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads   = 4;         // of a wave at a time
constexpr float kMost  = 65504.0f;  // float16's largest

/** What a wave works on: a token, one group of 64 elements of its keys or values, and heads. */
struct job {
  int64_t token, position;
  uint8_t* record;  // of head 0, NULL: the token is not in the pages
  int64_t head_bytes;
  int slot;         // in the record
  int dim, chunks, group;
  bool value;
  int h0, h1;
};

/** False where there is no such wave. */
__device__ __forceinline__ bool find_job(pack_args const& a, job* out)
{
  const int k_groups = (packed_chunks(a.pages.dim) + 1) / 2, groups = k_groups + (packed_chunks(a.pages.vdim) + 1) / 2;
  const int spans    = (a.pages.kv_heads + a.heads_per_wave - 1) / a.heads_per_wave;
  const int64_t wave = int64_t(blockIdx.x) * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int64_t row  = wave / groups;
  const int group    = int(wave - row * groups);
  const int64_t token = row / spans;
  if (token >= a.tokens) { return false; }
  const int span = int(row - token * spans);
  job j;
  j.token    = token;
  j.position = a.positions[token];
  j.value    = group >= k_groups;
  j.group    = j.value ? group - k_groups : group;
  j.dim      = j.value ? a.pages.vdim : a.pages.dim;
  j.chunks   = packed_chunks(j.dim);
  j.h0       = span * a.heads_per_wave;
  j.h1       = min(j.h0 + a.heads_per_wave, a.pages.kv_heads);
  j.record   = nullptr;
  page_map const& m = a.pages.map;
  const int64_t s   = a.sequences.p != nullptr ? a.sequences[token] : token, p = j.position;
  if (s >= 0 && s < m.sequences && p >= 0 && p < int64_t(m.width) * m.page) {
    const uint32_t entry = uint32_t(p) / uint32_t(m.page), in_page = uint32_t(p) - entry * uint32_t(m.page);
    const int32_t page   = m.table[s * m.width + entry];
    if (uint32_t(page) < uint32_t(m.n_pages)) {
      const int64_t record = a.pages.record();
      j.head_bytes         = record * (m.page / 8);
      j.record             = a.pages.p + int64_t(page) * a.pages.kv_heads * j.head_bytes + record * (in_page / 8) +
                 (j.value ? packed_pages::half_bytes(a.pages.dim) : 0);
      j.slot = int(in_page % 8);
    }
  }
  *out = j;
  return true;
}

/** Where codes are in a record's half: the word of the 8 dimensions from d on of a key; the byte of the dimensions d and
 *  d + 1 of a value (of 64 dimensions or of the last 32: 4 dimensions to 16 bytes). */
__device__ __forceinline__ int key_word(int chunks, int d, int slot)
{
  return slot * 16 * chunks + (d % 32 / 8 * chunks + d / 32) * 4;
}
__device__ __forceinline__ int value_byte(int d, int slot) { return d / 64 * 256 + d % 64 / 4 * 16 + d / 2 % 2 * 8 + slot; }

/** Nibble of the i-th of 8 dimensions in its word. */
__device__ __forceinline__ int nibble_of(int i) { return i / 2 + 4 * (i % 2); }

template <typename T>
__global__ __launch_bounds__(kThreads) void pack_kernel(pack_args a)
{
  job j;
  if (!find_job(a, &j) || j.record == nullptr) { return; }
  const int lane = threadIdx.x % 64, part = lane % 16, d = j.group * 64 + part * 4;
  pack_side const& side = j.value ? a.v : a.k;
  const T* src = static_cast<const T*>(side.src) + j.token * side.token;
  // these elements' pairs, if keys are turned: whether each is its pair's first, and where the other is
  const bool turns = !j.value && a.frequencies != nullptr && j.group * 64 < a.rotary;
  sines at[4];
  if (turns) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (d + i >= a.rotary) { continue; }
      const int half = a.rotary / 2;
      at[i] = sines_of(j.position, a.frequencies[a.interleaved ? (d + i) / 2 : (d + i) % half]);
      at[i].c *= a.magnitude;
      at[i].s *= a.magnitude;
    }
  }
  const int params = 128 * j.chunks + j.group * 32 + j.slot * 2;
  const auto take  = [&](int head, float* x) {
    const T* from = src + head * side.head + d;
    pack<T, 4> e{};
    if (d + 4 <= j.dim) {
      e = load_loose<T, 4>(from);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) { e.e[i] = d + i < j.dim ? from[i] : T(0.0f); }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = float(e.e[i]); }
  };
  const int h0 = j.h0 + lane / 16;
  float x[4];
  if (h0 < j.h1) { take(h0, x); }
  for (int h = h0;; h += kHeads) {
    float next[4] = {};
    if (h + kHeads < j.h1) { take(h + kHeads, next); }  // in flight during this head's
    if (h < j.h1) {
      if (turns) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = x[i];
          if (d + i >= a.rotary) { continue; }
          const int half   = a.rotary / 2;
          const bool first = a.interleaved ? i % 2 == 0 : d + i < half;
          const float other =
            a.interleaved ? x[i ^ 1] : float(src[h * side.head + (first ? d + i + half : d + i - half)]);
          y[i] = first ? float(turned_first<T>(x[i], other, at[i].c, at[i].s))
                       : float(turned_second<T>(other, x[i], at[i].c, at[i].s));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = y[i]; }
      }
      float low = INFINITY, high = -INFINITY;
      bool nan  = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (d + i >= j.dim) { continue; }
        low  = fminf(low, x[i]);
        high = fmaxf(high, x[i]);
        nan |= x[i] != x[i];
      }
      low  = lanes::min<16>(low);
      high = lanes::max<16>(high);
      nan  = (__ballot(nan) >> (lane & 48) & 0xffffu) != 0;
      const f16_t offset = nan ? f16_t(__builtin_nanf("")) : f16_t(fminf(fmaxf(low, -kMost), kMost));
      const f16_t scale  = nan ? offset : f16_t(fminf(fmaxf((high - float(offset)) * (1.0f / 15.0f), 0.0f), kMost));
      const float o = float(offset), s = float(scale), per = __builtin_amdgcn_rcpf(s);
      int code[4];
      bool close = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // off by less than 2^-17: x - o is below 16.1 s where its code is not cut, and rounded three times
        const float t = (x[i] - o) * per, near = __builtin_rintf(t);
        close |= __builtin_fabsf(t - near) > 0.5f - 0x1p-15f;
        code[i] = int(fminf(fmaxf(near, 0.0f), 15.0f));
      }
      if (__any(close)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double distance = double(x[i]) - double(o), rest = __builtin_fma(-double(code[i]), double(s), distance);
          const double of_o = distance - double(x[i]), lost = (double(x[i]) - (distance - of_o)) - (double(o) + of_o);
          const double half = 0.5 * double(s);
          // half a step to either side goes to the even code
          const bool odd = (code[i] & 1) != 0;
          if (rest > half || (rest == half && (lost > 0.0 || (lost == 0.0 && odd)))) {
            code[i] = min(code[i] + 1, 15);
          } else if (rest < -half || (rest == -half && (lost < 0.0 || (lost == 0.0 && odd)))) {
            code[i] = max(code[i] - 1, 0);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!(s > 0.0f) || d + i >= j.dim) { code[i] = 0; }
      }
      uint8_t* record = j.record + h * j.head_bytes;
      if (j.value) {
        if (d < 32 * j.chunks) {
          record[value_byte(d, j.slot)]     = uint8_t(code[0] | code[1] << 4);
          record[value_byte(d + 2, j.slot)] = uint8_t(code[2] | code[3] << 4);
        }
      } else {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) { word |= uint32_t(code[i]) << (4 * (part % 2 == 0 ? nibble_of(i) : nibble_of(i + 4))); }
        word |= uint32_t(lanes::exchange<1>(int(word)));
        if (part % 2 == 0 && d < 32 * j.chunks) { *reinterpret_cast<uint32_t*>(record + key_word(j.chunks, d, j.slot)) = word; }
      }
      if (part == 0) {
        *reinterpret_cast<f16_t*>(record + params)      = scale;
        *reinterpret_cast<f16_t*>(record + params + 16) = offset;
      }
    }
    if (j.h0 + (h - h0) + kHeads >= j.h1) { return; }
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = next[i]; }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack_kernel(pack_args a)
{
  job j;
  if (!find_job(a, &j)) { return; }
  const int lane = threadIdx.x % 64, d = j.group * 64 + lane % 16 * 4;
  if (d >= j.dim) { return; }
  pack_side const& side = j.value ? a.v : a.k;
  T* dst                = static_cast<T*>(side.dst) + j.token * side.token + d;
  const int params      = 128 * j.chunks + j.group * 32 + j.slot * 2;
#pragma unroll 2
  for (int h = j.h0 + lane / 16; h < j.h1; h += kHeads) {
    float x[4] = {};
    if (j.record != nullptr) {
      const uint8_t* record = j.record + h * j.head_bytes;
      uint32_t code[4];
      if (j.value) {
        const uint32_t first = record[value_byte(d, j.slot)], second = record[value_byte(d + 2, j.slot)];
        code[0] = first & 15u, code[1] = first >> 4, code[2] = second & 15u, code[3] = second >> 4;
      } else {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(record + key_word(j.chunks, d & ~7, j.slot));
#pragma unroll
        for (int i = 0; i < 4; ++i) { code[i] = word >> (4 * (d % 8 == 0 ? nibble_of(i) : nibble_of(i + 4))) & 15u; }
      }
      const float scale  = float(*reinterpret_cast<const f16_t*>(record + params));
      const float offset = float(*reinterpret_cast<const f16_t*>(record + params + 16));
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[i] = __builtin_fmaf(float(code[i]), scale, offset); }
    }
    pack<T, 4> e;
#pragma unroll
    for (int i = 0; i < 4; ++i) { e.e[i] = narrowed<T>(x[i]); }
    T* to = dst + h * side.head;
    if (d + 4 <= j.dim) {
      store_loose<T, 4>(to, e);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (d + i < j.dim) { to[i] = e.e[i]; }
      }
    }
  }
}

/** Waves, and the heads that each goes over: all, unless that would leave fewer waves than the chip holds; a multiple of
 *  those it takes at a time. */
uint32_t blocks_for(pack_args& a)
{
  const int groups    = (packed_chunks(a.pages.dim) + 1) / 2 + (packed_chunks(a.pages.vdim) + 1) / 2;
  const int64_t rows  = a.tokens * groups;
  const int64_t most  = (a.pages.kv_heads + kHeads - 1) / kHeads;
  a.heads_per_wave    = int32_t(kHeads * std::clamp<int64_t>(rows * most / (256 * 32), 1, most));
  const int64_t spans = (a.pages.kv_heads + a.heads_per_wave - 1) / a.heads_per_wave;
  const int64_t blocks = (rows * spans + kThreads / 64 - 1) / (kThreads / 64);
  if (blocks >= (int64_t(1) << 24)) { throw std::invalid_argument("certex: too many tokens in one call"); }
  return uint32_t(blocks);
}

}  // namespace

void pack_pages(elem type, pack_args a, hipStream_t stream)
{
  const uint32_t blocks = blocks_for(a);
  switch (type) {
    case elem::f32: pack_kernel<float><<<dim3(blocks), kThreads, 0, stream>>>(a); break;
    case elem::f16: pack_kernel<f16_t><<<dim3(blocks), kThreads, 0, stream>>>(a); break;
    case elem::bf16: pack_kernel<bf16_t><<<dim3(blocks), kThreads, 0, stream>>>(a); break;
  }
}

void unpack_pages(elem type, pack_args a, hipStream_t stream)
{
  const uint32_t blocks = blocks_for(a);
  switch (type) {
    case elem::f32: unpack_kernel<float><<<dim3(blocks), kThreads, 0, stream>>>(a); break;
    case elem::f16: unpack_kernel<f16_t><<<dim3(blocks), kThreads, 0, stream>>>(a); break;
    case elem::bf16: unpack_kernel<bf16_t><<<dim3(blocks), kThreads, 0, stream>>>(a); break;
  }
}

}  // namespace certex_amd::attention
