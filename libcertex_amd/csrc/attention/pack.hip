// Keys and values of new tokens into 4-bit pages, the keys turned on the way, and back from them.
//
// Of every 64 elements x of a head: offset o = float16(min x), scale s = float16((max x - o) * (1 / 15 as float32)), and codes
// c = round((x - o) / s) in 0..15, so that o + s c is x within s / 2 (and what o and s are rounded by). Which of two codes is
// nearer is decided in 64 bits: the distance x - o is exact there, and so is its remainder x - o - s c.
//
// What bounds it: every element is read once, and its half byte written. A wave takes a group, a lane an element, and goes
// over heads, so that sines are computed once for all of them.
#include "../kernels/lanes.hpp"
#include "attention.hpp"
#include "elements.hpp"
#include "turn.hpp"

#include <algorithm>
#include <stdexcept>

namespace certex_amd::attention {
namespace {

constexpr int kThreads = 256;
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

/** Where the code of a dimension is in a record's half: its byte, and of a value the dimensions d and d + 1 share it. */
__device__ __forceinline__ int value_byte(int chunks, int d, int slot)
{
  const int unit = d / 64, e = d % 64;
  return unit * 256 + (2 * unit + 1 < chunks ? e / 4 * 16 + e / 2 % 2 * 8 : e / 2 * 8) + slot;
}
__device__ __forceinline__ int key_word(int chunks, int d, int slot)
{
  return slot * 16 * chunks + (d % 32 / 8 * chunks + d / 32) * 4;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pack_kernel(pack_args a)
{
  job j;
  if (!find_job(a, &j) || j.record == nullptr) { return; }
  const int lane = threadIdx.x % 64, d = j.group * 64 + lane;
  pack_side const& side = j.value ? a.v : a.k;
  const T* src  = static_cast<const T*>(side.src) + j.token * side.token;
  const bool in = d < j.dim;
  // this element's pair, if keys are turned
  const bool turned = !j.value && a.frequencies != nullptr && d < a.rotary;
  int partner = d;
  bool first  = true;
  sines at{1.0f, 0.0f};
  if (turned) {
    const int half = a.rotary / 2, pair = a.interleaved ? d / 2 : d % half;
    first   = a.interleaved ? d % 2 == 0 : d < half;
    partner = a.interleaved ? d ^ 1 : first ? d + half : d - half;
    at      = sines_of(j.position, a.frequencies[pair]);
    at.c *= a.magnitude;
    at.s *= a.magnitude;
  }
  const int params = 128 * j.chunks + j.group * 32 + j.slot * 2;
  for (int h = j.h0; h < j.h1; ++h) {
    float x = in ? float(src[h * side.head + d]) : 0.0f;
    if (turned) {
      const float other = float(src[h * side.head + partner]);
      x = first ? float(turned_first<T>(x, other, at.c, at.s)) : float(turned_second<T>(other, x, at.c, at.s));
    }
    const float low = lanes::min<64>(in ? x : INFINITY), high = lanes::max<64>(in ? x : -INFINITY);
    const bool nan  = __any(x != x);
    const f16_t offset = nan ? f16_t(__builtin_nanf("")) : f16_t(fminf(fmaxf(low, -kMost), kMost));
    const f16_t scale  = nan ? offset : f16_t(fminf(fmaxf((high - float(offset)) * (1.0f / 15.0f), 0.0f), kMost));
    uint32_t code = 0;
    if (float(scale) > 0.0f) {
      const double s = double(float(scale)), distance = double(x) - double(float(offset));
      const float near = fminf(fmaxf(__builtin_rintf(float(distance) * __builtin_amdgcn_rcpf(float(scale))), 0.0f), 15.0f);
      const double rest = __builtin_fma(-double(near), s, distance);
      int c = int(near);
      // half a step to either side goes to the even code
      if (rest > 0.5 * s || (rest == 0.5 * s && (c & 1) != 0)) {
        ++c;
      } else if (rest < -0.5 * s || (rest == -0.5 * s && (c & 1) != 0)) {
        --c;
      }
      code = in ? uint32_t(min(max(c, 0), 15)) : 0u;
    }
    uint8_t* record = j.record + h * j.head_bytes;
    if (j.value) {
      const uint32_t both = code | uint32_t(lanes::exchange<1>(int(code))) << 4;
      if (d % 2 == 0 && d < 32 * j.chunks) { record[value_byte(j.chunks, d, j.slot)] = uint8_t(both); }
    } else {
      const int i = d % 8;
      const uint32_t word = uint32_t(lanes::butterfly<8>(int(code << (4 * (i / 2 + 4 * (i % 2)))), [](int u, int w) { return u | w; }));
      if (i == 0 && d < 32 * j.chunks) { *reinterpret_cast<uint32_t*>(record + key_word(j.chunks, d, j.slot)) = word; }
    }
    if (lane == 0) {
      *reinterpret_cast<f16_t*>(record + params)      = scale;
      *reinterpret_cast<f16_t*>(record + params + 16) = offset;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack_kernel(pack_args a)
{
  job j;
  if (!find_job(a, &j)) { return; }
  const int lane = threadIdx.x % 64, d = j.group * 64 + lane;
  if (d >= j.dim) { return; }
  pack_side const& side = j.value ? a.v : a.k;
  T* dst                = static_cast<T*>(side.dst) + j.token * side.token;
  const int params      = 128 * j.chunks + j.group * 32 + j.slot * 2;
  for (int h = j.h0; h < j.h1; ++h) {
    float x = 0.0f;
    if (j.record != nullptr) {
      const uint8_t* record = j.record + h * j.head_bytes;
      const int i           = d % 8;
      const uint32_t code =
        j.value ? uint32_t(record[value_byte(j.chunks, d & ~1, j.slot)]) >> (d % 2 * 4) & 15u
                : *reinterpret_cast<const uint32_t*>(record + key_word(j.chunks, d, j.slot)) >> (4 * (i / 2 + 4 * (i % 2))) & 15u;
      x = __builtin_fmaf(float(code), float(*reinterpret_cast<const f16_t*>(record + params)),
                         float(*reinterpret_cast<const f16_t*>(record + params + 16)));
    }
    dst[h * side.head + d] = narrowed<T>(x);
  }
}

/** Waves, and the heads that each goes over: all, unless that would leave fewer waves than the chip holds. */
uint32_t blocks_for(pack_args& a)
{
  const int groups    = (packed_chunks(a.pages.dim) + 1) / 2 + (packed_chunks(a.pages.vdim) + 1) / 2;
  const int64_t rows  = a.tokens * groups;
  a.heads_per_wave    = int32_t(std::clamp<int64_t>(rows * a.pages.kv_heads / (256 * 32), 1, a.pages.kv_heads));
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
