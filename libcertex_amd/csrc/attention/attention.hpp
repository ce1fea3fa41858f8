// Launchers of the gfx950 kernels of the attention operators: rotation by position, appending to
// a paged cache, attention of one new token over it, attention over a selected top k. Every
// launcher takes plain device pointers, sizes, strides in elements and the stream to queue on;
// none allocates or synchronises.
#pragma once

#include "scores.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace certex_amd::attention {

enum class elem : int { f32 = 0, f16 = 1, bf16 = 2 };
inline int elem_bytes(elem e) { return e == elem::f32 ? 4 : 2; }

/** A device vector of int32 or int64. */
struct int_vector {
  const void* p = nullptr;
  bool wide     = false;
#ifdef __HIPCC__
  __device__ __forceinline__ int64_t operator[](int64_t i) const
  {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
  }
#endif
};

/**
 * Pages by sequence: entry (s, j) is the page that holds positions [j page, (j + 1) page) of
 * sequence s. An entry outside [0, n_pages) is a page that the sequence does not have.
 */
struct page_map {
  const int32_t* table = nullptr;  // [sequences, width], rows `width` apart
  int64_t sequences    = 0;
  int32_t width        = 0;
  int32_t n_pages      = 0;
  int32_t page         = 0;  // positions per page
};

/** One tensor of a rotation: `heads` rows of `dim` elements per token, the first `rotary` rotated. */
struct turn_job {
  const void* src = nullptr;
  void* dst       = nullptr;
  int64_t src_outer = 0, src_token = 0, src_head = 0;
  int64_t dst_outer = 0, dst_token = 0, dst_head = 0;  // paged: of a page, of a slot, of a head
  int32_t heads = 0, dim = 0, rotary = 0;
  bool paged = false;
  // set by the launcher
  int32_t items = 0, turned = 0, groups = 0;  // vectors per row, those rotated, groups of heads
  bool lines = false;                         // one load of a row reads whole cache lines
  int64_t blocks = 0;
};

struct turn_args {
  const uint64_t* frequencies = nullptr;  // turns per position, times 2^64
  float magnitude             = 1.0f;
  bool interleaved            = false;
  bool transpose              = false;  // by the negative angle: the gradient of the rotation
  int_vector positions;
  int_vector sequences;  // of every token (paged jobs); none: token t belongs to sequence t
  int64_t tokens = 0;
  int64_t inner  = 1;  // token t is (t / inner, t % inner)
  page_map pages;
  turn_job job[3];
  int jobs = 0;
  int32_t heads_per_thread = 1;  // set by the launcher
};

void turn(elem type, turn_args args, hipStream_t stream);

struct attend_args {
  const void* q = nullptr;
  int64_t q_seq = 0, q_head = 0;
  const void* k = nullptr;
  int64_t k_page = 0, k_slot = 0, k_head = 0;
  const void* v = nullptr;
  int64_t v_page = 0, v_slot = 0, v_head = 0;
  page_map pages;
  int_vector lengths;
  int32_t heads = 0, kv_heads = 0, dim = 0, vdim = 0;
  float scale    = 0;
  score_shape shape;
  int64_t window = 0;  // the last `window` positions only; 0: all
  void* out      = nullptr;  // [sequences, heads, vdim] dense
  float* lse     = nullptr;  // [sequences, heads] dense, or NULL
  void* workspace = nullptr;
};

struct prompt_args {
  const void* q = nullptr;  // [tokens, heads, dim]
  int64_t q_token = 0, q_head = 0;
  const void* k = nullptr;
  int64_t k_page = 0, k_slot = 0, k_head = 0;
  const void* v = nullptr;
  int64_t v_page = 0, v_slot = 0, v_head = 0;
  page_map pages;
  int_vector lengths;
  int_vector first;   // [sequences + 1]: sequence s has the tokens [first[s], first[s + 1]), its last ones
  int_vector prefix;  // [sequences], or none: positions that every token sees
  int64_t tokens = 0;
  int32_t heads = 0, kv_heads = 0, dim = 0, vdim = 0;
  float scale = 0;
  score_shape shape;
  int64_t window = 0;
  void* out      = nullptr;  // [tokens, heads, vdim] dense
  float* lse     = nullptr;  // [tokens, heads] dense, or NULL
  void* workspace = nullptr;
};

// a source for each element type
size_t prompt_workspace_f32(prompt_args const& args);
size_t prompt_workspace_f16(prompt_args const& args);
size_t prompt_workspace_bf16(prompt_args const& args);
void prompt_f32(prompt_args const& args, hipStream_t stream);
void prompt_f16(prompt_args const& args, hipStream_t stream);
void prompt_bf16(prompt_args const& args, hipStream_t stream);

inline size_t prompt_workspace(elem type, prompt_args const& args)
{
  return type == elem::f32 ? prompt_workspace_f32(args) : type == elem::f16 ? prompt_workspace_f16(args) : prompt_workspace_bf16(args);
}
inline void prompt(elem type, prompt_args const& args, hipStream_t stream)
{
  type == elem::f32 ? prompt_f32(args, stream) : type == elem::f16 ? prompt_f16(args, stream) : prompt_bf16(args, stream);
}

/** Dimensions that a packed row of dim elements takes: its chunks of 32. */
#ifdef __HIPCC__
__host__ __device__
#endif
constexpr int packed_chunks(int dim) { return dim <= 64 ? 2 : dim <= 96 ? 3 : dim <= 128 ? 4 : dim <= 192 ? 6 : 8; }

/** Words that every piece of a packed key begins at a multiple of, which is a word of each chunk: keys of `chunks` chunks, or (not
 *  `full`) of any number up to that. */
constexpr int packed_key_align(int chunks, bool full) { return !full ? 1 : chunks % 4 == 0 ? 4 : chunks % 2 == 0 ? 2 : 1; }

/**
 * 4-bit pages, [n_pages][kv_heads][page / 8] records of 8 positions of a head. Every group of 64 elements of a key or value
 * has a scale s and an offset o (float16); an element is o + s code. A record holds, for C chunks of 32 dimensions and
 * G = (C + 1) / 2 groups, of the key and then of the value:
 * - the codes, 128 C bytes. Keys: 16 C bytes a position, word (g C + c) the dimensions [32 c + 8 g, + 8), of which the i-th
 *   is nibble i / 2 + 4 (i % 2). Values: 64 dimensions are 16 x 2 x 8 bytes, (l, j, position) the dimensions 4 l + 2 j in the
 *   low nibble and 4 l + 2 j + 1 in the high one; 32 dimensions at the end are 16 x 8 bytes, (l, position) 2 l and 2 l + 1;
 * - 32 G bytes: of each group the scales of the 8 positions, then their offsets.
 */
struct packed_pages {
  uint8_t* p       = nullptr;
  int32_t kv_heads = 0, dim = 0, vdim = 0;
  page_map map;
#ifdef __HIPCC__
  __host__ __device__
#endif
  static constexpr int
  half_bytes(int dim)
  {
    return 128 * packed_chunks(dim) + 32 * ((packed_chunks(dim) + 1) / 2);
  }
#ifdef __HIPCC__
  __host__ __device__
#endif
  [[nodiscard]] int record() const
  {
    return half_bytes(dim) + half_bytes(vdim);
  }
};

/** One side (keys or values) of tokens that are packed into pages, or read from them. */
struct pack_side {
  const void* src = nullptr;  // packed from
  void* dst       = nullptr;  // read into
  int64_t token = 0, head = 0;
};

struct pack_args {
  packed_pages pages;
  pack_side k, v;
  const uint64_t* frequencies = nullptr;  // as turn_args; none: keys as they are
  float magnitude             = 1.0f;
  bool interleaved            = false;
  int32_t rotary              = 0;
  int_vector positions;
  int_vector sequences;  // none: token t belongs to sequence t
  int64_t tokens = 0;
  int32_t heads_per_wave = 0;  // set by the launcher
};

void pack_pages(elem type, pack_args args, hipStream_t stream);
void unpack_pages(elem type, pack_args args, hipStream_t stream);

/** attend_args whose keys and values are packed: k, v and their strides are not used. */
struct packed_args {
  attend_args a;
  packed_pages pages;
};

size_t packed_workspace(elem type, packed_args const& args);
void packed_attend(elem type, packed_args const& args, hipStream_t stream);

/** Largest head dimension of keys and of values. */
constexpr int kMaxHeadDim = 256;
/** Positions per page are a multiple of this. */
constexpr int kPageUnit = 8;

size_t attend_workspace(elem type, attend_args const& args);
void attend(elem type, attend_args const& args, hipStream_t stream);

struct select_args {
  const float* scores = nullptr;  // [heads, queries, k] dense
  int_vector ids;                 // the same shape
  const void* v = nullptr;
  int64_t v_page = 0, v_slot = 0, v_head = 0;  // without pages: v_slot of a row
  page_map pages;                               // one sequence; table NULL: rows by id
  int64_t n = 0;                                // rows, or positions of the pages
  int32_t heads = 0, kv_heads = 0, vdim = 0;
  int64_t queries = 0, k = 0;
  float scale = 0;
  void* out   = nullptr;  // [heads, queries, vdim] dense
  float* lse  = nullptr;  // [heads, queries] dense, or NULL
  void* workspace = nullptr;
};

size_t select_workspace(elem type, select_args const& args);
void select(elem type, select_args const& args, hipStream_t stream);

}  // namespace certex_amd::attention
