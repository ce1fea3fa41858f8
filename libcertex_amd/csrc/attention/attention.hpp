// Launchers of the gfx950 kernels of the attention operators: rotation by position, appending to
// a paged cache, attention of one new token over it, attention over a selected top k. Every
// launcher takes plain device pointers, sizes, strides in elements and the stream to queue on;
// none allocates or synchronises.
#pragma once

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
  int64_t window = 0;  // the last `window` positions only; 0: all
  void* out      = nullptr;  // [sequences, heads, vdim] dense
  float* lse     = nullptr;  // [sequences, heads] dense, or NULL
  void* workspace = nullptr;
};

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
