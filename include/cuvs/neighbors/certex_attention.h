/*
 * C API of the attention operators next to the key cache: rotation by position, appending keys and
 * values to a paged cache, attention of one new token over it, and attention over the top k that
 * a search of the cache returned.
 *
 * They have no counterpart in the reference, whose attention support ends at the ids and scores of
 * the top k (certex/attention.py:84-106). As in certex.h every call returns CUVS_SUCCESS or CUVS_ERROR with
 * a message in cuvsGetLastErrorText(), tensors are borrowed DLPack v1.0 tensors in device memory of
 * the device of `res`, and the work is queued on the stream of `res` and not waited for. The calls
 * allocate nothing and read nothing back, so that a stream capture records them.
 *
 * "Rows": a tensor whose last dimension is dense and whose other dimensions have any strides.
 * "Dense": row major without gaps. What a call writes must share no memory with what it reads, nor within itself, unless
 * its description says so. Elements are float32, float16 or bfloat16, the same for all
 * row tensors of a call; "integers" are int32 or int64. Sums, maxima and the rotation are computed in
 * float32 or more.
 */
#pragma once

#include <cuvs/core/c_api.h>
#include <dlpack/dlpack.h>
#include <stdbool.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/** Pairs of a rotated head: (i, i + rotary_dim / 2), or (2 i, 2 i + 1). */
enum cuvsCertexRotaryLayout { CERTEX_ROTARY_HALF = 0, CERTEX_ROTARY_INTERLEAVED = 1 };

/**
 * How the frequencies f_i = base^(-2 i / rotary_dim), i < rotary_dim / 2, are scaled for contexts
 * `factor` times as long as the original one:
 *   NONE    f_i
 *   LINEAR  f_i / factor
 *   BASE    those of the base  base * factor^(rotary_dim / (rotary_dim - 2))
 *   RAMP    f_i (g + (1 - g) / factor) with g = clamp((t - ramp_low) / (ramp_high - ramp_low), 0, 1)
 *           and t = original_length f_i / (2 pi), the turns within the original context: fast pairs
 *           keep their frequency, slow ones are interpolated
 */
enum cuvsCertexRotaryScaling {
  CERTEX_ROTARY_NONE   = 0,
  CERTEX_ROTARY_LINEAR = 1,
  CERTEX_ROTARY_BASE   = 2,
  CERTEX_ROTARY_RAMP   = 3
};

struct cuvsCertexRotaryParams {
  int32_t rotary_dim; /* even, at least 2: the leading elements of a head that are rotated */
  int32_t layout;
  double base;
  int32_t scaling;
  double factor;
  double original_length;
  double ramp_low;
  double ramp_high;
  double magnitude; /* of the rotated elements; 0: 1, or 0.1 ln(factor) + 1 with the ramp */
};
typedef struct cuvsCertexRotaryParams* cuvsCertexRotaryParams_t;

/** rotary_dim 128, half layout, base 10000, no scaling (factor 1, length 8192, ramp 1 to 32). */
CUVS_EXPORT cuvsError_t cuvsCertexRotaryParamsCreate(cuvsCertexRotaryParams_t* params);
CUVS_EXPORT cuvsError_t cuvsCertexRotaryParamsDestroy(cuvsCertexRotaryParams_t params);

/** A rotation: its frequencies in the memory of one device. A recorded graph reads them there: destroy it after the graph. */
typedef uintptr_t cuvsCertexRotary_t;
CUVS_EXPORT cuvsError_t cuvsCertexRotaryCreate(cuvsResources_t res,
                                               cuvsCertexRotaryParams_t params,
                                               cuvsCertexRotary_t* rotary);
CUVS_EXPORT cuvsError_t cuvsCertexRotaryDestroy(cuvsCertexRotary_t rotary);
/** The rotary_dim / 2 scaled frequencies (radians per position, to host memory) and the magnitude
 *  that these parameters stand for; needs no device. */
CUVS_EXPORT cuvsError_t cuvsCertexRotaryFrequencies(cuvsCertexRotaryParams_t params,
                                                    double* frequencies,
                                                    double* magnitude);

/**
 * y = x with the first rotary_dim elements of every head rotated: pair (a, b) of position p and
 * frequency f becomes magnitude * (a cos pf - b sin pf, a sin pf + b cos pf).
 * x and y: rows [tokens, heads, dim] or [batch, tokens, heads, dim]; y may be x itself (the same address and
 * strides), and else shares no memory with it. positions: dense integers [tokens] or [batch, tokens], of any sign and size. With `transpose` the matrix of
 * the rotation is transposed (the negative angle, the same magnitude): x is then the gradient
 * of y, and y the gradient of x.
 */
CUVS_EXPORT cuvsError_t cuvsCertexRotate(cuvsResources_t res,
                                         cuvsCertexRotary_t rotary,
                                         DLManagedTensor* x,
                                         DLManagedTensor* positions,
                                         DLManagedTensor* y,
                                         bool transpose);

/**
 * Writes token t's keys and values to position positions[t] of sequence sequences[t] of a paged
 * cache, the keys rotated on the way unless `rotary` is 0. Position p of sequence s is slot
 * p % page_size of page page_table[s, p / page_size].
 * k: rows [tokens, kv_heads, dim]; v: rows [tokens, kv_heads, vdim]; k_pages: rows [n_pages,
 * page_size, kv_heads, dim]; v_pages: the same with vdim; page_table: dense int32 [n_sequences, n]; positions:
 * dense integers [tokens]; sequences: the same, or NULL: token t belongs to sequence t. With q
 * (rows [tokens, heads, dim], or NULL) the same launch rotates the tokens' queries into q_out, which may be
 * q itself and else shares no memory with q, k, v or the pages. The slots that are written must not lie in k, v or q.
 * A token of a negative position or sequence (padding), or whose page the table does not hold
 * (an entry outside [0, n_pages)), is not written. The tokens of one call are to have positions of their own: a slot
 * that several name ends with elements of any of them mixed.
 */
CUVS_EXPORT cuvsError_t cuvsCertexAppendPages(cuvsResources_t res,
                                              cuvsCertexRotary_t rotary,
                                              DLManagedTensor* k,
                                              DLManagedTensor* v,
                                              DLManagedTensor* k_pages,
                                              DLManagedTensor* v_pages,
                                              DLManagedTensor* page_table,
                                              DLManagedTensor* positions,
                                              DLManagedTensor* sequences,
                                              DLManagedTensor* q,
                                              DLManagedTensor* q_out);

/**
 * Attention of one new token per sequence: out[s, h] = sum_t w_t v_t with w the softmax of
 * scale * <q[s, h], k_t> over the positions t of [max(0, length - window), length) (window 0: all),
 * key and value head h / (heads / kv_heads).
 * q: rows [n_sequences, heads, dim]; pages and page_table as for cuvsCertexAppendPages, dim and vdim at most
 * 256, page_size a multiple of 8; lengths: dense integers [n_sequences], cut to the table's pages;
 * out: dense [n_sequences, heads, vdim]; lse (or NULL): dense float32 [n_sequences, heads], the
 * logarithm of the softmax's denominator. Positions whose page the table does not hold do not count; a row
 * without positions gives zeros, and lse -inf. Slots at and past a sequence's length are not used,
 * whatever they hold. An infinite value that counts, however little it weighs, makes its column of out infinite or NaN.
 * workspace: a dense uint8 vector of at least the bytes that cuvsCertexPagedAttentionWorkspace reports
 * for the same tensors (NULL if 0), in use until the queued work is done.
 */
CUVS_EXPORT cuvsError_t cuvsCertexPagedAttention(cuvsResources_t res,
                                                 DLManagedTensor* q,
                                                 DLManagedTensor* k_pages,
                                                 DLManagedTensor* v_pages,
                                                 DLManagedTensor* page_table,
                                                 DLManagedTensor* lengths,
                                                 float scale,
                                                 int64_t window,
                                                 DLManagedTensor* workspace,
                                                 DLManagedTensor* out,
                                                 DLManagedTensor* lse);
CUVS_EXPORT cuvsError_t cuvsCertexPagedAttentionWorkspace(DLManagedTensor* q,
                                                          DLManagedTensor* k_pages,
                                                          DLManagedTensor* v_pages,
                                                          DLManagedTensor* page_table,
                                                          int64_t window,
                                                          int64_t* bytes);

/**
 * Attention over a selected top k: out[h, i] = sum_j w_j values[id_j] with w the softmax of
 * scale * scores[h, i, j] over j, value head h / (heads / kv_heads); scores and ids as
 * cuvsCertexSearchWithLabelsMapped returns them for a key cache.
 * scores: dense float32 [heads, queries, k]; ids: dense integers of that shape; values: rows
 * [kv_heads, n, vdim], or with page_table (dense int32 [n], one sequence) the pages
 * [n_pages, page_size, kv_heads, vdim]; vdim at most 256; out: dense [heads, queries, vdim]; lse (or NULL):
 * dense float32 [heads, queries]. An id outside the values (as -1) and a score of -inf do not count;
 * a row of none gives zeros, and lse -inf. Infinite values and workspace: as for cuvsCertexPagedAttention.
 */
CUVS_EXPORT cuvsError_t cuvsCertexSelectedAttention(cuvsResources_t res,
                                                    DLManagedTensor* scores,
                                                    DLManagedTensor* ids,
                                                    DLManagedTensor* values,
                                                    DLManagedTensor* page_table,
                                                    float scale,
                                                    DLManagedTensor* workspace,
                                                    DLManagedTensor* out,
                                                    DLManagedTensor* lse);
CUVS_EXPORT cuvsError_t cuvsCertexSelectedAttentionWorkspace(DLManagedTensor* scores,
                                                             DLManagedTensor* values,
                                                             DLManagedTensor* page_table,
                                                             int64_t* bytes);

#ifdef __cplusplus
}
#endif
