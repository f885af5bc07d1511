/*
 * adaptq_paged.h -- the quantised cache in pages, for batches whose sequences have
 * different lengths, and rotary positions.
 *
 * The rows are those of the ring caches of adaptq.h (norm, signs, Walsh-Hadamard
 * transform, Lloyd-Max codes, most significant bits first), so a page holds upstream's
 * row bytes; what upstream has no counterpart for is where they lie: `page_size` tokens
 * of every KV head form a page, a sequence is a row of a block table (page numbers) and a
 * length.  Block tables, lengths and positions stay on the device: no call copies to the
 * host, waits or allocates, so all of them can be captured into a CUDA graph.
 *
 * All pointers are DEVICE memory of the device `adaptq_paged_t.device` unless stated.
 * Element types: 0 = float32, 1 = float16, 2 = bfloat16.  Strides count elements; the
 * last dimension of every tensor is contiguous, pointers are aligned to their elements.
 * `stream` is a cudaStream_t (NULL = the default stream).  Functions return 0, or -1 and set adaptq_last_error().
 *
 * Values that only the device knows are checked there: an entry that would leave the
 * pool or the table is skipped and leaves a bit in *status -- 1: a page number outside the
 * pool, 2: a position or length that the block table has no room for, 256: an index check of the
 * checked build failed.  The caller zeroes the
 * word at first; adaptq_paged_take_status() reads and zeroes it in one step, beside whatever
 * calls are under way.
 */
#ifndef ADAPTQ_PAGED_H
#define ADAPTQ_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The pool.  Row s of head h in page g starts at ((g * n_kv_heads + h) * page_size + s)
 * rows; padded = the power of two at or above dim.  33 <= dim <= 256, page_size 16, 32,
 * 64, 128 or 256, bits 2, 3 or 4. */
typedef struct {
  void *k_pages, *v_pages;     /* uint8 [n_pages][n_kv_heads][page_size][padded * bits / 8], 16-byte aligned */
  float *k_scales, *v_scales;  /* [n_pages][n_kv_heads][page_size], 16-byte aligned */
  const uint32_t *signs;       /* [n_kv_heads][padded / 32], bit i set: coordinate i is negated */
  int *status;                 /* one word, see above */
  int64_t n_pages;
  int n_kv_heads, page_size, dim, k_bits, v_bits, device;
} adaptq_paged_t;

/* Rotary positions over the first `dim` coordinates of a head: pair i turns by
 * position * turns[i] / 2^64 of a full circle, and is multiplied by `factor`.  Pair i is
 * (x[2i], x[2i+1]) if interleaved, else (x[i], x[i + dim/2]). */
typedef struct {
  const uint64_t *turns;  /* [dim / 2] */
  float factor;
  int dim, interleaved;
} adaptq_rotary_t;

/* y[t][h] = x[t][h] rotated by positions[t] (by -positions[t] if `inverse`: the gradient
 * with respect to x of a forward call, given that of y).  y may be x.  positions: int32, or
 * int64 if positions_64. */
int adaptq_rotary_apply(const adaptq_rotary_t *rotary, const void *x, int64_t x_token_stride, int64_t x_head_stride,
                        void *y, int64_t y_token_stride, int64_t y_head_stride, int type, const void *positions,
                        int positions_64, int64_t n_tokens, int n_heads, int dim, int inverse, int device, void *stream);

/* The sign words that adaptq_mha_create gives the heads of a handle with this seed.
 * words: HOST memory, [n_heads][padded / 32]. */
int adaptq_paged_signs(uint64_t seed, int n_heads, int dim, uint32_t *words);

/* *taken = *status, *status = 0, in one step and in the order of `stream`: bits that calls on
 * other streams set are in this result or in the next. */
int adaptq_paged_take_status(const adaptq_paged_t *cache, int *taken, void *stream);

/* Append.  Tokens cu_tokens[b] .. cu_tokens[b+1]-1 of k and v ([n_tokens][n_kv_heads][dim])
 * belong to sequence b and take its positions starts[b] + start_bias and following; without
 * cu_tokens (NULL) token b belongs to sequence b.  Tokens outside every sequence are left
 * out.  Keys are rotated by their positions first, if `rotary`.  The norm is a float32 sum
 * in an order of its own, so a row equals the one that adaptq_mha_append stores up to the
 * last bit of the norm and codes whose coordinate lies that close to a threshold; rows of
 * norm below 1e-5 are not clipped.  A slot that two tokens of a call share holds parts of
 * either. */
int adaptq_paged_append(const adaptq_paged_t *cache, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                        const void *v, int64_t v_token_stride, int64_t v_head_stride, int type, const int *table,
                        int64_t table_stride, int table_width, const int *starts, int start_bias, const int *cu_tokens,
                        int n_seqs, int64_t n_tokens, const adaptq_rotary_t *rotary, void *stream);

/* Read back: the same tokens as above, as rows of the model: sign * H(codebook[code]) *
 * norm / padded.  Keys come as they were stored, that is rotated.  Rows of k_out and v_out
 * outside every sequence, and rows of pages or positions that do not exist, are left as
 * they were. */
int adaptq_paged_read(const adaptq_paged_t *cache, void *k_out, int64_t k_token_stride, int64_t k_head_stride,
                      void *v_out, int64_t v_token_stride, int64_t v_head_stride, int type, const int *table,
                      int64_t table_stride, int table_width, const int *starts, const int *cu_tokens, int n_seqs,
                      int64_t n_tokens, void *stream);

/* Attention of one new token per sequence over its first lengths[b] tokens.  q, out:
 * [n_seqs][n_q_heads][dim], query head j reading KV head j / (n_q_heads / n_kv_heads).
 * Logits are scale * q.k (scale > 0; the rings' is 1 / sqrt(dim)); queries are rotated by
 * position lengths[b] - 1 first, if `rotary`.  A sequence of length 0 gives zeros.  float32
 * calls are computed to float32's precision throughout (codebook, queries and weights in two
 * float16 parts); float16 calls hold queries and weights in two parts, bfloat16 calls in one,
 * both the codebook in one (off by 1.0e-4 of a value at 4 bits, 3.7e-6 at 3, 1.7e-8 at 2);
 * sums are float32, over at most 4096 tokens at a time.  Tokens are taken 64 at a time (32 above 128 coordinates): one page that
 * does not exist leaves all of its 64 out.
 * workspace: adaptq_paged_attend_workspace() bytes, 16-byte aligned, whose contents need not
 * be kept between calls; calls that may overlap need one each. */
size_t adaptq_paged_attend_workspace(const adaptq_paged_t *cache, int n_seqs, int n_q_heads, int type);
int adaptq_paged_attend(const adaptq_paged_t *cache, const void *q, int64_t q_seq_stride, int64_t q_head_stride,
                        void *out, int64_t out_seq_stride, int64_t out_head_stride, int type, const int *table,
                        int64_t table_stride, int table_width, const int *lengths, int n_seqs, int n_q_heads,
                        float scale, const adaptq_rotary_t *rotary, void *workspace, size_t workspace_bytes,
                        void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ADAPTQ_PAGED_H */
