/* The operators around the projections of a decode step: rotary positions
 * written into a paged key-value cache, attention of the new tokens over it,
 * eviction by accumulated attention weight, probabilities from logits, and
 * the verification of drafted tokens.  The reference's single-sequence forms
 * of the first two are si_rope (metal.rs:1655), si_attention_decode
 * (metal.rs:1681) and KvCache (cache.rs:10-171); the others have no
 * counterpart there.
 *
 * Same conventions as si_hip.h: SI_HIP_OK or a negative SI_HIP_ERR_* code with
 * a message in si_hip_last_error(), validation before the context is touched,
 * shapes before pointers.  Every *_device call is asynchronous on the
 * context's stream and is recorded while a capture is open.  Activations,
 * weights and probabilities are f32; a cache holds F32, F16 or BF16.  What
 * only the device knows (lengths, page ids, token ids) is checked by the
 * kernels: they leave out what lies out of range, end normally, and the next
 * synchronisation returns SI_HIP_ERR_DEVICE.
 *
 * A decode step, captured once and replayed: si_hip_rope_append_device,
 * si_hip_paged_attention_device, ..., si_hip_softmax_device,
 * si_hip_verify_draft_device, si_hip_kv_advance_device. */
#ifndef SI_HIP_DECODE_H
#define SI_HIP_DECODE_H

#include <stddef.h>
#include <stdint.h>

#include "si_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SI_HIP_GGML_TYPE_F32 0u
#define SI_HIP_GGML_TYPE_F16 1u
#define SI_HIP_GGML_TYPE_BF16 30u

#define SI_HIP_MAX_HEAD_DIM 256u
/* New tokens a sequence may bring to one attention call, and drafted tokens
 * to one verification: the batch that the multi-token projections take. */
#define SI_HIP_MAX_STEP_TOKENS SI_HIP_MAX_BATCH

/* A paged key-value cache in device memory that the caller owns.  Sequence s
 * holds d_lengths[s] tokens in slots 0, 1, ...; slot i of head h is row
 * i % page_tokens of page d_page_table[s * max_pages + i / page_tokens]:
 * d_keys and d_values are [pages][kv_heads][page_tokens][head_dim] of
 * ggml_type (F32, F16 or BF16).  Keys are held rotated.  A sequence's
 * capacity is max_pages * page_tokens slots; table entries behind the slots
 * in use are not read. */
typedef struct si_hip_kv_cache {
  uint32_t ggml_type;
  uint32_t kv_heads;
  uint32_t head_dim; /* at most SI_HIP_MAX_HEAD_DIM */
  uint32_t page_tokens;
  uint32_t pages;
  uint32_t sequences;
  uint32_t max_pages;
  uint32_t reserved; /* 0 */
  void *d_keys;
  void *d_values;
  const uint32_t *d_page_table;
  uint32_t *d_lengths;
} si_hip_kv_cache;

/* ---- rotary positions ---------------------------------------------------- */
#define SI_HIP_ROPE_HALF 0u        /* pairs (i, i + rotary_dim / 2) */
#define SI_HIP_ROPE_INTERLEAVED 1u /* pairs (2 i, 2 i + 1) */

#define SI_HIP_ROPE_SCALING_NONE 0u
#define SI_HIP_ROPE_SCALING_LINEAR 1u /* frequencies / factor */
#define SI_HIP_ROPE_SCALING_YARN 2u   /* long waves / factor, short ones kept, a ramp between */

/* Rotation of the first rotary_dim values of a head by position p: pair i
 * turns by p * d_frequencies[i] / 2^64 of a full turn, (a, b) -> magnitude *
 * (a cos - b sin, b cos + a sin).  As fractions of a turn in 64-bit fixed
 * point the product's whole turns drop out in the wrapping multiplication, so
 * an entry's own error, times the position, is the angle's: half a unit of
 * 2^-64 of a turn makes 2^-33 at position 2^32 - 1. */
typedef struct si_hip_rope {
  uint32_t layout;
  uint32_t rotary_dim; /* even, at least 2 */
  float magnitude;
  uint32_t reserved;             /* 0 */
  const uint64_t *d_frequencies; /* rotary_dim / 2 entries, device memory */
} si_hip_rope;

/* Host computation of such a table: frequency i is theta^(-2 i / rotary_dim)
 * radians a position, theta >= 1.  LINEAR divides all by `factor` (> 0).  YARN:
 * with dim(t) = rotary_dim ln(original_length / (2 pi t)) / (2 ln theta), the
 * pair that turns t times within original_length positions, the frequencies
 * go from unchanged at floor(dim(beta_fast)) to divided by factor at
 * ceil(dim(beta_slow)) along a linear ramp, and *magnitude is
 * 0.1 ln(factor) + 1 where factor > 1 (1 else, and without YARN).  factor,
 * original_length and the betas are read where the scaling uses them.  Entries
 * are good to two units of 2^-64 of a turn where factor >= 1. */
int si_hip_rope_frequencies(size_t rotary_dim, double theta, uint32_t scaling, double factor,
                            double original_length, double beta_fast, double beta_slow,
                            uint64_t *frequencies, float *magnitude);

/* Rotates rows of `heads` heads: token t's head h is at d_x + t * token_stride +
 * h * head_stride (floats), its position d_positions[t]; d_y is laid out with
 * its own strides and may be d_x with the same ones.  Values behind
 * rotary_dim are copied. */
int si_hip_rope_device(si_hip_context *ctx, const si_hip_rope *rope, const float *d_x,
                       size_t tokens, size_t heads, size_t head_dim, size_t token_stride,
                       size_t head_stride, const uint32_t *d_positions, float *d_y,
                       size_t y_token_stride, size_t y_head_stride);

/* One launch that takes `tokens` new tokens a sequence into the cache: rotates
 * their keys (rope NULL: not) and stores them, and their values, in the slots
 * behind d_lengths[s], which it leaves as it is.  Row s * tokens + t belongs to
 * token t of sequence s; k and v rows are kv_heads * head_dim floats,
 * k_token_stride / v_token_stride apart.  With d_counts sequence s brings only
 * d_counts[s] <= tokens of them; the rows behind are not read.  d_positions
 * (NULL: the slots' numbers) has a position for each row.  With d_q, the same
 * launch rotates the rows' `heads` query heads into d_q_out (contiguous rows
 * of heads * head_dim; d_q itself where it is laid out so). */
int si_hip_rope_append_device(si_hip_context *ctx, const si_hip_kv_cache *cache,
                              const si_hip_rope *rope, size_t tokens, const uint32_t *d_counts,
                              const uint32_t *d_positions, const float *d_k, size_t k_token_stride,
                              const float *d_v, size_t v_token_stride, const float *d_q,
                              size_t heads, size_t q_token_stride, size_t q_head_stride,
                              float *d_q_out);

/* d_lengths[s] += d_counts[s] (NULL: 0) + more, at most the capacity: the new
 * tokens become part of the sequence (after a verification: the accepted
 * drafts, and `more` = 1 for the token whose row they followed). */
int si_hip_kv_advance_device(si_hip_context *ctx, const si_hip_kv_cache *cache,
                             const uint32_t *d_counts, uint32_t more);

/* ---- norms of heads, positions of several axes ------------------------------ */
/* RMS norm of a head's values before they turn: y = x * inv * w, or with plus_one
 * x * inv * (1 + w), inv = 1 / sqrt(mean(x^2) + eps) over head_dim values (the
 * squares' sum has to be within f32's range); a
 * weight that is NULL is all ones (plus_one does not apply to it). */
typedef struct si_hip_head_norm {
  float eps;         /* finite, above 0 */
  uint32_t plus_one; /* 0 or 1 */
  const float *d_q_weight; /* head_dim entries, device memory: rows of queries, and of
                              si_hip_norm_rope_device */
  const float *d_k_weight; /* those of keys */
} si_hip_head_norm;

/* Positions of several axes (time, height and width of an image's or a video's
 * patches): pair i turns by the row's position on axis d_axis[i].  An entry of
 * `axes` or more is reported, and counts as axis 0. */
#define SI_HIP_MAX_ROPE_AXES 4u
typedef struct si_hip_rope_axes {
  uint32_t axes;         /* 1..SI_HIP_MAX_ROPE_AXES */
  uint32_t reserved;     /* 0 */
  const uint8_t *d_axis; /* rotary_dim / 2 entries, device memory */
} si_hip_rope_axes;

/* Host computation of such a table from the number of pairs each axis has (their sum
 * is rotary_dim / 2).  BLOCKS: axis 0's pairs, then axis 1's, ...  TURNS: pair i belongs to
 * axis a = i mod axes while i < axes * sections[a], to axis 0 otherwise; sections that do not
 * come out so are refused. */
#define SI_HIP_ROPE_AXES_BLOCKS 0u
#define SI_HIP_ROPE_AXES_TURNS 1u
int si_hip_rope_axis_table(size_t rotary_dim, const uint32_t *sections, size_t axes, uint32_t order,
                           uint8_t *axis);

/* si_hip_rope_device with the heads' norm before the rotation, and positions of one
 * or several axes: d_positions[axis * tokens + t].  norm NULL: rotation alone; rope NULL: the norm
 * alone (no axes, no positions).  One of the two is there.  d_y may be d_x with the same strides;
 * other rows of it that share memory with d_x, or with a parameter, are refused. */
int si_hip_norm_rope_device(si_hip_context *ctx, const si_hip_head_norm *norm,
                            const si_hip_rope *rope, const si_hip_rope_axes *axes,
                            const float *d_x, size_t tokens, size_t heads, size_t head_dim,
                            size_t token_stride, size_t head_stride, const uint32_t *d_positions,
                            float *d_y, size_t y_token_stride, size_t y_head_stride);

/* si_hip_rope_append_device with the norms of query and key heads before their rotation, in
 * the same launch, and positions of one or several axes: d_positions[axis * sequences * tokens +
 * s * tokens + t] (NULL: the slots' numbers, on every axis).  norm NULL: none.  Query rows need a
 * norm or a rotation.  d_q_out that shares memory with k, v, a parameter or, but for d_q itself, q is
 * refused. */
int si_hip_norm_rope_append_device(si_hip_context *ctx, const si_hip_kv_cache *cache,
                                   const si_hip_head_norm *norm, const si_hip_rope *rope,
                                   const si_hip_rope_axes *axes, size_t tokens,
                                   const uint32_t *d_counts, const uint32_t *d_positions,
                                   const float *d_k, size_t k_token_stride, const float *d_v,
                                   size_t v_token_stride, const float *d_q, size_t heads,
                                   size_t q_token_stride, size_t q_head_stride, float *d_q_out);

/* ---- attention ----------------------------------------------------------- */
/* Attention of 1..SI_HIP_MAX_STEP_TOKENS new tokens a sequence whose rows are
 * in the cache behind d_lengths[s]: token t attends to the slots below n =
 * d_lengths[s] + t + 1, with window > 0 to the last `window` of them.
 * out = sum_i p_i v_i, p_i = exp(scale q.k_i) / sum; query head h reads kv head
 * h / (heads / kv_heads).  Rows d_q + (s * tokens + t) * q_token_stride + h *
 * q_head_stride; d_out contiguous [sequences][tokens][heads][head_dim].  A row
 * with nothing to attend to (t >= d_counts[s], slots on pages beyond the pool)
 * is zeros.  Slots that a row does not see have no part in it, whatever they
 * hold: NaN and infinities in them do not reach it, and a page before the window
 * may lie beyond the pool.  A row that sees a key or value that is no finite
 * number is not a number, in part or as a whole.
 * Sums, maxima and exponentials are f32.  Over an F16 cache a row's query values
 * are held to 22 bits down to 2^-28 of the largest and smaller ones to 2^-51 of it,
 * its p_i to 22 bits down to 2^-17 of the largest and smaller ones to 2^-39 of it;
 * over the others both to 24 bits.
 *
 * With d_weights, [sequences][kv_heads][weights_stride], entry i of kv head h
 * grows by the sum of p_i over the head's query heads and the new tokens;
 * weights_stride is at least the capacity.  Entries of slots that a later call
 * fills anew (refused drafts') are the caller's to clear.
 *
 * d_workspace: si_hip_paged_attention_workspace() bytes of 16-byte aligned
 * device memory that this call may write until it has run.  With d_weights they
 * hold a score for each row and slot of the capacity, whatever the lengths are:
 * 4 * sequences * tokens * heads * capacity bytes beside the rest. */
size_t si_hip_paged_attention_workspace(const si_hip_kv_cache *cache, size_t heads, size_t tokens,
                                        int with_weights); /* 0: invalid arguments */
int si_hip_paged_attention_device(si_hip_context *ctx, const si_hip_kv_cache *cache, size_t heads,
                                  size_t tokens, uint32_t window, float scale,
                                  const uint32_t *d_counts, const float *d_q,
                                  size_t q_token_stride, size_t q_head_stride, float *d_out,
                                  float *d_weights, size_t weights_stride, void *d_workspace,
                                  size_t workspace_bytes);

/* ---- eviction ------------------------------------------------------------ */
/* Every kv head of a sequence that holds more than `keep` tokens keeps keep of
 * them: the first `sinks`, the last `recent` (sinks + recent <= keep), and of
 * the others those of the largest d_weights [sequences][kv_heads]
 * [weights_stride], the lower slot where two are equal (a NaN weighs least).
 * The kept rows go, in their order, to slots 0, 1, ... of `to`, and their
 * weights to d_to_weights; to->d_lengths becomes min(length, keep).  `to` has
 * the type, heads and sequences of `from` and a capacity of keep at least; it
 * may lie in the same pool, on pages that `from`'s table does not name (none of
 * the buffers written may be one that is read).  d_kept, [sequences][kv_heads]
 * [keep], receives the kept slots, 0xffffffff behind the last. */
int si_hip_kv_evict_device(si_hip_context *ctx, const si_hip_kv_cache *from,
                           const float *d_weights, size_t weights_stride, size_t keep,
                           size_t sinks, size_t recent, const si_hip_kv_cache *to,
                           float *d_to_weights, size_t to_weights_stride, uint32_t *d_kept);

/* ---- probabilities and verification -------------------------------------- */
/* d_y[r] = softmax(d_x[r] / temperature) of rows x cols contiguous floats,
 * temperature at least 1e-30 and finite.  d_y may be d_x. */
int si_hip_softmax_device(si_hip_context *ctx, const float *d_x, size_t rows, size_t cols,
                          float temperature, float *d_y);

#define SI_HIP_TOKEN_NONE 0xffffffffu
/* Verification of drafted tokens, `drafts` (1..SI_HIP_MAX_STEP_TOKENS) a
 * sequence or d_counts[s] <= drafts (0 too) of them.  d_target [sequences]
 * [drafts + 1][vocab]: the target's probabilities p before each draft and
 * after the last; d_draft [sequences][drafts][vocab]: the drafter's q (NULL: it
 * drafts with certainty, q is 1 at its token and 0 elsewhere); d_uniform
 * [sequences][drafts + 1]: numbers in [0, 1).
 * Draft i, token x, is accepted while u_i q_i(x) < p_i(x).  After the first
 * that is not, the next token is drawn from max(p_i - q_i, 0), or, where that
 * is zero throughout or all drafts were accepted, from p: the lowest token whose
 * running sum exceeds u_drafts, taken down to a multiple of 2^-24, times the
 * whole sum.  Each term is clamped to [0, 1] (a NaN counts as 0) and taken down
 * to a multiple of 2^-36, so the sums (below 2^28) are exact in any order and so
 * is the token.
 * d_accepted[s]: the number accepted; d_out_tokens [sequences][drafts + 1]:
 * those tokens, the drawn one, then SI_HIP_TOKEN_NONE.  A drafted token beyond
 * the vocabulary is refused and reported; so is a row of probabilities that is
 * zero throughout, whose drawn token is SI_HIP_TOKEN_NONE. */
int si_hip_verify_draft_device(si_hip_context *ctx, const float *d_target, const float *d_draft,
                               const uint32_t *d_tokens, const uint32_t *d_counts,
                               const float *d_uniform, size_t sequences, size_t drafts,
                               size_t vocab, uint32_t *d_accepted, uint32_t *d_out_tokens);

#ifdef __cplusplus
}
#endif
#endif /* SI_HIP_DECODE_H */
