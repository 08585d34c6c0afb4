/* The recurrent layers of a hybrid decoder: the short causal convolution over the
 * projected channels, and the scan that keeps a matrix of state a head.  The
 * reference's single-token forms are causal_conv1d_step (qwen35.rs:93;
 * si_causal_conv1d_step, metal.rs:745) and GatedDeltaState (qwen35.rs:133;
 * si_gated_delta_step, metal.rs:630-692).
 *
 * Same conventions as si_hip_decode.h: validation before the context is
 * touched, device memory that the caller owns, calls that are asynchronous on
 * the context's stream and recorded while a capture is open.  Everything is f32.
 *
 * Both take `tokens` rows a sequence, row s * tokens + t being token t of
 * sequence s, from one token to whole prompts.  With d_counts sequence s has
 * only min(d_counts[s] + more, tokens) of them; the rows behind are not read
 * and their outputs stay as they were.  d_state NULL: sequences begin (their
 * state is zero).  d_state_out may be d_state, or NULL: the new state is not
 * kept.  The outputs may be NULL where only the state is wanted.  An output
 * that shares memory with an input, a parameter or another output is refused, but for
 * d_state_out = d_state; what lies between the rows of a strided argument is none
 * of it.  So drafted
 * tokens are verified without touching the state, and when it is known how many were
 * accepted a second call with d_counts = the accepted and more = 1 (for the
 * token before them) takes the state that far. */
#ifndef SI_HIP_MIXER_H
#define SI_HIP_MIXER_H

#include <stddef.h>
#include <stdint.h>

#include "si_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- causal convolution ------------------------------------------------------ */
#define SI_HIP_MAX_CONV_WIDTH 8u
#define SI_HIP_CONV_NONE 0u
#define SI_HIP_CONV_SILU 1u /* y / (1 + exp(-y)) */

/* d_y[t][c] = act(d_bias[c] + sum_j d_weight[c * width + j] * x[t - width + 1 + j][c]), a
 * convolution of each channel by itself; inputs before the first token are the
 * state, [sequences][width - 1][channels], the oldest first.  2 <= width <=
 * SI_HIP_MAX_CONV_WIDTH; d_bias NULL: none.  Rows are x_token_stride / y_token_stride floats
 * apart.  A token's output depends on its own and the
 * width - 1 inputs before it alone. */
int si_hip_causal_conv_device(si_hip_context *ctx, size_t sequences, size_t tokens,
                              const uint32_t *d_counts, uint32_t more, size_t channels,
                              size_t width, const float *d_x, size_t x_token_stride,
                              const float *d_weight, const float *d_bias, uint32_t activation,
                              const float *d_state, float *d_state_out, float *d_y,
                              size_t y_token_stride);

/* ---- state scan ---------------------------------------------------------------- */
#define SI_HIP_SCAN_DELTA 0u     /* the gated delta rule */
#define SI_HIP_SCAN_SELECTIVE 1u /* the selective state space form */
#define SI_HIP_SCAN_GROUPED 0u   /* value head h reads key head h / (value_heads / key_heads) */
#define SI_HIP_SCAN_TILED 1u     /* value head h reads key head h % key_heads */

/* A value head's state S is key_dim x value_dim.  With s_t = softplus(gate_t + bias) =
 * ln(1 + exp(gate_t + bias)) and a_t = exp(decay * s_t):
 *   DELTA:     q_t and k_t are divided by sqrt(sum of their squares + eps);
 *              u_t = sigmoid(beta_t) (v_t - a_t S_{t-1}^T k_t)
 *   SELECTIVE: u_t = s_t v_t
 *   S_t = a_t S_{t-1} + k_t u_t^T,  o_t = scale S_t^T q_t + skip v_t
 * decay, bias and skip are one number a value head; bias and skip may be NULL (0).
 * decay is at most 0 where the state is meant to fade. */
typedef struct si_hip_state_scan {
  uint32_t rule;
  uint32_t head_order;
  uint32_t key_heads;   /* of q and k */
  uint32_t value_heads; /* of v, the gates, the state and the output; a multiple of key_heads */
  uint32_t key_dim;     /* at most SI_HIP_MAX_STATE_DIM, like value_dim */
  uint32_t value_dim;
  float scale;
  float eps; /* DELTA: finite, at least 0 */
  const float *d_decay;
  const float *d_bias;
  const float *d_skip;
} si_hip_state_scan;
#define SI_HIP_MAX_STATE_DIM 256u

/* Rows q_token_stride / k_token_stride / v_token_stride floats apart, their heads contiguous (so the
 * three may lie in one row of a convolution's outputs); d_gate and d_beta (SELECTIVE:
 * NULL) contiguous [sequences * tokens][value_heads]; d_state [sequences][value_heads]
 * [key_dim][value_dim]; d_out contiguous [sequences * tokens][value_heads][value_dim].  Without
 * d_out, d_q is not read (NULL then).  A value that is no finite number reaches the outputs and
 * states of its own and later tokens alone.
 *
 * States, sums and decays are f32, or wider.  Single tokens, and rows more than 2^23
 * floats apart, are taken token by token in f32; prompts and most calls of four
 * tokens and more in chunks of 32 on the matrix cores, each f32 operand as a sum of two f16 (22 bits of the
 * largest value of its row or column) or three bf16 (all of its bits), but for
 * SI_HIP_KERNEL_GENERIC: f32 token by token.  What a chunk forgets
 * to less than 2^-126 of it within 32 tokens counts as forgotten, and none grows to 2^127 times what it was.
 * DELTA: a row's squares are added up in f32 (with eps the sum has to be 2^-126 at least, and finite);
 * chunks with a row, but for zeros, that is shorter than 2^-8 of eps's root are taken token by token. */
int si_hip_state_scan_device(si_hip_context *ctx, const si_hip_state_scan *scan, size_t sequences,
                             size_t tokens, const uint32_t *d_counts, uint32_t more,
                             const float *d_q, size_t q_token_stride, const float *d_k,
                             size_t k_token_stride, const float *d_v, size_t v_token_stride,
                             const float *d_gate, const float *d_beta, const float *d_state,
                             float *d_state_out, float *d_out);

#ifdef __cplusplus
}
#endif
#endif /* SI_HIP_MIXER_H */
