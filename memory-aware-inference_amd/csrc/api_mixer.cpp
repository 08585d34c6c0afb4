// C ABI of a hybrid decoder's recurrent layers (include/si_hip_mixer.h): their
// checks, which need no device, and the hand-over to the kernels' launch functions.
#include "si_hip_mixer.h"

#include <hip/hip_runtime.h>

#include <cmath>

#include "mixer_internal.h"
#include "overlap.h"
#include "si_hip_status.h"

using namespace sihip;

namespace {

template <class F>
int submit(si_hip_context *ctx, const char *what, F launch) {
  return submit_device(
      ctx, what,
      [](void *f, const Workspace &ws, hipStream_t s, bool tuned) {
        return (*static_cast<F *>(f))(ws, s, tuned);
      },
      &launch);
}

bool product(size_t a, size_t b, size_t *out) { return !__builtin_mul_overflow(a, b, out); }

// sequences * tokens rows: within the kernels' 31 bits, the sequences within a grid's
int check_rows(size_t sequences, size_t tokens, const uint32_t *d_counts, uint32_t more,
               const char *what) {
  size_t rows;
  if (sequences == 0 || tokens == 0 || (more && !d_counts))
    return set_error(SI_HIP_ERR_DIMENSIONS, "%s rows are invalid", what);
  if (sequences > 65535u || !product(sequences, tokens, &rows) || rows > 0x7fffffffu)
    return set_error(SI_HIP_ERR_OVERFLOW, "%s rows exceed HIP limits", what);
  return SI_HIP_OK;
}

// Rows of `size` floats, `stride` apart.
int check_stride(size_t stride, size_t size, const char *what) {
  if (stride < size)
    return set_error(SI_HIP_ERR_DIMENSIONS, "%s strides are shorter than their rows", what);
  if (stride > SIZE_MAX / 16 / 0x7fffffffu)
    return set_error(SI_HIP_ERR_OVERFLOW, "%s strides overflow", what);
  return SI_HIP_OK;
}

}  // namespace

extern "C" {

int si_hip_causal_conv_device(si_hip_context *ctx, size_t sequences, size_t tokens,
                              const uint32_t *d_counts, uint32_t more, size_t channels,
                              size_t width, const float *d_x, size_t x_token_stride,
                              const float *d_weight, const float *d_bias, uint32_t activation,
                              const float *d_state, float *d_state_out, float *d_y,
                              size_t y_token_stride) {
  int rc = check_rows(sequences, tokens, d_counts, more, "causal convolution");
  if (rc) return rc;
  if (activation > SI_HIP_CONV_SILU)
    return set_error(SI_HIP_ERR_UNSUPPORTED_TYPE, "unsupported activation %u", activation);
  if (channels == 0 || width < 2 || width > SI_HIP_MAX_CONV_WIDTH)
    return set_error(SI_HIP_ERR_DIMENSIONS, "causal convolution dimensions are invalid");
  if (channels > 0x7fffff00u)
    return set_error(SI_HIP_ERR_OVERFLOW, "causal convolution dimensions exceed HIP limits");
  if ((rc = check_stride(x_token_stride, channels, "causal convolution")) != 0) return rc;
  if (d_y && (rc = check_stride(y_token_stride, channels, "causal convolution")) != 0) return rc;
  if (!ctx || !d_x || !d_weight || (!d_y && !d_state_out))
    return set_error(SI_HIP_ERR_NULL, "device causal convolution argument is null");
  const size_t rows = sequences * tokens, held = sequences * (width - 1);
  const Region y(d_y, rows, 4 * y_token_stride, 4 * channels);
  const Region state(d_state, held, 4 * channels, 4 * channels);
  const Region state_out(d_state_out, held, 4 * channels, 4 * channels);
  const Region in[] = {Region(d_x, rows, 4 * x_token_stride, 4 * channels),
                       Region(d_weight, channels, 4 * width, 4 * width),
                       Region(d_bias, 4 * channels), Region(d_counts, 4 * sequences)};
  if (overlaps_any(y, in) || overlaps_any(state_out, in) || overlap(y, state) ||
      overlap(y, state_out) || (d_state_out != d_state && overlap(state_out, state)))
    return set_error(SI_HIP_ERR_RANGE, "causal convolution writes what it reads");
  const ConvArgs a{(uint32_t)sequences,
                   (uint32_t)channels,
                   (uint32_t)width,
                   activation == SI_HIP_CONV_SILU,
                   Counts{d_counts, more, (uint32_t)tokens},
                   d_x,
                   d_weight,
                   d_bias,
                   d_state,
                   d_state_out,
                   d_y,
                   x_token_stride,
                   y_token_stride};
  return submit(ctx, "causal convolution launch", [&](const Workspace &, hipStream_t s, bool) {
    return launch_conv(a, s);
  });
}

int si_hip_state_scan_device(si_hip_context *ctx, const si_hip_state_scan *scan, size_t sequences,
                             size_t tokens, const uint32_t *d_counts, uint32_t more,
                             const float *d_q, size_t q_token_stride, const float *d_k,
                             size_t k_token_stride, const float *d_v, size_t v_token_stride,
                             const float *d_gate, const float *d_beta, const float *d_state,
                             float *d_state_out, float *d_out) {
  if (!scan) return set_error(SI_HIP_ERR_NULL, "state scan description is null");
  if (scan->rule > SI_HIP_SCAN_SELECTIVE)
    return set_error(SI_HIP_ERR_UNSUPPORTED_TYPE, "unsupported scan rule %u", scan->rule);
  if (scan->head_order > SI_HIP_SCAN_TILED)
    return set_error(SI_HIP_ERR_UNSUPPORTED_TYPE, "unsupported order of scan heads %u",
                     scan->head_order);
  const bool delta = scan->rule == SI_HIP_SCAN_DELTA;
  if (scan->key_heads == 0 || scan->value_heads == 0 ||
      scan->value_heads % scan->key_heads != 0 || scan->key_dim == 0 ||
      scan->key_dim > SI_HIP_MAX_STATE_DIM || scan->value_dim == 0 ||
      scan->value_dim > SI_HIP_MAX_STATE_DIM || !std::isfinite(scan->scale) ||
      (delta && !(std::isfinite(scan->eps) && scan->eps >= 0.0f)))
    return set_error(SI_HIP_ERR_DIMENSIONS, "state scan dimensions are invalid");
  if (scan->value_heads > 65535u)
    return set_error(SI_HIP_ERR_OVERFLOW, "state scan heads exceed HIP limits");
  int rc = check_rows(sequences, tokens, d_counts, more, "state scan");
  if (rc) return rc;
  const size_t key_row = (size_t)scan->key_heads * scan->key_dim;
  const size_t value_row = (size_t)scan->value_heads * scan->value_dim;
  if (d_out && (rc = check_stride(q_token_stride, key_row, "state scan query")) != 0) return rc;
  if ((rc = check_stride(k_token_stride, key_row, "state scan key")) != 0) return rc;
  if ((rc = check_stride(v_token_stride, value_row, "state scan value")) != 0) return rc;
  if (!ctx || !scan->d_decay || !d_k || !d_v || !d_gate || (delta && !d_beta) ||
      (d_out && !d_q) || (!d_out && !d_state_out))
    return set_error(SI_HIP_ERR_NULL, "device state scan argument is null");
  const size_t rows = sequences * tokens, gates = 4 * (size_t)scan->value_heads;
  const size_t held = 4 * value_row * scan->key_dim;
  const Region out(d_out, rows, 4 * value_row, 4 * value_row);
  const Region state(d_state, sequences, held, held), state_out(d_state_out, sequences, held, held);
  const Region in[] = {Region(d_out ? d_q : nullptr, rows, 4 * q_token_stride, 4 * key_row),
                       Region(d_k, rows, 4 * k_token_stride, 4 * key_row),
                       Region(d_v, rows, 4 * v_token_stride, 4 * value_row),
                       Region(d_gate, rows, gates, gates),
                       Region(delta ? d_beta : nullptr, rows, gates, gates),
                       Region(scan->d_decay, gates), Region(scan->d_bias, gates),
                       Region(scan->d_skip, gates), Region(d_counts, 4 * sequences)};
  if (overlaps_any(out, in) || overlaps_any(state_out, in) || overlap(out, state) ||
      overlap(out, state_out) || (d_state_out != d_state && overlap(state_out, state)))
    return set_error(SI_HIP_ERR_RANGE, "state scan writes what it reads");
  const ScanArgs a{delta,
                   scan->head_order == SI_HIP_SCAN_TILED,
                   (uint32_t)sequences,
                   scan->key_heads,
                   scan->value_heads,
                   scan->key_dim,
                   scan->value_dim,
                   divisor_of(scan->head_order == SI_HIP_SCAN_TILED
                                  ? scan->key_heads
                                  : scan->value_heads / scan->key_heads),
                   scan->scale,
                   scan->eps,
                   Counts{d_counts, more, (uint32_t)tokens},
                   scan->d_decay,
                   scan->d_bias,
                   scan->d_skip,
                   d_q,
                   d_k,
                   d_v,
                   d_gate,
                   d_beta,
                   d_state,
                   d_state_out,
                   d_out,
                   q_token_stride,
                   k_token_stride,
                   v_token_stride};
  return submit(ctx, "state scan launch", [&](const Workspace &, hipStream_t s, bool tuned) {
    return launch_scan(a, tuned, s);
  });
}

}  // extern "C"
