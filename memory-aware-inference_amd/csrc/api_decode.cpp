// C ABI of the decode-step operators (include/si_hip_decode.h): their checks,
// which need no device, and the hand-over to the kernels' launch functions.
#include "si_hip_decode.h"

#include <hip/hip_runtime.h>

#include <cmath>

#include "decode_internal.h"
#include "si_hip_status.h"

using namespace sihip;

namespace {

// A lambda `launch(workspace, stream, tuned)` as one device call.
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

// A cache's shape; then `view` is what the kernels take.
int check_cache(const si_hip_kv_cache *c, CacheView *view) {
  if (!c) return set_error(SI_HIP_ERR_NULL, "key-value cache is null");
  if (c->ggml_type != kKvF32 && c->ggml_type != kKvF16 && c->ggml_type != kKvBF16)
    return set_error(SI_HIP_ERR_UNSUPPORTED_TYPE, "unsupported key-value cache type %u",
                     c->ggml_type);
  if (c->kv_heads == 0 || c->head_dim == 0 || c->head_dim > SI_HIP_MAX_HEAD_DIM ||
      c->page_tokens == 0 || c->pages == 0 || c->sequences == 0 || c->max_pages == 0)
    return set_error(SI_HIP_ERR_DIMENSIONS, "key-value cache dimensions are invalid");
  size_t capacity, rows;
  if (!product(c->max_pages, c->page_tokens, &capacity) || capacity > 0x7fffff00u ||
      !product((size_t)c->pages * c->kv_heads, c->page_tokens, &rows) || rows > 0xffffffffu ||
      c->kv_heads > 65535u || c->sequences > 65535u)
    return set_error(SI_HIP_ERR_OVERFLOW, "key-value cache dimensions exceed HIP limits");
  *view = CacheView{c->ggml_type, c->kv_heads, c->head_dim, c->page_tokens, c->pages, c->sequences,
                    c->max_pages, (uint32_t)capacity, 0, 0, c->d_keys, c->d_values,
                    c->d_page_table, c->d_lengths};
  division_by(c->page_tokens, &view->div_mul, &view->div_shift);
  return SI_HIP_OK;
}

int check_cache_buffers(const CacheView &v) {
  if (!v.keys || !v.values || !v.table || !v.lengths)
    return set_error(SI_HIP_ERR_NULL, "key-value cache buffer is null");
  const uintptr_t size = v.type == kKvF32 ? 4u : 2u;
  if (((uintptr_t)v.keys | (uintptr_t)v.values) % size != 0)
    return set_error(SI_HIP_ERR_RANGE, "key-value cache pages are not aligned to their type");
  return SI_HIP_OK;
}

int check_rope(const si_hip_rope *r, size_t head_dim) {
  if (r->layout > SI_HIP_ROPE_INTERLEAVED)
    return set_error(SI_HIP_ERR_UNSUPPORTED_TYPE, "unsupported rotary layout %u", r->layout);
  if (r->rotary_dim == 0 || r->rotary_dim % 2 != 0 || r->rotary_dim > head_dim ||
      !std::isfinite(r->magnitude))
    return set_error(SI_HIP_ERR_DIMENSIONS, "rotary dimensions are invalid");
  if (!r->d_frequencies) return set_error(SI_HIP_ERR_NULL, "rotary frequencies are null");
  return SI_HIP_OK;
}
RopeArgs rope_args(const si_hip_rope *r) {
  return {r->layout, r->rotary_dim, r->magnitude, r->d_frequencies};
}

// sequences * tokens rows of a step: within the kernels' 31 bits
int check_step(const CacheView &v, size_t tokens, size_t most, const char *what) {
  size_t rows;
  if (tokens == 0 || tokens > most)
    return set_error(SI_HIP_ERR_BATCH, "%s takes 1..%zu new tokens a sequence", what, most);
  if (!product(v.sequences, tokens, &rows) || rows > 0x7fffffffu)
    return set_error(SI_HIP_ERR_OVERFLOW, "%s rows exceed HIP limits", what);
  return SI_HIP_OK;
}

int check_heads(const CacheView &v, size_t heads) {
  if (heads == 0 || heads % v.kv_heads != 0)
    return set_error(SI_HIP_ERR_DIMENSIONS, "query heads are not a multiple of the cache's heads");
  if (heads > 65535u) return set_error(SI_HIP_ERR_OVERFLOW, "query heads exceed HIP limits");
  return SI_HIP_OK;
}

// The kept scores of a call with weights: a row of slots for each row of queries.
int check_scores(const CacheView &v, size_t heads, size_t tokens) {
  size_t n;
  if (!product((size_t)v.sequences * heads * tokens, (size_t)v.capacity + 3u, &n) ||
      n > SIZE_MAX / 16)
    return set_error(SI_HIP_ERR_OVERFLOW, "attention weights exceed HIP limits");
  return SI_HIP_OK;
}

// Rows of heads a stride apart hold `heads` heads of `dim` values each.
int check_strides(size_t token_stride, size_t head_stride, size_t heads, size_t dim,
                  const char *what) {
  size_t span;
  if (!product(heads - 1, head_stride, &span) || span > SIZE_MAX / 16 - dim)
    return set_error(SI_HIP_ERR_OVERFLOW, "%s strides overflow", what);
  if (head_stride < dim || token_stride < span + dim)
    return set_error(SI_HIP_ERR_DIMENSIONS, "%s strides are shorter than their rows", what);
  return SI_HIP_OK;
}

}  // namespace

extern "C" {

int si_hip_rope_frequencies(size_t rotary_dim, double theta, uint32_t scaling, double factor,
                            double original_length, double beta_fast, double beta_slow,
                            uint64_t *frequencies, float *magnitude) {
  if (scaling > SI_HIP_ROPE_SCALING_YARN)
    return set_error(SI_HIP_ERR_UNSUPPORTED_TYPE, "unsupported rotary scaling %u", scaling);
  const bool yarn = scaling == SI_HIP_ROPE_SCALING_YARN;
  if (rotary_dim == 0 || rotary_dim % 2 != 0 || rotary_dim > SI_HIP_MAX_HEAD_DIM ||
      !std::isfinite(theta) || theta < 1.0 || (yarn && theta <= 1.0) ||
      (scaling != SI_HIP_ROPE_SCALING_NONE && !(std::isfinite(factor) && factor > 0.0)) ||
      (yarn && !(std::isfinite(original_length) && original_length > 0.0 &&
                 std::isfinite(beta_fast) && std::isfinite(beta_slow) && beta_slow > 0.0 &&
                 beta_fast >= beta_slow)))
    return set_error(SI_HIP_ERR_DIMENSIONS, "rotary scaling parameters are invalid");
  if (!frequencies || !magnitude) return set_error(SI_HIP_ERR_NULL, "rotary frequencies are null");
  // (Arithmetic of 64 bits, for 64-bit entries: with one of 53 the angle 2^32 positions on would
  // be off by up to 2^-25 of a turn.)
  const long double n = (long double)rotary_dim, pi = 3.14159265358979323846264338327950288L;
  long double low = 0.0L, high = 0.0L;
  if (yarn) {
    auto dim = [&](long double turns) {
      return n * std::log(original_length / (2.0L * pi * turns)) /
             (2.0L * std::log((long double)theta));
    };
    low = std::fmax(std::floor(dim(beta_fast)), 0.0L);
    high = std::fmin(std::ceil(dim(beta_slow)), n - 1.0L);
  }
  for (size_t i = 0; i < rotary_dim / 2; ++i) {
    long double f = std::pow((long double)theta, -2.0L * (long double)i / n);
    if (scaling == SI_HIP_ROPE_SCALING_LINEAR) {
      f /= factor;
    } else if (yarn) {
      const long double at = ((long double)i - low) / std::fmax(high - low, 0.001L);
      const long double ramp = std::fmin(std::fmax(at, 0.0L), 1.0L);
      f = f / factor * ramp + f * (1.0L - ramp);
    }
    // the fraction of a turn: whole turns a position (factor < 1) change no angle
    long double turns = f / (2.0L * pi);
    turns -= std::floor(turns);
    const long double fixed = std::rint(turns * 18446744073709551616.0L);
    frequencies[i] = fixed >= 18446744073709551616.0L ? 0u : (uint64_t)fixed;
  }
  *magnitude = yarn && factor > 1.0 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  return clear_error();
}

int si_hip_rope_device(si_hip_context *ctx, const si_hip_rope *rope, const float *d_x,
                       size_t tokens, size_t heads, size_t head_dim, size_t token_stride,
                       size_t head_stride, const uint32_t *d_positions, float *d_y,
                       size_t y_token_stride, size_t y_head_stride) {
  if (!rope) return set_error(SI_HIP_ERR_NULL, "rotary description is null");
  if (tokens == 0 || heads == 0 || head_dim == 0 || head_dim > SI_HIP_MAX_HEAD_DIM)
    return set_error(SI_HIP_ERR_DIMENSIONS, "rotary dimensions are invalid");
  int rc = check_rope(rope, head_dim);
  if (rc) return rc;
  if (tokens > 0x7fffffffu || heads > 0xffffu)
    return set_error(SI_HIP_ERR_OVERFLOW, "rotary rows exceed HIP limits");
  rc = check_strides(token_stride, head_stride, heads, head_dim, "rotary input");
  if (rc) return rc;
  rc = check_strides(y_token_stride, y_head_stride, heads, head_dim, "rotary output");
  if (rc) return rc;
  if (!ctx || !d_x || !d_positions || !d_y)
    return set_error(SI_HIP_ERR_NULL, "device rotary argument is null");
  if (d_x == d_y && (token_stride != y_token_stride || head_stride != y_head_stride))
    return set_error(SI_HIP_ERR_DIMENSIONS, "rotation in place needs one set of strides");
  const RopeRows rows{d_x, d_y, token_stride, head_stride, y_token_stride, y_head_stride,
                      (uint32_t)heads};
  return submit(ctx, "rotary launch", [&](const Workspace &, hipStream_t s, bool) {
    return launch_rope(rope_args(rope), rows, (uint32_t)tokens, (uint32_t)head_dim, d_positions, s);
  });
}

int si_hip_rope_append_device(si_hip_context *ctx, const si_hip_kv_cache *cache,
                              const si_hip_rope *rope, size_t tokens, const uint32_t *d_counts,
                              const uint32_t *d_positions, const float *d_k, size_t k_token_stride,
                              const float *d_v, size_t v_token_stride, const float *d_q,
                              size_t heads, size_t q_token_stride, size_t q_head_stride,
                              float *d_q_out) {
  CacheView view;
  int rc = check_cache(cache, &view);
  if (rc) return rc;
  if (rope && (rc = check_rope(rope, view.head_dim)) != 0) return rc;
  if ((rc = check_step(view, tokens, 0x7fffffffu, "cache append")) != 0) return rc;
  const size_t dim = view.head_dim;
  for (size_t stride : {k_token_stride, v_token_stride})
    if ((rc = check_strides(stride, dim, view.kv_heads, dim, "cache append")) != 0) return rc;
  if (d_q) {
    if ((rc = check_heads(view, heads)) != 0) return rc;
    if ((rc = check_strides(q_token_stride, q_head_stride, heads, dim, "query")) != 0) return rc;
    if (!rope) return set_error(SI_HIP_ERR_NULL, "query rows need a rotary description");
    if (!d_q_out) return set_error(SI_HIP_ERR_NULL, "query output is null");
    if (d_q == d_q_out && (q_head_stride != dim || q_token_stride != heads * dim))
      return set_error(SI_HIP_ERR_DIMENSIONS, "rotation in place needs contiguous query rows");
  }
  if (!ctx || !d_k || !d_v) return set_error(SI_HIP_ERR_NULL, "cache append argument is null");
  if ((rc = check_cache_buffers(view)) != 0) return rc;
  const RopeArgs r = rope ? rope_args(rope) : RopeArgs{};
  const RopeRows q{d_q, d_q_out, q_token_stride, q_head_stride, heads * dim, dim, (uint32_t)heads};
  return submit(ctx, "cache append launch", [&](const Workspace &ws, hipStream_t s, bool) {
    return launch_rope_append(view, rope ? &r : nullptr, (uint32_t)tokens, d_counts, d_positions,
                              d_k, k_token_stride, d_v, v_token_stride, d_q ? &q : nullptr, ws.ptr,
                              s);
  });
}

int si_hip_kv_advance_device(si_hip_context *ctx, const si_hip_kv_cache *cache,
                             const uint32_t *d_counts, uint32_t more) {
  CacheView view;
  int rc = check_cache(cache, &view);
  if (rc) return rc;
  if (!ctx || !view.lengths) return set_error(SI_HIP_ERR_NULL, "cache advance argument is null");
  return submit(ctx, "cache advance launch", [&](const Workspace &, hipStream_t s, bool) {
    return launch_kv_advance(view, d_counts, more, s);
  });
}

size_t si_hip_paged_attention_workspace(const si_hip_kv_cache *cache, size_t heads, size_t tokens,
                                        int with_weights) {
  CacheView view;
  if (check_cache(cache, &view) || check_step(view, tokens, SI_HIP_MAX_STEP_TOKENS, "attention") ||
      check_heads(view, heads) || (with_weights && check_scores(view, heads, tokens)))
    return 0;
  clear_error();
  return attention_workspace_bytes(view, (uint32_t)heads, (uint32_t)tokens, with_weights != 0);
}

int si_hip_paged_attention_device(si_hip_context *ctx, const si_hip_kv_cache *cache, size_t heads,
                                  size_t tokens, uint32_t window, float scale,
                                  const uint32_t *d_counts, const float *d_q,
                                  size_t q_token_stride, size_t q_head_stride, float *d_out,
                                  float *d_weights, size_t weights_stride, void *d_workspace,
                                  size_t workspace_bytes) {
  AttentionArgs a{};
  int rc = check_cache(cache, &a.cache);
  if (rc) return rc;
  if ((rc = check_step(a.cache, tokens, SI_HIP_MAX_STEP_TOKENS, "attention")) != 0) return rc;
  if ((rc = check_heads(a.cache, heads)) != 0) return rc;
  if ((rc = check_strides(q_token_stride, q_head_stride, heads, a.cache.head_dim, "query")) != 0)
    return rc;
  if (!std::isfinite(scale))
    return set_error(SI_HIP_ERR_DIMENSIONS, "attention scale is not finite");
  if (d_weights && (rc = check_scores(a.cache, heads, tokens)) != 0) return rc;
  if (d_weights && weights_stride < a.cache.capacity)
    return set_error(SI_HIP_ERR_DIMENSIONS, "attention weights are shorter than the capacity");
  if (workspace_bytes < attention_workspace_bytes(a.cache, (uint32_t)heads, (uint32_t)tokens,
                                                  d_weights != nullptr))
    return set_error(SI_HIP_ERR_BYTE_LENGTH, "attention workspace is too small");
  if (!ctx || !d_q || !d_out || !d_workspace)
    return set_error(SI_HIP_ERR_NULL, "device attention argument is null");
  if ((rc = check_cache_buffers(a.cache)) != 0) return rc;
  if ((uintptr_t)d_workspace % 16 != 0)
    return set_error(SI_HIP_ERR_RANGE, "attention workspace is not 16-byte aligned");
  a.heads = (uint32_t)heads;
  a.group = (uint32_t)heads / a.cache.kv_heads;
  a.tokens = (uint32_t)tokens;
  a.window = window;
  a.scale = scale;
  a.counts = d_counts;
  a.q = d_q;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.out = d_out;
  a.weights = d_weights;
  a.weights_stride = weights_stride;
  a.workspace = d_workspace;
  return submit(ctx, "attention launch", [&](const Workspace &ws, hipStream_t s, bool tuned) {
    a.report = ws.ptr;
    return launch_attention(a, tuned, s);
  });
}

int si_hip_kv_evict_device(si_hip_context *ctx, const si_hip_kv_cache *from,
                           const float *d_weights, size_t weights_stride, size_t keep,
                           size_t sinks, size_t recent, const si_hip_kv_cache *to,
                           float *d_to_weights, size_t to_weights_stride, uint32_t *d_kept) {
  EvictArgs a{};
  int rc = check_cache(from, &a.from);
  if (rc) return rc;
  if ((rc = check_cache(to, &a.to)) != 0) return rc;
  if (a.from.type != a.to.type || a.from.kv_heads != a.to.kv_heads ||
      a.from.head_dim != a.to.head_dim || a.from.sequences != a.to.sequences)
    return set_error(SI_HIP_ERR_DIMENSIONS, "eviction between caches of different shapes");
  if (keep == 0 || keep > a.to.capacity || sinks > keep || recent > keep - sinks ||
      weights_stride < a.from.capacity || to_weights_stride < keep)
    return set_error(SI_HIP_ERR_DIMENSIONS, "eviction dimensions are invalid");
  if (!ctx || !d_weights || !d_to_weights || !d_kept)
    return set_error(SI_HIP_ERR_NULL, "device eviction argument is null");
  if ((rc = check_cache_buffers(a.from)) != 0 || (rc = check_cache_buffers(a.to)) != 0) return rc;
  if (a.from.table == a.to.table || a.from.lengths == a.to.lengths || d_weights == d_to_weights)
    return set_error(SI_HIP_ERR_RANGE, "eviction writes what it reads");
  a.weights = d_weights;
  a.to_weights = d_to_weights;
  a.weights_stride = weights_stride;
  a.to_weights_stride = to_weights_stride;
  a.keep = (uint32_t)keep;
  a.sinks = (uint32_t)sinks;
  a.recent = (uint32_t)recent;
  a.kept = d_kept;
  return submit(ctx, "eviction launch", [&](const Workspace &ws, hipStream_t s, bool) {
    a.report = ws.ptr;
    return launch_evict(a, s);
  });
}

int si_hip_softmax_device(si_hip_context *ctx, const float *d_x, size_t rows, size_t cols,
                          float temperature, float *d_y) {
  size_t n;
  if (!product(rows, cols, &n) || cols > 0x7fffffffu || n > SIZE_MAX / 16)
    return set_error(SI_HIP_ERR_OVERFLOW, "softmax dimensions exceed HIP limits");
  if (n == 0) return set_error(SI_HIP_ERR_DIMENSIONS, "softmax dimensions are invalid");
  if (!std::isfinite(temperature) || temperature < 1e-30f)
    return set_error(SI_HIP_ERR_RANGE, "softmax temperature is invalid");
  if (!ctx || !d_x || !d_y) return set_error(SI_HIP_ERR_NULL, "device softmax argument is null");
  return submit(ctx, "softmax launch", [&](const Workspace &ws, hipStream_t s, bool) {
    return launch_softmax(d_x, d_y, rows, cols, temperature, ws, s);
  });
}

int si_hip_verify_draft_device(si_hip_context *ctx, const float *d_target, const float *d_draft,
                               const uint32_t *d_tokens, const uint32_t *d_counts,
                               const float *d_uniform, size_t sequences, size_t drafts,
                               size_t vocab, uint32_t *d_accepted, uint32_t *d_out_tokens) {
  if (sequences == 0 || vocab == 0)
    return set_error(SI_HIP_ERR_DIMENSIONS, "draft verification dimensions are invalid");
  if (drafts == 0 || drafts > SI_HIP_MAX_STEP_TOKENS)
    return set_error(SI_HIP_ERR_BATCH, "draft verification takes 1..%u drafts a sequence",
                     SI_HIP_MAX_STEP_TOKENS);
  if (sequences > 0x7fffffffu || vocab > 0x7ffff000u)
    return set_error(SI_HIP_ERR_OVERFLOW, "draft verification dimensions exceed HIP limits");
  if (!ctx || !d_target || !d_tokens || !d_uniform || !d_accepted || !d_out_tokens)
    return set_error(SI_HIP_ERR_NULL, "device draft verification argument is null");
  const VerifyArgs a{d_target, d_draft,           d_uniform,        d_tokens,        d_counts,
                     (uint32_t)sequences, (uint32_t)drafts, (uint32_t)vocab, d_accepted,
                     d_out_tokens};
  return submit(ctx, "draft verification launch", [&](const Workspace &ws, hipStream_t s, bool) {
    return launch_verify(a, ws, s);
  });
}

}  // extern "C"
