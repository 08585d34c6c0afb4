// Internal interface of the decode-step operators (include/si_hip_decode.h):
// what api_decode.cpp hands to the kernels, and the cache's addressing.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stddef.h>
#include <stdint.h>

#include "si_hip_internal.h"

namespace sihip {

enum KvType : uint32_t { kKvF32 = 0, kKvF16 = 1, kKvBF16 = 30 };  // ggml type ids
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint32_t kMaxHeadDim = 256;  // SI_HIP_MAX_HEAD_DIM

// Sixteen and eight bytes of memory that is aligned to four: the card's wide
// accesses need no more.
typedef float Floats4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Words2 __attribute__((ext_vector_type(2), aligned(4)));
inline bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0u; }

// A si_hip_kv_cache as the kernels take it.  Rows (one head's values of one
// slot) are numbered through the pool: (page * kv_heads + head) * page_tokens +
// the slot's place in its page; the host has checked that the numbers fit
// 32 bits and the capacity 31.
struct CacheView {
  uint32_t type, kv_heads, head_dim, page_tokens, pages, sequences, max_pages, capacity;
  uint32_t div_mul, div_shift;  // slot / page_tokens = slot * div_mul >> (31 + div_shift)
  void* keys;
  void* values;
  const uint32_t* table;
  uint32_t* lengths;
};

// floor(n / d) for n < 2^31 by one multiplication: with 2^s >= d > 2^(s-1) and
// m = floor(2^(31+s) / d) + 1, n m / 2^(31+s) exceeds n / d by at most
// n / 2^(31+s) < 1 / d.
inline void division_by(uint32_t d, uint32_t* mul, uint32_t* shift) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  *mul = (uint32_t)((uint64_t(1) << (31u + s)) / d + 1u);
  *shift = s;
}
__host__ __device__ __forceinline__ uint32_t divided(uint32_t n, uint32_t mul, uint32_t shift) {
  return (uint32_t)(((uint64_t)n * mul) >> (31u + shift));
}

struct Divisor {
  uint32_t mul, shift;
  __host__ __device__ __forceinline__ uint32_t of(uint32_t n) const { return divided(n, mul, shift); }
};
inline Divisor divisor_of(uint32_t d) {
  Divisor r;
  division_by(d, &r.mul, &r.shift);
  return r;
}

// The row of head `head` in slot `slot` of sequence `seq`; kNone where the
// slot's page lies beyond the pool.  slot < capacity.
__device__ __forceinline__ uint32_t cache_row(const CacheView& c, uint32_t seq, uint32_t head,
                                              uint32_t slot) {
  const uint32_t at = divided(slot, c.div_mul, c.div_shift);
  const uint32_t page = c.table[(size_t)seq * c.max_pages + at];
  if (page >= c.pages) return kNone;
  return (page * c.kv_heads + head) * c.page_tokens + (slot - at * c.page_tokens);
}

// The tokens that sequence `seq` holds and those it brings, cut to its capacity.
__device__ __forceinline__ uint32_t held(const CacheView& c, uint32_t seq) {
  return min(c.lengths[seq], c.capacity);
}
__device__ __forceinline__ uint32_t brought(const uint32_t* counts, uint32_t seq, uint32_t tokens) {
  return counts ? min(counts[seq], tokens) : tokens;
}

struct RopeArgs {
  uint32_t layout, rotary_dim;
  float magnitude;
  const uint64_t* frequencies;
};

// Rows of heads to rotate: head h of row t is at x + t * token_stride + h * head_stride.
struct RopeRows {
  const float* x;
  float* y;
  size_t token_stride, head_stride, y_token_stride, y_head_stride;
  uint32_t heads;
};

// kernels_rope.hip
hipError_t launch_rope(const RopeArgs& rope, const RopeRows& rows, uint32_t tokens,
                       uint32_t head_dim, const uint32_t* positions, hipStream_t s);
// `rope` null: the keys are stored as they are; `q` null: no query rows.
hipError_t launch_rope_append(const CacheView& cache, const RopeArgs* rope, uint32_t tokens,
                              const uint32_t* counts, const uint32_t* positions, const float* k,
                              size_t k_stride, const float* v, size_t v_stride, const RopeRows* q,
                              void* ws, hipStream_t s);
hipError_t launch_kv_advance(const CacheView& cache, const uint32_t* counts, uint32_t more,
                             hipStream_t s);

// kernels_norm_rope.hip
struct NormArgs {
  float eps, shift;            // y = x * inv * (shift + w)
  const float *q, *k;          // null: y = x * inv
  bool on;                     // false: no norm
};
struct AxesArgs {
  uint32_t axes;
  const uint8_t* axis;         // of each pair; null: all on axis 0
};
hipError_t launch_norm_rope(const NormArgs& norm, const RopeArgs& rope, const AxesArgs& axes,
                            const RopeRows& rows, uint32_t tokens, uint32_t head_dim,
                            const uint32_t* positions, void* ws, hipStream_t s);
// rope.rotary_dim 0: no rotation
hipError_t launch_norm_rope_append(const CacheView& cache, const NormArgs& norm,
                                   const RopeArgs& rope, const AxesArgs& axes, uint32_t tokens,
                                   const uint32_t* counts, const uint32_t* positions,
                                   const float* k, size_t k_stride, const float* v,
                                   size_t v_stride, const RopeRows* q, void* ws, hipStream_t s);

// kernels_attention.hip
struct AttentionArgs {
  CacheView cache;
  uint32_t heads, group, tokens, window;  // group = heads / kv_heads
  float scale;
  const uint32_t* counts;
  const float* q;
  size_t q_token_stride, q_head_stride;
  float* out;
  float* weights;
  size_t weights_stride;
  void* workspace;
  void* report;  // the context's workspace: device errors
};
size_t attention_workspace_bytes(const CacheView& cache, uint32_t heads, uint32_t tokens,
                                 bool weights);
hipError_t launch_attention(const AttentionArgs& a, bool tuned, hipStream_t s);

// kernels_evict.hip
struct EvictArgs {
  CacheView from, to;
  const float* weights;
  float* to_weights;
  size_t weights_stride, to_weights_stride;
  uint32_t keep, sinks, recent;
  uint32_t* kept;
  void* report;
};
hipError_t launch_evict(const EvictArgs& a, hipStream_t s);

// kernels_sampling.hip
hipError_t launch_softmax(const float* x, float* y, size_t rows, size_t cols, float temperature,
                          const Workspace& ws, hipStream_t s);
struct VerifyArgs {
  const float *target, *draft, *uniform;
  const uint32_t *tokens, *counts;
  uint32_t sequences, drafts, vocab;
  uint32_t *accepted, *out_tokens;
};
hipError_t launch_verify(const VerifyArgs& a, const Workspace& ws, hipStream_t s);

}  // namespace sihip
