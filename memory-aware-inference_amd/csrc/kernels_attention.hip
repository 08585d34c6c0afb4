// Attention of a sequence's new tokens over its paged cache.
//
// out = sum_i p_i v_i, p_i = exp(scale q.k_i - m) / l, over the slots a row
// sees; m and l run along with the slots, and every sum is held in 32 bits.
// Scores are taken times log2(e), so that p is an exp2.
//
// Rows of one kv head: row r = t * group + g is token t's query head
// kv_head * group + g.
#include "attention_common.h"

namespace sihip {
using namespace attn;

namespace {

constexpr uint32_t kThreads = 256;

template <typename T>
__device__ __forceinline__ float value_of(T v);
template <>
__device__ __forceinline__ float value_of<float>(float v) { return v; }
template <>
__device__ __forceinline__ float value_of<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float value_of<__hip_bfloat16>(__hip_bfloat16 v) {
  return __bfloat162float(v);
}

template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* part) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float w = __shfl_xor(v, o, 64);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  __syncthreads();
  if ((threadIdx.x & 63u) == 0u) part[threadIdx.x / 64u] = v;
  __syncthreads();
  float r = part[0];
#pragma unroll
  for (uint32_t i = 1; i < kThreads / 64u; ++i) r = MAX ? fmaxf(r, part[i]) : r + part[i];
  return r;
}

// ---- one workgroup a row, any head size and alignment --------------------------
// grid (heads, tokens, sequences).  A thread takes a slot's score, then a
// value of the head's output.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_generic(AttentionArgs a, float2* stats,
                                                              float* scores,
                                                              uint32_t score_stride) {
  __shared__ float q[kMaxHeadDim], p[kThreads], part[kThreads / 64];
  __shared__ uint32_t row[kThreads];
  const CacheView& c = a.cache;
  const uint32_t h = blockIdx.x, t = blockIdx.y, s = blockIdx.z, dim = c.head_dim;
  const uint32_t kv = h / a.group, i = threadIdx.x;
  float* out = a.out + (((size_t)s * a.tokens + t) * a.heads + h) * dim;
  const uint32_t rows = a.tokens * a.group, r = t * a.group + (h - kv * a.group);
  const size_t at = ((size_t)s * c.kv_heads + kv) * rows + r;
  float* score = scores ? scores + at * score_stride : nullptr;
  const uint32_t count = brought(a.counts, s, a.tokens);
  if (t >= count) {
    if (i < dim) out[i] = 0.0f;
    if (stats && i == 0u) stats[at] = make_float2(0.0f, 0.0f);
    return;
  }
  if (t == 0u && h == 0u && i == 0u &&
      (uint64_t)c.lengths[s] + count > c.capacity)
    report_device_error(a.report, kDevErrCacheFull);
  uint32_t begin, end;
  seen_slots(held(c, s), t, c.capacity, a.window, begin, end);
  const float scale = a.scale * kLog2e;
  if (i < dim)
    q[i] = a.q[((size_t)s * a.tokens + t) * a.q_token_stride + h * a.q_head_stride + i] * scale;
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  bool any = false, bad = false;
  for (uint32_t base = begin; base < end; base += kThreads) {
    const uint32_t slot = base + i;
    uint32_t at_row = kNone;
    if (slot < end) {
      at_row = cache_row(c, s, kv, slot);
      bad |= at_row == kNone;
    }
    __syncthreads();  // the values of the last tile are taken, and q is there
    row[i] = at_row;
    float v = -INFINITY;
    if (at_row != kNone) {
      const T* key = static_cast<const T*>(c.keys) + (size_t)at_row * dim;
      v = 0.0f;
      for (uint32_t d = 0; d < dim; ++d) v = fmaf(q[d], value_of<T>(key[d]), v);
    }
    if (score && slot < end) score[slot] = v;
    any |= __syncthreads_or(at_row != kNone) != 0;
    const float top = fmaxf(m, block_reduce<true>(v, part));
    const float from = top == -INFINITY ? 0.0f : top;
    const float e = at_row != kNone ? exp2f(v - from) : 0.0f;
    const float keep = exp2f(m - from);
    p[i] = e;
    l = l * keep + block_reduce<false>(e, part);  // (its barriers publish p and row)
    m = top;
    acc *= keep;
    if (i < dim)
      for (uint32_t j = 0; j < min(kThreads, end - base); ++j)
        if (row[j] != kNone)
          acc = fmaf(p[j], value_of<T>(static_cast<const T*>(c.values)[(size_t)row[j] * dim + i]),
                     acc);
  }
  if (bad) report_device_error(a.report, kDevErrCachePage);
  if (i < dim) out[i] = any ? acc / l : 0.0f;
  if (stats && i == 0u)
    stats[at] = any ? make_float2(m == -INFINITY ? 0.0f : m, 1.0f / l) : make_float2(0.0f, 0.0f);
}

// weights[slot] += sum over the kv head's rows of exp2(score - m) / l.  grid
// (blocks of 256 / PARTS slots, from `first_block` on, kv_heads, sequences): the
// waves of a workgroup add up 1 / PARTS of the rows each, in their order, kAhead
// rows' loads under way at once; the parts are added in theirs.  Up to eight rows are one part, more
// four (24 sequences of 2000 slots, four rows a head: with the attention 96.4
// us in one part, 106.3 in four; 25 of 65 slots, 112 rows: 47.9 and 39.1, 72.1
// row by row).
constexpr uint32_t kFewRows = 8;
template <uint32_t PARTS>
__global__ __launch_bounds__(kThreads) void attention_weights(AttentionArgs a, const float2* stats,
                                                              const float* scores,
                                                              uint32_t score_stride,
                                                              uint32_t first_block) {
  constexpr uint32_t kSlots = kThreads / PARTS, kAhead = PARTS == 1 ? 4 : 8;
  __shared__ float sums[PARTS][kSlots];
  const CacheView& c = a.cache;
  const uint32_t lane = threadIdx.x % kSlots, part = uniform(threadIdx.x / kSlots);
  const uint32_t slot0 = (first_block + blockIdx.x) * kSlots, slot = slot0 + lane;
  const uint32_t kv = blockIdx.y, s = blockIdx.z;
  const uint32_t count = brought(a.counts, s, a.tokens), length = held(c, s);
  const uint32_t rows = a.tokens * a.group, used = count * a.group;
  const uint32_t slots = min(length + count, c.capacity);
  if (count == 0u || slot0 >= slots) return;
  const size_t at = ((size_t)s * c.kv_heads + kv) * rows;
  const uint32_t each = (used + PARTS - 1u) / PARTS;
  const uint32_t first = min(part * each, used), last = min(first + each, used);
  const uint32_t from = min(slot, slots - 1u);
  float sum = 0.0f;
  uint32_t t = first / a.group, g = first - t * a.group;
  for (uint32_t r0 = first; r0 < last; r0 += kAhead) {
    // (what a row did not see is there to be read, and is left out)
    float2 st[kAhead];
    float score[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      const size_t r = at + min(r0 + k, last - 1u);
      st[k] = stats[r];
      score[k] = scores[r * score_stride + from];
    }
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      uint32_t begin, end;
      seen_slots(length, t, c.capacity, a.window, begin, end);
      if (r0 + k < last && slot >= begin && slot < end && st[k].y != 0.0f)
        sum += exp2f(score[k] - st[k].x) * st[k].y;
      if (++g == a.group) {
        g = 0u;
        ++t;
      }
    }
  }
  if constexpr (PARTS > 1) {
    sums[part][lane] = sum;
    __syncthreads();
  }
  if (part != 0u || slot >= slots) return;
#pragma unroll
  for (uint32_t i = 1; i < PARTS; ++i) sum += sums[i][lane];
  a.weights[((size_t)s * c.kv_heads + kv) * a.weights_stride + slot] += sum;
}

// (A launch takes less than 2^32 threads in x, and runs fewer than it was asked for, without an
// error, from there on.)
template <uint32_t PARTS>
hipError_t launch_weights(const AttentionArgs& a, const float2* stats, const float* scores,
                          uint32_t score_stride, hipStream_t s) {
  constexpr uint32_t kSlots = kThreads / PARTS, kMost = 0xffffffffu / kThreads;
  const CacheView& c = a.cache;
  const uint32_t blocks = (c.capacity + kSlots - 1u) / kSlots;
  for (uint32_t b = 0; b < blocks; b += std::min(kMost, blocks - b)) {
    attention_weights<PARTS>
        <<<dim3(std::min(kMost, blocks - b), c.kv_heads, c.sequences), kThreads, 0, s>>>(
            a, stats, scores, score_stride, b);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

size_t attention_workspace_bytes(const CacheView& cache, uint32_t heads, uint32_t tokens,
                                 bool weights) {
  return space_of(cache, heads, tokens, weights).bytes;
}

hipError_t launch_attention(const AttentionArgs& a, bool tuned, hipStream_t s) {
  const CacheView& c = a.cache;
  const Space sp = space_of(c, a.heads, a.tokens, a.weights != nullptr);
  uint8_t* w = static_cast<uint8_t*>(a.workspace);
  float2* stats = a.weights ? reinterpret_cast<float2*>(w + sp.stats) : nullptr;
  float* scores = a.weights ? reinterpret_cast<float*>(w + sp.scores) : nullptr;
  bool taken = false;
  hipError_t e = hipSuccess;
  if (tuned) e = launch_attention_mfma(a, sp, &taken, s);
  if (e != hipSuccess) return e;
  if (!taken) {
    const dim3 grid(a.heads, a.tokens, c.sequences);
    if (c.type == kKvF32)
      attention_generic<float><<<grid, kThreads, 0, s>>>(a, stats, scores, sp.score_stride);
    else if (c.type == kKvF16)
      attention_generic<__half><<<grid, kThreads, 0, s>>>(a, stats, scores, sp.score_stride);
    else
      attention_generic<__hip_bfloat16><<<grid, kThreads, 0, s>>>(a, stats, scores,
                                                                  sp.score_stride);
    e = hipGetLastError();
  }
  if (e != hipSuccess || !a.weights) return e;
  if (a.tokens * a.group <= kFewRows) return launch_weights<1>(a, stats, scores, sp.score_stride, s);
  return launch_weights<4>(a, stats, scores, sp.score_stride, s);
}

}  // namespace sihip
