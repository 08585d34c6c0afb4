// Probabilities from logits, and the verification of drafted tokens.
#include "decode_internal.h"

namespace sihip {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kEach = 16;                 // values a thread
constexpr uint32_t kChunk = kThreads * kEach;  // values a workgroup
constexpr float kLog2e = 1.4426950408889634f;

// ---- softmax ------------------------------------------------------------------
// y = exp((x - m) / T) / l: a workgroup a chunk of a row, once for the chunk's
// maximum and sum (scratch), once, with the row's from all of them, for y.

// (maximum, sum of exp2((x - maximum) per)) of two parts of a row; `per` is
// log2(e) / T.  The difference is taken first, so its rounding is that of a
// small number where the value is a large one.
__device__ __forceinline__ float2 joined(float2 a, float2 b, float per) {
  const float m = fmaxf(a.x, b.x), from = m == -INFINITY ? 0.0f : m;
  return make_float2(m, a.y * exp2f((a.x - from) * per) + b.y * exp2f((b.x - from) * per));
}
__device__ __forceinline__ float2 block_joined(float2 v, float per, float2* part) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v = joined(v, make_float2(__shfl_xor(v.x, o, 64), __shfl_xor(v.y, o, 64)), per);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0u) part[threadIdx.x / 64u] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (uint32_t i = 1; i < kWaves; ++i) v = joined(v, part[i], per);
  return v;
}

// grid (chunks, rows)
__global__ __launch_bounds__(kThreads) void softmax_stats(const float* __restrict__ x, size_t cols,
                                                          float per, float2* stats) {
  __shared__ float2 part[kWaves];
  const float* row = x + blockIdx.y * cols;
  const size_t base = (size_t)blockIdx.x * kChunk;
  float v[kEach], m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const size_t c = base + i * kThreads + threadIdx.x;
    v[i] = c < cols ? row[c] : -INFINITY;
    m = fmaxf(m, v[i]);
  }
  const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) sum += exp2f((v[i] - from) * per);
  const float2 r = block_joined(make_float2(m, sum), per, part);
  if (threadIdx.x == 0u) stats[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = r;
}
__global__ __launch_bounds__(kThreads) void softmax_values(const float* x, size_t cols, float per,
                                                           const float2* stats, float* y) {
  __shared__ float2 part[kWaves];
  const float2* st = stats + (size_t)blockIdx.y * gridDim.x;
  float2 r = make_float2(-INFINITY, 0.0f);
  for (uint32_t i = threadIdx.x; i < gridDim.x; i += kThreads) r = joined(r, st[i], per);
  r = block_joined(r, per, part);
  const float from = r.x == -INFINITY ? 0.0f : r.x, scale = 1.0f / r.y;
  const size_t row = blockIdx.y * cols, base = (size_t)blockIdx.x * kChunk;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const size_t c = base + i * kThreads + threadIdx.x;
    if (c < cols) y[row + c] = exp2f((x[row + c] - from) * per) * scale;
  }
}

// ---- verification ---------------------------------------------------------------
// Terms in 2^-36 fixed point: their sums are exact in any order, so the
// workgroups' shares of a row add up to what one pass over it would give.

// floor(clamp(x, 0, 1) 2^36); a NaN is 0.  The 24-bit significand, moved.
__device__ __forceinline__ uint64_t fixed(float x) {
  if (!(x > 0.0f)) return 0u;
  const uint32_t b = __float_as_uint(fminf(x, 1.0f));
  const uint32_t e = b >> 23;  // x = (b & mask | 2^23) 2^(e - 150)
  const uint64_t m = (b & 0x7fffffu) | 0x800000u;
  return e >= 114u ? m << (e - 114u) : e > 90u ? m >> (114u - e) : 0u;
}

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* part) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0u) part[threadIdx.x / 64u] = v;
  __syncthreads();
  v = 0u;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) v += part[i];
  return v;
}

// Where a sequence's drafts end: how many are accepted, of how many.
struct Ends {
  uint32_t accepted, count;
  bool beyond;  // the refused token lies beyond the vocabulary
};
__device__ __forceinline__ Ends ends_of(const VerifyArgs& a, uint32_t s, uint32_t* shared) {
  if (threadIdx.x < 64u) {
    const uint32_t i = threadIdx.x, count = brought(a.counts, s, a.drafts);
    bool accept = false, beyond = false;
    if (i < count) {
      const uint32_t token = a.tokens[(size_t)s * a.drafts + i];
      beyond = token >= a.vocab;
      if (!beyond) {
        const float p = a.target[((size_t)s * (a.drafts + 1u) + i) * a.vocab + token];
        const float q = a.draft ? a.draft[((size_t)s * a.drafts + i) * a.vocab + token] : 1.0f;
        accept = a.uniform[(size_t)s * (a.drafts + 1u) + i] * q < p;
      }
    }
    const uint64_t refused = ~__builtin_amdgcn_ballot_w64(accept);
    const uint64_t off = __builtin_amdgcn_ballot_w64(beyond);
    const uint32_t n = (uint32_t)__builtin_ctzll(refused);  // at most 16
    if (i == 0u) {
      shared[0] = n;
      shared[1] = count;
      shared[2] = n < count ? (uint32_t)(off >> n) & 1u : 0u;
    }
  }
  __syncthreads();
  return {shared[0], shared[1], shared[2] != 0u};
}

// The rows that the next token is drawn from: p, and q where one is taken away.
struct Rows {
  const float *p, *q;
  uint32_t certain;  // the token whose q is 1 (kNone: none)
};
__device__ __forceinline__ Rows rows_of(const VerifyArgs& a, uint32_t s, const Ends& e) {
  Rows r{a.target + ((size_t)s * (a.drafts + 1u) + e.accepted) * a.vocab, nullptr, kNone};
  if (e.accepted < e.count) {
    if (a.draft) r.q = a.draft + ((size_t)s * a.drafts + e.accepted) * a.vocab;
    else r.certain = a.tokens[(size_t)s * a.drafts + e.accepted];
  }
  return r;
}
__device__ __forceinline__ uint64_t rest_of(const Rows& r, uint32_t v, float p) {
  if (r.q) return fixed(p - r.q[v]);
  return fixed(v == r.certain ? p - 1.0f : p);
}

// grid (chunks, sequences): the chunk's sums of max(p - q, 0) and of p
__global__ __launch_bounds__(kThreads) void verify_sums(VerifyArgs a, ulonglong2* sums) {
  __shared__ uint32_t shared[3];
  __shared__ uint64_t part[kWaves];
  const uint32_t s = blockIdx.y, base = blockIdx.x * kChunk;
  const Ends e = ends_of(a, s, shared);
  const Rows r = rows_of(a, s, e);
  uint64_t rest = 0u, all = 0u;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint32_t v = base + i * kThreads + threadIdx.x;
    if (v < a.vocab) {
      const float p = r.p[v];
      rest += rest_of(r, v, p);
      all += fixed(p);
    }
  }
  rest = block_sum(rest, part);
  all = block_sum(all, part);
  if (threadIdx.x == 0u)
    sums[(size_t)s * gridDim.x + blockIdx.x] = make_ulonglong2(rest, all);
}

// grid (sequences): the token whose running sum first exceeds the threshold
__global__ __launch_bounds__(kThreads) void verify_draw(VerifyArgs a, const ulonglong2* sums,
                                                        uint32_t chunks, void* ws) {
  __shared__ uint32_t shared[3], at;
  __shared__ uint64_t part[kWaves], left;
  const uint32_t s = blockIdx.x, tid = threadIdx.x;
  const Ends e = ends_of(a, s, shared);
  Rows r = rows_of(a, s, e);
  sums += (size_t)s * chunks;
  uint64_t rest = 0u, all = 0u;
  for (uint32_t i = tid; i < chunks; i += kThreads) {
    rest += sums[i].x;
    all += sums[i].y;
  }
  rest = block_sum(rest, part);
  all = block_sum(all, part);
  const bool whole = rest == 0u;  // p itself (the same sums where nothing was taken away)
  if (whole) r.q = nullptr, r.certain = kNone;
  const uint64_t total = whole ? all : rest;
  const float u = a.uniform[(size_t)s * (a.drafts + 1u) + a.drafts];
  const uint32_t n24 = u > 0.0f ? (uint32_t)fminf(u * 0x1p24f, 16777215.0f) : 0u;
  const uint64_t lo = total * n24, hi = __umul64hi(total, n24);
  const uint64_t threshold = hi << 40 | lo >> 24;
  // the chunk: sums up to it, one after another
  if (tid == 0u) {
    uint64_t before = 0u;
    uint32_t c = 0u;
    if (total != 0u)
      for (;; ++c) {
        const uint64_t one = whole ? sums[c].y : sums[c].x;
        if (before + one > threshold) break;
        before += one;
      }
    at = c;
    left = threshold - before;
  }
  __syncthreads();
  // its values: a thread's are next to each other
  const uint32_t first = at * kChunk + tid * kEach;
  uint64_t mine = 0u;
  for (uint32_t i = 0; i < kEach; ++i)
    if (first + i < a.vocab) mine += rest_of(r, first + i, r.p[first + i]);
  uint64_t upto = mine;
  const uint32_t lane = tid & 63u, wave = tid / 64u;
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) {
    const uint64_t y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  __syncthreads();
  if (lane == 63u) part[wave] = upto;
  __syncthreads();
  for (uint32_t i = 0; i < wave; ++i) upto += part[i];
  uint32_t* out = a.out_tokens + (size_t)s * (a.drafts + 1u);
  if (total != 0u && upto > left && upto - mine <= left) {
    uint64_t before = upto - mine;
    uint32_t v = first;
    for (;; ++v) {
      before += rest_of(r, v, r.p[v]);
      if (before > left) break;
    }
    out[e.accepted] = v;
  }
  if (tid == 0u) {
    a.accepted[s] = e.accepted;
    if (total == 0u) {
      out[e.accepted] = kNone;
      report_device_error(ws, kDevErrNoMass);
    }
    if (e.beyond) report_device_error(ws, kDevErrDraftToken);
  }
  if (tid <= a.drafts && tid != e.accepted)
    out[tid] = tid < e.accepted ? a.tokens[(size_t)s * a.drafts + tid] : kNone;
}

}  // namespace

hipError_t launch_softmax(const float* x, float* y, size_t rows, size_t cols, float temperature,
                          const Workspace& ws, hipStream_t s) {
  const uint32_t chunks = (uint32_t)((cols + kChunk - 1u) / kChunk);
  const size_t most = std::min<size_t>(ws.scratch_bytes / sizeof(float2) / chunks, 65535u);
  const float per = kLog2e / temperature;
  float2* stats = reinterpret_cast<float2*>(ws.scratch);
  for (size_t r = 0; r < rows; r += most) {
    const dim3 grid(chunks, (uint32_t)std::min(most, rows - r));
    softmax_stats<<<grid, kThreads, 0, s>>>(x + r * cols, cols, per, stats);
    softmax_values<<<grid, kThreads, 0, s>>>(x + r * cols, cols, per, stats, y + r * cols);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_verify(const VerifyArgs& a, const Workspace& ws, hipStream_t s) {
  const uint32_t chunks = (a.vocab + kChunk - 1u) / kChunk;
  ulonglong2* sums = reinterpret_cast<ulonglong2*>(ws.scratch);
  const uint32_t most = (uint32_t)std::min<size_t>(ws.scratch_bytes / sizeof(ulonglong2) / chunks, 65535u);
  for (uint32_t n = 0; n < a.sequences; n += most) {
    VerifyArgs b = a;
    b.sequences = std::min(most, a.sequences - n);
    b.target += (size_t)n * (a.drafts + 1u) * a.vocab;
    if (b.draft) b.draft += (size_t)n * a.drafts * a.vocab;
    b.tokens += (size_t)n * a.drafts;
    if (b.counts) b.counts += n;
    b.uniform += (size_t)n * (a.drafts + 1u);
    b.accepted += n;
    b.out_tokens += (size_t)n * (a.drafts + 1u);
    verify_sums<<<dim3(chunks, b.sequences), kThreads, 0, s>>>(b, sums);
    verify_draw<<<b.sequences, kThreads, 0, s>>>(b, sums, chunks, ws.ptr);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace sihip
