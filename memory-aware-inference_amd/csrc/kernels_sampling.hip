// Probabilities from logits, and the verification of drafted tokens.
#include "decode_internal.h"

namespace sihip {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;

// Rows of an odd number of values are read and written four values at once too (288 rows of
// 151,936 logits, moved by four bytes: 134 us value by value, 83 so; 81 where they begin on
// sixteen bytes).

// Whether a row ends inside four values of the chunk of `fours` a thread from `base` on.
__device__ __forceinline__ bool ends_inside(size_t base, size_t cols, uint32_t fours) {
  return cols % 4u != 0u && base + 4u * fours * kThreads > cols;
}

// Values [base + 4 (j kThreads + thread), + 4), j < FOURS, of a row of `cols`;
// `rest` where there is none.  LAST: nothing reads them again, so they pass the caches by (288
// rows 81.4 us so, 85 without).
template <bool LAST, uint32_t FOURS>
__device__ __forceinline__ void load_fours(const float* row, size_t base, size_t cols, float rest,
                                           float4 (&v)[FOURS]) {
#pragma unroll
  for (uint32_t j = 0; j < FOURS; ++j) {
    const size_t c = base + 4u * (j * kThreads + threadIdx.x);
    Floats4 f{rest, rest, rest, rest};
    if (c + 3u < cols) {
      const Floats4* from = reinterpret_cast<const Floats4*>(row + c);
      f = LAST ? __builtin_nontemporal_load(from) : *from;
    }
    v[j] = make_float4(f.x, f.y, f.z, f.w);
  }
  if (!ends_inside(base, cols, FOURS)) return;
#pragma unroll
  for (uint32_t j = 0; j < FOURS; ++j) {
    const size_t c = base + 4u * (j * kThreads + threadIdx.x);
    if (c + 3u < cols) continue;
    if (c < cols) v[j].x = row[c];
    if (c + 1u < cols) v[j].y = row[c + 1u];
    if (c + 2u < cols) v[j].z = row[c + 2u];
  }
}

// ---- softmax ------------------------------------------------------------------
// y = exp((x - m) / T) / l: a workgroup a chunk of a row, once for the chunk's
// maximum and sum (scratch), once, with the row's from all of them, for y.  288
// rows of 151,936 logits: 81 us, 31 and 50, for 350 MB read, read again (half
// of it from the caches) and written, 4.3 TB/s of what has to move once; 5 rows
// 7.6 us, two launches of little more than an empty one.

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

// grid (chunks, rows): a chunk is 4 FOURS values a thread
template <uint32_t FOURS>
__global__ __launch_bounds__(kThreads) void softmax_stats(const float* __restrict__ x, size_t cols,
                                                          float per, float2* stats) {
  __shared__ float2 part[kWaves];
  float4 v[FOURS];
  load_fours<false>(x + blockIdx.y * cols, (size_t)blockIdx.x * 4u * FOURS * kThreads, cols,
                  -INFINITY, v);
  float m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < FOURS; ++j) m = fmaxf(fmaxf(fmaxf(m, v[j].x), fmaxf(v[j].y, v[j].z)), v[j].w);
  const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (uint32_t j = 0; j < FOURS; ++j)
    sum += (exp2f((v[j].x - from) * per) + exp2f((v[j].y - from) * per)) +
           (exp2f((v[j].z - from) * per) + exp2f((v[j].w - from) * per));
  const float2 r = block_joined(make_float2(m, sum), per, part);
  if (threadIdx.x == 0u) stats[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = r;
}
template <uint32_t FOURS>
__global__ __launch_bounds__(kThreads) void softmax_values(const float* x, size_t cols, float per,
                                                           const float2* stats, float* y) {
  __shared__ float2 part[kWaves];
  const size_t base = (size_t)blockIdx.x * 4u * FOURS * kThreads;
  float4 v[FOURS];
  load_fours<true>(x + blockIdx.y * cols, base, cols, 0.0f, v);
  const float2* st = stats + (size_t)blockIdx.y * gridDim.x;
  float2 r = make_float2(-INFINITY, 0.0f);
  for (uint32_t i = threadIdx.x; i < gridDim.x; i += kThreads) r = joined(r, st[i], per);
  r = block_joined(r, per, part);
  const float from = r.x == -INFINITY ? 0.0f : r.x, scale = 1.0f / r.y;
  float* row = y + blockIdx.y * cols;
  Floats4 e[FOURS];
#pragma unroll
  for (uint32_t j = 0; j < FOURS; ++j) {
    const size_t c = base + 4u * (j * kThreads + threadIdx.x);
    e[j] = Floats4{exp2f((v[j].x - from) * per) * scale, exp2f((v[j].y - from) * per) * scale,
                 exp2f((v[j].z - from) * per) * scale, exp2f((v[j].w - from) * per) * scale};
    if (c + 3u < cols) __builtin_nontemporal_store(e[j], reinterpret_cast<Floats4*>(row + c));
  }
  if (!ends_inside(base, cols, FOURS)) return;
#pragma unroll
  for (uint32_t j = 0; j < FOURS; ++j) {
    const size_t c = base + 4u * (j * kThreads + threadIdx.x);
    if (c + 3u < cols) continue;
    if (c < cols) row[c] = e[j].x;
    if (c + 1u < cols) row[c + 1u] = e[j].y;
    if (c + 2u < cols) row[c + 2u] = e[j].z;
  }
}

// ---- verification ---------------------------------------------------------------
// Terms in 2^-36 fixed point: their sums are exact in any order, so the
// workgroups' shares of a row add up to what one pass over it would give.  One
// launch: 32 sequences of up to 8 drafts over 151,936 tokens 20 us for 38.9 MB
// (two rows a sequence); one sequence 6.5 us, the launch, the chain of
// acceptances that leads to the rows, their chunks, and the hand-over to the
// last workgroup.

// floor(clamp(x, 0, 1) 2^36) = high 2^18 + low; a NaN is 0.  x 2^18 less its
// whole part has no more bits than x, so both conversions are exact.  Sums of
// up to 2^13 terms stay within 32 bits in each half.
struct Fixed {
  uint32_t high = 0u, low = 0u;
  __device__ __forceinline__ void add(float x) {
    const float y = fminf(fmaxf(x, 0.0f), 1.0f) * 0x1p18f;
    const uint32_t h = (uint32_t)y;
    high += h;
    low += (uint32_t)((y - (float)h) * 0x1p18f);
  }
  __device__ __forceinline__ uint64_t value() const { return ((uint64_t)high << 18) + low; }
};
__device__ __forceinline__ uint64_t fixed(float x) {
  Fixed f;
  f.add(x);
  return f.value();
}

// A workgroup's sum of its threads' terms, for thread 0.
__device__ __forceinline__ uint64_t block_sum(Fixed v, uint64_t* part) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v.high += __shfl_xor(v.high, o, 64);
    v.low += __shfl_xor(v.low, o, 64);
  }
  if ((threadIdx.x & 63u) == 0u) part[threadIdx.x / 64u] = v.value();
  __syncthreads();
  uint64_t total = 0u;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) total += part[i];
  return total;
}

// Sum of v over the workgroup's threads up to and with this one, and of all.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u;
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) {
    const uint64_t y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 63u) part[wave] = v;
  __syncthreads();
  uint64_t before = 0u;
  total = 0u;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) {
    if (i < wave) before += part[i];
    total += part[i];
  }
  return before + v;
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
// Device-coherent (sc1) accesses: each XCD has its own L2.
__device__ __forceinline__ void store_coherent(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t load_coherent(const uint64_t* p) {
  return __hip_atomic_load(const_cast<uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The values of a row that a workgroup takes: 16 a thread, next to each other.
constexpr uint32_t kEach = 16, kChunk = kThreads * kEach;

__device__ __forceinline__ void load_each(const float* row, uint32_t first, uint32_t vocab,
                                          float (&v)[kEach]) {
#pragma unroll
  for (uint32_t i = 0; i < kEach; i += 4) {
    if (first + i + 3u < vocab) {
      const Floats4 f = *reinterpret_cast<const Floats4*>(row + first + i);
      v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    } else {
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) v[i + k] = first + i + k < vocab ? row[first + i + k] : 0.0f;
    }
  }
}

// grid (chunks, sequences): each workgroup adds up its chunk's max(p - q, 0); the
// one that is done last finds the token whose running sum first exceeds the
// threshold: its chunk from the chunks' sums, then its place in that chunk.
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a, uint64_t* sums,
                                                          uint32_t* counters, void* ws) {
  __shared__ uint32_t shared[3], is_last, at;
  __shared__ uint64_t part[kWaves], left;
  const uint32_t s = blockIdx.y, tid = threadIdx.x, chunks = gridDim.x;
  const Ends e = ends_of(a, s, shared);
  Rows r = rows_of(a, s, e);
  sums += (size_t)s * chunks;
  // the thread's values of a chunk, p or what is left of it
  float v[kEach];
  const auto load = [&](uint32_t chunk) {
    const uint32_t first = chunk * kChunk + tid * kEach;
    load_each(r.p, first, a.vocab, v);
    if (r.q) {
      float q[kEach];
      load_each(r.q, first, a.vocab, q);
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) v[i] -= q[i];
    } else if (r.certain - first < kEach) {
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i)
        if (first + i == r.certain) v[i] -= 1.0f;
    }
  };
  const auto own = [&] {
    Fixed f;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) f.add(v[i]);
    return f;
  };
  load(blockIdx.x);
  const uint64_t sum = block_sum(own(), part);
  if (tid == 0u) {
    // Device-coherent stores, in place before the chunk is counted, and read by loads of
    // the same kind: the sums are known to the last workgroup on whatever XCD without a
    // write-back of its L2.
    store_coherent(sums + blockIdx.x, sum);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    is_last = __hip_atomic_fetch_add(counters + s, 1u, __ATOMIC_RELAXED,
                                     __HIP_MEMORY_SCOPE_AGENT) == chunks - 1u;
    if (is_last)
      __hip_atomic_store(counters + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!is_last) return;
  // the chunks' sums: a thread's are next to each other
  const uint32_t per = (chunks + kThreads - 1u) / kThreads;
  const uint32_t c0 = min(tid * per, chunks), c1 = min(c0 + per, chunks);
  uint64_t mine, upto, total;
  const auto add_chunks = [&] {
    mine = 0u;
    for (uint32_t i = c0; i < c1; ++i) mine += load_coherent(sums + i);
    upto = block_scan(mine, part, total);
  };
  add_chunks();
  if (total == 0u && (r.q || r.certain != kNone)) {
    // nothing is left of p: p itself (rare, so its sums are taken here)
    r.q = nullptr;
    r.certain = kNone;
    for (uint32_t c = 0; c < chunks; ++c) {
      load(c);
      __syncthreads();
      const uint64_t one = block_sum(own(), part);
      if (tid == 0u) store_coherent(sums + c, one);
    }
    if (tid == 0u) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    add_chunks();
  }
  // (u in steps of 2^-24, those that a float has just below 1: the product is an integer's)
  const float u = a.uniform[(size_t)s * (a.drafts + 1u) + a.drafts];
  const uint32_t n24 = u > 0.0f ? (uint32_t)fminf(u * 0x1p24f, 16777215.0f) : 0u;
  const uint64_t threshold = __umul64hi(total, n24) << 40 | (total * n24) >> 24;
  if (total != 0u && upto - mine <= threshold && threshold < upto) {
    uint64_t before = upto - mine;
    uint32_t i = c0;
    for (;; ++i) {
      const uint64_t one = load_coherent(sums + i);
      if (before + one > threshold) break;
      before += one;
    }
    at = i;
    left = threshold - before;
  }
  __syncthreads();
  uint32_t* out = a.out_tokens + (size_t)s * (a.drafts + 1u);
  if (total != 0u) {
    load(at);
    uint64_t whole;
    mine = own().value();
    upto = block_scan(mine, part, whole);
    if (upto - mine <= left && left < upto) {
      uint64_t running = upto - mine;
      uint32_t token = kNone;
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i) {
        running += fixed(v[i]);
        if (token == kNone && running > left) token = at * kChunk + tid * kEach + i;
      }
      out[e.accepted] = token;
    }
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

template <uint32_t FOURS>
hipError_t softmax_rows(const float* x, float* y, size_t rows, size_t cols, float per,
                        const Workspace& ws, hipStream_t s) {
  const uint32_t chunk = 4u * FOURS * kThreads, chunks = (uint32_t)((cols + chunk - 1u) / chunk);
  const size_t most = std::min<size_t>(ws.scratch_bytes / sizeof(float2) / chunks, 65535u);
  float2* stats = reinterpret_cast<float2*>(ws.scratch);
  for (size_t r = 0; r < rows; r += most) {
    const dim3 grid(chunks, (uint32_t)std::min(most, rows - r));
    softmax_stats<FOURS><<<grid, kThreads, 0, s>>>(x + r * cols, cols, per, stats);
    softmax_values<FOURS><<<grid, kThreads, 0, s>>>(x + r * cols, cols, per, stats,
                                                         y + r * cols);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_softmax(const float* x, float* y, size_t rows, size_t cols, float temperature,
                          const Workspace& ws, hipStream_t s) {
  const float per = kLog2e / temperature;
  // Chunks of 8192 values where they make a workgroup a CU, else of 2048, so that a few rows
  // have more of them (of 151,936 logits 24 rows 10.1 us by 8192 and 12.0 by 2048, 16 rows
  // 9.8 both; 5 rows 7.6 by 2048).
  const bool many = rows * ((cols + 8191u) / 8192u) >= 256u;
  return many ? softmax_rows<8>(x, y, rows, cols, per, ws, s)
              : softmax_rows<2>(x, y, rows, cols, per, ws, s);
}

hipError_t launch_verify(const VerifyArgs& a, const Workspace& ws, hipStream_t s) {
  const uint32_t chunks = (a.vocab + kChunk - 1u) / kChunk;
  uint64_t* sums = reinterpret_cast<uint64_t*>(ws.scratch);
  uint32_t* counters = static_cast<uint32_t*>(ws.ptr);  // at rest zero, and left so
  static_assert(65535u * 4u + 64u <= kWorkspaceCounterBytes, "a counter for each sequence");
  const uint32_t most =
      (uint32_t)std::min<size_t>(ws.scratch_bytes / sizeof(uint64_t) / chunks, 65535u);
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
    const dim3 grid(chunks, b.sequences);
    verify_kernel<<<grid, kThreads, 0, s>>>(b, sums, counters, ws.ptr);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace sihip
