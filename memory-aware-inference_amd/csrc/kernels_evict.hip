// Eviction from a paged cache by accumulated attention weight.
//
// Weights are compared as 32-bit integers whose order is theirs, so the
// selection is exact and its ties are too: the `need`-th largest integer T of
// the slots between the first `sinks` and the last `recent` is found digit by
// digit from histograms, then a pass over the slots in order keeps those above
// T and the first ones equal to it.  A second kernel moves the kept rows.
#include "decode_internal.h"

namespace sihip {
namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64;

// Integers in the order of the weights: a NaN is the least, -0 equals +0.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sum of v over the workgroup's threads, and all of it.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* part, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u;
  uint32_t x = v;
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63u) part[wave] = x;
  __syncthreads();
  uint32_t before = 0u;
  total = 0u;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) {
    if (i < wave) before += part[i];
    total += part[i];
  }
  return before + x - v;
}

// grid (kv_heads, sequences): the kept slots of one head, and their weights.
__global__ __launch_bounds__(kThreads) void evict_select(EvictArgs a) {
  __shared__ uint32_t bins[2048], part[kWaves], found[2];
  const CacheView& c = a.from;
  const uint32_t h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  const size_t head = (size_t)s * c.kv_heads + h;
  const float* w = a.weights + head * a.weights_stride;
  float* to_w = a.to_weights + head * a.to_weights_stride;
  uint32_t* kept = a.kept + head * a.keep;
  const uint32_t n = held(c, s);
  const uint32_t left = min(n, a.keep);
  if (tid == 0u && h == 0u) {
    a.to.lengths[s] = left;
    if (c.lengths[s] > c.capacity) report_device_error(a.report, kDevErrCacheFull);
  }
  for (uint32_t i = left + tid; i < a.keep; i += kThreads) kept[i] = kNone;
  if (n <= a.keep) {
    for (uint32_t i = tid; i < n; i += kThreads) {
      kept[i] = i;
      to_w[i] = w[i];
    }
    return;
  }
  // the need-th largest of the slots in [lo, hi)
  const uint32_t lo = a.sinks, hi = n - a.recent;
  uint32_t need = a.keep - a.sinks - a.recent, prefix = 0u, known = 0u;
  if (need != 0u) {
    for (uint32_t digit = 0; digit < 3u; ++digit) {
      const uint32_t shift = digit == 0u ? 21u : digit == 1u ? 10u : 0u;
      const uint32_t size = digit == 2u ? 1024u : 2048u;
      for (uint32_t i = tid; i < size; i += kThreads) bins[i] = 0u;
      __syncthreads();
      for (uint32_t i = lo + tid; i < hi; i += kThreads) {
        const uint32_t k = rank_of(w[i]);
        if ((k & known) == prefix) atomicAdd(&bins[(k >> shift) & (size - 1u)], 1u);
      }
      __syncthreads();
      // thread i has the bins size - 1 - (size / kThreads) i and below
      const uint32_t each = size / kThreads;
      uint32_t mine = 0u;
      for (uint32_t j = 0; j < each; ++j) mine += bins[size - 1u - (tid * each + j)];
      uint32_t total;
      uint32_t before = block_scan(mine, part, total);
      if (before < need && need <= before + mine)
        for (uint32_t j = 0; j < each; ++j) {
          const uint32_t bin = size - 1u - (tid * each + j);
          if (before < need && need <= before + bins[bin]) {
            found[0] = bin;
            found[1] = need - before;
          }
          before += bins[bin];
        }
      __syncthreads();
      prefix |= found[0] << shift;
      known |= (size - 1u) << shift;
      need = found[1];
      __syncthreads();
    }
  }
  // the slots above T and the first `need` equal to it (none where nothing is needed)
  const bool none = known == 0u;
  uint32_t out = 0u, ties = 0u;
  for (uint32_t base = 0; base < n; base += kThreads) {
    const uint32_t i = base + tid;
    const bool inside = i >= lo && i < hi;
    const uint32_t k = inside && !none ? rank_of(w[i]) : 0u;
    const bool tie = inside && !none && k == prefix;
    uint32_t total;
    const uint32_t tie_rank = ties + block_scan(tie ? 1u : 0u, part, total);
    ties += total;
    const bool keep = i < n && (!inside || (!none && (k > prefix || (tie && tie_rank < need))));
    const uint32_t at = out + block_scan(keep ? 1u : 0u, part, total);
    out += total;
    if (keep) {
      kept[at] = i;
      to_w[at] = w[i];
    }
  }
}

// grid (rows / rows a workgroup, kv_heads, sequences): U is the unit that rows
// are moved in.
template <typename U>
__global__ __launch_bounds__(256) void evict_move(EvictArgs a, uint32_t units) {
  const uint32_t h = blockIdx.y, s = blockIdx.z;
  const uint32_t left = min(held(a.from, s), a.keep);
  const uint32_t* kept = a.kept + ((size_t)s * a.from.kv_heads + h) * a.keep;
  const uint32_t rows = 256u / units ? 256u / units : 1u;
  const uint32_t mine = threadIdx.x / units, u0 = threadIdx.x - mine * units;
  if (mine >= rows) return;
  for (uint32_t i = blockIdx.x * rows + mine; i < left; i += gridDim.x * rows) {
    const uint32_t src = cache_row(a.from, s, h, kept[i]);
    const uint32_t dst = cache_row(a.to, s, h, i);
    if (src == kNone || dst == kNone) {
      if (u0 == 0u) report_device_error(a.report, kDevErrCachePage);
      continue;
    }
    for (uint32_t u = u0; u < units; u += 256u) {
      static_cast<U*>(a.to.keys)[(size_t)dst * units + u] =
          static_cast<const U*>(a.from.keys)[(size_t)src * units + u];
      static_cast<U*>(a.to.values)[(size_t)dst * units + u] =
          static_cast<const U*>(a.from.values)[(size_t)src * units + u];
    }
  }
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t s) {
  const CacheView& c = a.from;
  evict_select<<<dim3(c.kv_heads, c.sequences), kThreads, 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t bytes = c.head_dim * (c.type == kKvF32 ? 4u : 2u);
  uintptr_t at = (uintptr_t)c.keys | (uintptr_t)c.values | (uintptr_t)a.to.keys |
                 (uintptr_t)a.to.values | bytes;
  auto go = [&](auto kernel, uint32_t units) {
    const uint32_t rows = std::max(1u, 256u / units);
    const uint32_t blocks = std::min((a.keep + rows - 1u) / rows, 65535u);
    kernel<<<dim3(blocks, c.kv_heads, c.sequences), 256, 0, s>>>(a, units);
  };
  if (at % 16u == 0u)
    go(evict_move<uint4>, bytes / 16u);
  else if (at % 4u == 0u)
    go(evict_move<uint32_t>, bytes / 4u);
  else
    go(evict_move<uint16_t>, bytes / 2u);
  return hipGetLastError();
}

}  // namespace sihip
