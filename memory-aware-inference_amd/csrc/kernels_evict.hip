// Eviction from a paged cache by accumulated attention weight.
//
// Weights are compared as 32-bit integers whose order is theirs, so the
// selection is exact and its ties are too: the `need`-th largest integer T of
// the slots between the first `sinks` and the last `recent` is found digit by
// digit from histograms in LDS (as far as one bin holds both kept slots and
// others), then the slots above T and the first ones equal to it are kept.  A
// second kernel moves the kept rows; it is bound by memory, the selection by
// the chain of its passes.  So a head's selection is one workgroup's, whose
// threads read their slots, next to each other, once and hold them (up to 32768
// slots; more are read in each pass), and one scan over the threads places all
// that is kept.  Measured: 4 heads of 4111 slots of 256 values, 3001 kept,
// 15.9 us (selection 10, move 6) for 24.8 MB; 64 heads of up to 16,384 slots of
// 128, 6144 kept, 94 us (17 and 77) for 379 MB, the move at 4.9 TB/s read and
// written.
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
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* part, V& total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u;
  V x = v;
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) {
    const V y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63u) part[wave] = x;
  __syncthreads();
  V before = 0u;
  total = 0u;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) {
    if (i < wave) before += part[i];
    total += part[i];
  }
  return before + x - v;
}

// grid (kv_heads, sequences): the kept slots of one head, and their weights.
// HELD: a thread's slots, in registers; 0: any number, read in each pass.
template <uint32_t HELD>
__global__ __launch_bounds__(kThreads) void evict_select(EvictArgs a) {
  __shared__ uint4 bins[2048];  // (four counts a bin, by lane, so that fewer wait for one)
  __shared__ uint32_t part[kWaves], found[3], zeros;
  __shared__ uint64_t part64[kWaves];
  __shared__ uint16_t order[HELD ? HELD * kThreads : 1u];
  const CacheView& c = a.from;
  const uint32_t h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  const auto clear = [&](uint32_t size) {
    for (uint32_t i = tid; i < size; i += kThreads) bins[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0u) zeros = 0u;
  };
  clear(2048u);  // (while the length is read)
  const size_t head = (size_t)s * c.kv_heads + h;
  const float* w = a.weights + head * a.weights_stride;
  float* to_w = a.to_weights + head * a.to_weights_stride;
  uint32_t* kept = a.kept + head * a.keep;
  const uint32_t n = held(c, s), left = min(n, a.keep);
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
  // the thread's slots, in fours: [first, first + 4 fours)
  const uint32_t fours = (n + 4u * kThreads - 1u) / (4u * kThreads), first = tid * 4u * fours;
  const auto load = [&](uint32_t f) {
    const uint32_t at = first + 4u * f;
    Floats4 v{0.0f, 0.0f, 0.0f, 0.0f};
    if (at + 3u < n) {
      v = *reinterpret_cast<const Floats4*>(w + at);
    } else {
      if (at < n) v.x = w[at];
      if (at + 1u < n) v.y = w[at + 1u];
      if (at + 2u < n) v.z = w[at + 2u];
      if (at + 3u < n) v.w = w[at + 3u];
    }
    return v;
  };
  const uint32_t lo = a.sinks, hi = n - a.recent;
  // the held slots' ranks, and a bit for each: one of those in question; kept anyway
  constexpr uint32_t kFours = HELD ? HELD / 4u : 1u;
  uint32_t rank[4u * kFours], asked = 0u, safe = 0u;
  if constexpr (HELD != 0u) {
    Floats4 v[kFours];
#pragma unroll
    for (uint32_t f = 0; f < kFours; ++f) {
      v[f] = Floats4{0.0f, 0.0f, 0.0f, 0.0f};
      if (f < fours) v[f] = load(f);
    }
#pragma unroll
    for (uint32_t f = 0; f < kFours; ++f) {
      if (f >= fours) break;
      rank[4u * f] = rank_of(v[f].x), rank[4u * f + 1u] = rank_of(v[f].y);
      rank[4u * f + 2u] = rank_of(v[f].z), rank[4u * f + 3u] = rank_of(v[f].w);
#pragma unroll
      for (uint32_t j = 4u * f; j < 4u * f + 4u; ++j) {
        const uint32_t i = first + j;
        if (i < n) (i >= lo && i < hi ? asked : safe) |= 1u << j;
      }
    }
  }
  // every slot in question with its rank
  const auto each = [&](auto&& visit) {
    if constexpr (HELD != 0u) {
#pragma unroll
      for (uint32_t f = 0; f < kFours; ++f) {
        if (f >= fours) break;
#pragma unroll
        for (uint32_t j = 4u * f; j < 4u * f + 4u; ++j)
          if (asked >> j & 1u) visit(j, rank[j]);
      }
    } else {
      for (uint32_t f = 0; f < fours; ++f) {
        const Floats4 v = load(f);
        const uint32_t i = first + 4u * f;
        if (i >= lo && i < hi) visit(i, rank_of(v.x));
        if (i + 1u >= lo && i + 1u < hi) visit(i + 1u, rank_of(v.y));
        if (i + 2u >= lo && i + 2u < hi) visit(i + 2u, rank_of(v.z));
        if (i + 3u >= lo && i + 3u < hi) visit(i + 3u, rank_of(v.w));
      }
    }
  };
  // the need-th largest of the slots in [lo, hi)
  uint32_t need = a.keep - a.sinks - a.recent, prefix = 0u, known = 0u;
  const uint32_t zero = rank_of(0.0f);
  if (need != 0u) {
    for (uint32_t digit = 0; digit < 3u; ++digit) {
      const uint32_t shift = digit == 0u ? 21u : digit == 1u ? 10u : 0u;
      const uint32_t size = digit == 2u ? 1024u : 2048u;
      if (digit != 0u) clear(size);
      __syncthreads();
      // (slots that nothing ever saw weigh 0, many of them: counted apart, they do not
      // queue for one bin)
      uint32_t nothing = 0u;
      each([&](uint32_t, uint32_t k) {
        if ((k & known) == prefix) {
          if (k == zero) ++nothing;
          else
            atomicAdd(reinterpret_cast<uint32_t*>(bins) + 4u * ((k >> shift) & (size - 1u)) +
                          (tid & 3u),
                      1u);
        }
      });
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) nothing += __shfl_xor(nothing, o, 64);
      if ((tid & 63u) == 0u && nothing != 0u) atomicAdd(&zeros, nothing);
      __syncthreads();
      // thread i has the bins size - 1 - (size / kThreads) i and below
      const uint32_t every = size / kThreads, zero_bin = (zero >> shift) & (size - 1u);
      const auto bin_of = [&](uint32_t j) { return size - 1u - (tid * every + j); };
      const auto count_of = [&](uint32_t b) {
        return bins[b].x + bins[b].y + bins[b].z + bins[b].w + (b == zero_bin ? zeros : 0u);
      };
      uint32_t own = 0u, total;
      for (uint32_t j = 0; j < every; ++j) own += count_of(bin_of(j));
      uint32_t before = block_scan(own, part, total);
      if (before < need && need <= before + own)
        for (uint32_t j = 0; j < every; ++j) {
          const uint32_t count = count_of(bin_of(j));
          if (before < need && need <= before + count) {
            found[0] = bin_of(j);
            found[1] = need - before;
            found[2] = count;
          }
          before += count;
        }
      __syncthreads();
      prefix |= found[0] << shift;
      known |= (size - 1u) << shift;
      need = found[1];
      if (need == found[2]) break;  // all of the bin are kept: their other digits do not matter
      __syncthreads();
    }
  }
  // what is kept: the slots outside, those above T, and the first `need` equal to it
  const bool none = known == 0u;
  uint64_t total;
  if constexpr (HELD != 0u) {
    uint32_t equal = 0u;
    if (!none)
#pragma unroll
      for (uint32_t j = 0; j < HELD; ++j) {
        if (j % 4u == 0u && j / 4u >= fours) break;
        safe |= (asked >> j & 1u) != 0u && (rank[j] & known) > prefix ? 1u << j : 0u;
        equal |= (asked >> j & 1u) != 0u && (rank[j] & known) == prefix ? 1u << j : 0u;
      }
    const uint64_t own = (uint64_t)__popc(safe) << 32 | __popc(equal);
    const uint64_t before = block_scan(own, part64, total);
    const uint32_t ties = (uint32_t)before;
    for (uint32_t left_over = ties < need ? need - ties : 0u; equal != 0u && left_over != 0u;
         --left_over) {
      safe |= equal & -equal;
      equal &= equal - 1u;
    }
    // (a thread's slots go to places of their own: through LDS, so that the stores to
    // memory are of whole lines)
    for (uint32_t at = (uint32_t)(before >> 32) + min(ties, need); safe != 0u; safe &= safe - 1u)
      order[at++] = (uint16_t)(first + (uint32_t)__ffs(safe) - 1u);
    __syncthreads();
    for (uint32_t i = tid; i < left; i += kThreads) {
      const uint32_t slot = order[i];
      kept[i] = slot;
      to_w[i] = w[slot];
    }
  } else {
    const auto kind = [&](uint32_t i, float v) -> uint32_t {  // 2: kept, 1: equal, 0: not
      if (i >= n) return 0u;
      if (i < lo || i >= hi) return 2u;
      const uint32_t k = rank_of(v) & known;
      return none ? 0u : k > prefix ? 2u : k == prefix ? 1u : 0u;
    };
    const auto all = [&](auto&& visit) {
      for (uint32_t f = 0; f < fours; ++f) {
        const Floats4 v = load(f);
        visit(first + 4u * f, v.x);
        visit(first + 4u * f + 1u, v.y);
        visit(first + 4u * f + 2u, v.z);
        visit(first + 4u * f + 3u, v.w);
      }
    };
    uint64_t own = 0u;
    all([&](uint32_t i, float v) {
      const uint32_t k = kind(i, v);
      own += k == 2u ? 1ull << 32 : k;
    });
    const uint64_t before = block_scan(own, part64, total);
    uint32_t ties = (uint32_t)before, at = (uint32_t)(before >> 32) + min(ties, need);
    all([&](uint32_t i, float v) {
      const uint32_t k = kind(i, v);
      if (k == 2u || (k == 1u && ties < need)) {
        kept[at] = i;
        to_w[at] = v;
        ++at;
      }
      ties += k & 1u;
    });
  }
}

// grid (rows, kv_heads, sequences): U is the unit that rows are moved in.  A
// thread has four rows under way at once, each behind three dependent reads
// (its slot, the page, the row).  The rows are not used again here: their
// stores pass the caches by.
constexpr uint32_t kMoveThreads = 256, kMoveRows = 4;
template <typename U>
__global__ __launch_bounds__(kMoveThreads) void evict_move(EvictArgs a, uint32_t units) {
  const uint32_t h = blockIdx.y, s = blockIdx.z;
  const uint32_t left = min(held(a.from, s), a.keep);
  const uint32_t* kept = a.kept + ((size_t)s * a.from.kv_heads + h) * a.keep;
  const uint32_t rows = kMoveThreads / units;  // (a row has at most as many units)
  const uint32_t row = threadIdx.x / units, u = threadIdx.x - row * units;
  if (row >= rows) return;
  const U* keys = static_cast<const U*>(a.from.keys);
  const U* values = static_cast<const U*>(a.from.values);
  for (uint32_t i0 = blockIdx.x * rows * kMoveRows + row; i0 < left;
       i0 += gridDim.x * rows * kMoveRows) {
    uint32_t src[kMoveRows], dst[kMoveRows];
#pragma unroll
    for (uint32_t k = 0; k < kMoveRows; ++k) {
      const uint32_t i = i0 + k * rows;
      src[k] = i < left ? kept[i] : 0u;
    }
    U key[kMoveRows], value[kMoveRows];
#pragma unroll
    for (uint32_t k = 0; k < kMoveRows; ++k) {
      const uint32_t i = i0 + k * rows;
      src[k] = i < left ? cache_row(a.from, s, h, src[k]) : kNone;
      dst[k] = i < left ? cache_row(a.to, s, h, i) : kNone;
      if (i < left && (src[k] == kNone || dst[k] == kNone) && u == 0u)
        report_device_error(a.report, kDevErrCachePage);
    }
#pragma unroll
    for (uint32_t k = 0; k < kMoveRows; ++k)
      if (src[k] != kNone && dst[k] != kNone) {
        key[k] = keys[(size_t)src[k] * units + u];
        value[k] = values[(size_t)src[k] * units + u];
      }
#pragma unroll
    for (uint32_t k = 0; k < kMoveRows; ++k)
      if (src[k] != kNone && dst[k] != kNone) {
        __builtin_nontemporal_store(key[k], static_cast<U*>(a.to.keys) + (size_t)dst[k] * units + u);
        __builtin_nontemporal_store(value[k],
                                    static_cast<U*>(a.to.values) + (size_t)dst[k] * units + u);
      }
  }
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t s) {
  const CacheView& c = a.from;
  const dim3 heads(c.kv_heads, c.sequences);
  // (Selection and move of 4 heads of 4111 slots of 256: held in a place of 16,384 15.9 us, of
  // 32,768 17.0, read in each pass 17.5; 64 heads of 30,000 slots of 16: held 70 us, read 96.)
  if (c.capacity <= 16u * kThreads)
    evict_select<16><<<heads, kThreads, 0, s>>>(a);
  else if (c.capacity <= 32u * kThreads)
    evict_select<32><<<heads, kThreads, 0, s>>>(a);
  else
    evict_select<0><<<heads, kThreads, 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t bytes = c.head_dim * (c.type == kKvF32 ? 4u : 2u);
  const bool words =
      aligned4(c.keys) && aligned4(c.values) && aligned4(a.to.keys) && aligned4(a.to.values);
  auto go = [&](auto kernel, uint32_t units) {
    const uint32_t rows = kMoveThreads / units * kMoveRows;
    const uint32_t blocks = std::min((a.keep + rows - 1u) / rows, 65535u);
    kernel<<<dim3(blocks, c.kv_heads, c.sequences), kMoveThreads, 0, s>>>(a, units);
  };
  if (words && bytes % 16u == 0u)
    go(evict_move<Words4>, bytes / 16u);
  else if (words && bytes % 4u == 0u)
    go(evict_move<uint32_t>, bytes / 4u);
  else
    go(evict_move<uint16_t>, bytes / 2u);
  return hipGetLastError();
}

}  // namespace sihip
