// Attention over a paged cache on the matrix cores.
//
// A wave takes tiles of slots (32 of a 16-bit cache, 16 of an f32 one) with 16
// rows (a row is one query head of one new token) and keeps the running
// maximum, sum and output of each row in registers:
//
//   scores^T = K q^T   A: a lane's slot and 8 of its values, B: a row's query
//   out^T   += V^T p^T A: 8 slots of one value, B: the row's p of those slots
//
// The first product leaves a lane with four slots of one row in each of its
// results, and the slots of the second product's sum may stand in any order,
// so p enters it from the registers it is in.  V's tile is loaded row by row,
// 16 lanes a row, and turned in registers (one byte permutation for two
// values).  A row's maximum, sum and scale belong to its lanes.
//
// Precision: q and p are f32.  With a 16-bit cache they go to the matrix cores
// as sums of 16-bit numbers: for BF16 three, the leading 8 bits, the next 8
// and the last 8 (exact); for F16 two of 11 bits, q scaled by a power of two
// that puts its row's largest value at 2^14, and p times 2^14, so that neither
// half loses bits to F16's range.  An f32 cache takes the f32 instructions.
// Products and sums are f32.
//
// The slots of all sequences are dealt to workgroups in equal parts; the four
// waves of one take its tiles in turn and join at its end.  A sequence of
// several parts is joined by a second kernel.
#include "attention_common.h"

namespace sihip {

using namespace attn;

namespace {

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}
constexpr uint32_t kLows = 0x05040100u, kHighs = 0x07060302u;  // of two words: (lo, hi) halves

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- types of cache ------------------------------------------------------------
struct Bf16 {
  // (words of values: exponents, and what carries out of one that is all ones)
  static constexpr uint32_t kSlots = 32, kBytes = 2, kPieces = 3;
  static constexpr float kShift = 0.0f;  // p is held times 2^kShift
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  // The pieces of x and y, in the halves of one word each.  What is no number
  // is its first piece alone.
  static __device__ __forceinline__ void split(float x, float y, uint32_t (&w)[kPieces]) {
    const uint32_t top = 0xffff0000u;
    float r = x, s = y;
#pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
      const uint32_t a = __float_as_uint(r), b = __float_as_uint(s);
      w[i] = perm(b, a, kHighs);
      r -= __uint_as_float(a & top);
      s -= __uint_as_float(b & top);
    }
  }
  static constexpr uint32_t kExponent = 0x7f807f80u, kUnit = 0x00800080u,
                            kCarry = 0x80008000u;
};
struct F16 {
  static constexpr uint32_t kSlots = 32, kBytes = 2, kPieces = 2;
  static constexpr float kShift = 14.0f;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ void split(float x, float y, uint32_t (&w)[kPieces]) {
    const _Float16 a = (_Float16)x, b = (_Float16)y;
    const _Float16 c = (_Float16)(x - (float)a), d = (_Float16)(y - (float)b);
    w[0] = (uint32_t)__builtin_bit_cast(uint16_t, a) |
           (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
    w[1] = (uint32_t)__builtin_bit_cast(uint16_t, c) |
           (uint32_t)__builtin_bit_cast(uint16_t, d) << 16;
  }
  static constexpr uint32_t kExponent = 0x7c007c00u, kUnit = 0x04000400u,
                            kCarry = 0x80008000u;
};
struct F32 {
  static constexpr uint32_t kSlots = 16, kBytes = 4, kPieces = 1;
  static constexpr float kShift = 0.0f;
  static constexpr uint32_t kExponent = 0x7f800000u, kUnit = 0x00800000u, kCarry = 0x80000000u;
};

template <typename T, uint32_t DC>
struct Shape {
  static constexpr bool kWide = T::kBytes == 4;            // f32 instructions
  static constexpr uint32_t kSubs = T::kSlots / 16;        // score tiles of 16 slots
  static constexpr uint32_t kSteps = DC / (kWide ? 16 : 32);  // 16-byte pieces of a key a lane
  static constexpr uint32_t kRows = kWide ? 4 : 8;         // value rows a lane
  // values of a row that a lane loads at once, and how often
  static constexpr uint32_t kEach = kWide ? 4 : DC >= 128 ? 8 : 4;
  static constexpr uint32_t kPasses = DC / (16 * kEach);
  static constexpr uint32_t kWords = kEach * T::kBytes / 4;
  static constexpr uint32_t kQueryBytes = T::kPieces * kSteps * 64 * 16;
  static constexpr uint32_t kOutStride = DC + 4;  // words of a row of the join
  static constexpr uint32_t kOutBytes = kWaves * 16 * kOutStride * 4;
  static constexpr uint32_t kShared = kQueryBytes > kOutBytes ? kQueryBytes : kOutBytes;
};

// ---- how the work is dealt -------------------------------------------------------
// A part: the slots [c0, c1) of one sequence, the `index`-th of its `parts`
// ones, which are numbered from `first` through all sequences.
struct Part {
  uint32_t seq, c0, c1, index, parts, first;
};

// The slots that any row of a sequence sees, from a multiple of `unit` on.
__device__ __forceinline__ void sequence_span(const AttentionArgs& a, uint32_t seq, uint32_t unit,
                                              uint32_t& start, uint32_t& slots) {
  const uint32_t count = brought(a.counts, seq, a.tokens);
  start = slots = 0u;
  if (count == 0u) return;
  const uint32_t length = held(a.cache, seq);
  uint32_t begin, end, other;
  seen_slots(length, 0u, a.cache.capacity, a.window, begin, other);
  seen_slots(length, count - 1u, a.cache.capacity, a.window, other, end);
  start = begin / unit * unit;
  slots = end > start ? end - start : 0u;
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t lane) {
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) {
    const uint32_t w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  return v;
}

// Slots a part: all sequences' over the parts wanted, in whole rounds of the
// workgroup's waves.  Every lane of a wave takes part; kernels of one launch
// agree on it since they go by the same lengths.
__device__ __forceinline__ uint32_t part_slots(const AttentionArgs& a, uint32_t unit,
                                               uint32_t wanted) {
  const uint32_t lane = threadIdx.x & 63u, round = unit * kWaves;
  uint64_t total = 0u;
  for (uint32_t base = 0; base < a.cache.sequences; base += 64u) {
    uint32_t start, slots = 0u;
    if (base + lane < a.cache.sequences) sequence_span(a, base + lane, unit, start, slots);
    // (in rounds: a sum of 64 spans below 2^31 would not fit 32 bits)
    total += wave_sum((slots + round - 1u) / round);
  }
  const uint64_t each = (total + wanted - 1u) / wanted;
  return (uint32_t)min(max(each, (uint64_t)1u), (uint64_t)(0x80000000u / round)) * round;
}
// The part numbered `number`; parts = 0 where there is none.  With BY_SEQUENCE
// the first part of sequence `number`.
template <bool BY_SEQUENCE = false>
__device__ __forceinline__ Part find_part(const AttentionArgs& a, uint32_t unit, uint32_t wanted,
                                          uint32_t number) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t each = part_slots(a, unit, wanted);
  Part p{};
  uint32_t first = 0u;
  for (uint32_t base = 0; base < a.cache.sequences; base += 64u) {
    uint32_t start = 0u, slots = 0u, n = 0u;
    if (base + lane < a.cache.sequences) {
      sequence_span(a, base + lane, unit, start, slots);
      n = max(1u, (slots + each - 1u) / each);
    }
    const uint32_t upto = wave_scan(n, lane);
    const uint64_t here = __builtin_amdgcn_ballot_w64(
        BY_SEQUENCE ? base + lane == number : n != 0u && number < first + upto);
    if (here) {
      const uint32_t at = (uint32_t)__builtin_ctzll(here);
      start = __shfl(start, at, 64);
      slots = __shfl(slots, at, 64);
      p.parts = __shfl(n, at, 64);
      p.first = first + __shfl(upto, at, 64) - p.parts;
      p.seq = base + at;
      p.index = BY_SEQUENCE ? 0u : number - p.first;
      p.c0 = start + p.index * each;
      p.c1 = min(p.c0 + each, start + slots);
      return p;
    }
    first += __shfl(upto, 63, 64);
  }
  return p;
}

// ---- running maxima and sums -------------------------------------------------------
// (m, l) of two sets of a row's slots, joined.  l < 0: there are slots, and all
// scores are -inf, which says nothing beside a set that has others.
__device__ __forceinline__ float2 joined(float2 x, float2 y) {
  const float m = fmaxf(x.x, y.x);
  const float u = x.x == -INFINITY ? (x.y < 0.0f ? 0.0f : x.y) : x.y * exp2_of(x.x - m);
  const float v = y.x == -INFINITY ? (y.y < 0.0f ? 0.0f : y.y) : y.y * exp2_of(y.x - m);
  const bool no_more = m == -INFINITY && (x.y < 0.0f || y.y < 0.0f) && u + v == 0.0f;
  return make_float2(m, no_more ? -1.0f : u + v);
}
// What a row's sums are taken times in the end, and its (m, 1 / l) for the
// weights: 0 / 0 where every score is -inf.
__device__ __forceinline__ float row_times(float2 st) {
  return st.y < 0.0f ? NAN : 1.0f / st.y;
}
template <typename T>
__device__ __forceinline__ float2 row_stats(float2 st) {
  if (st.y == 0.0f) return make_float2(0.0f, 0.0f);
  return make_float2(st.x == -INFINITY ? 0.0f : st.x - T::kShift, row_times(st));
}

// ---- the kernel ------------------------------------------------------------------
struct Outputs {
  float2* part_stats;
  float* part_out;
  float2* stats;
  float* scores;
  uint32_t score_stride, wanted, tiles, units;  // units: workgroups of one row tile
};

// Blocks of the row tiles of one part and head follow each other on one XCD
// (blocks are dealt to the eight in turn), so its L2 serves them the same rows.
__device__ __forceinline__ void block_work(const Outputs& o, uint32_t& unit, uint32_t& tile) {
  const uint32_t b = blockIdx.x;
  if (o.tiles == 1u) {
    unit = b;
    tile = 0u;
    return;
  }
  const uint32_t xcd = b & 7u, i = b >> 3, row = i / o.tiles;
  tile = i - row * o.tiles;
  unit = row * 8u + xcd;
}

template <typename T, uint32_t DC, bool FULL>
__global__ __launch_bounds__(kThreads, 2) void attention_mfma(AttentionArgs a, Outputs o) {
  using S = Shape<T, DC>;
  __shared__ __attribute__((aligned(16))) uint8_t shared[S::kShared];
  __shared__ float row_m[kWaves][16], row_l[kWaves][16], row_scale[16];
  const CacheView& c = a.cache;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid / 64u;
  const uint32_t n = lane & 15u, j = lane >> 4;
  const uint32_t dim = FULL ? DC : c.head_dim;
  uint32_t unit, tile;
  block_work(o, unit, tile);
  if (unit >= o.units) return;
  const uint32_t kv = unit % c.kv_heads;
  const Part part = find_part(a, T::kSlots, o.wanted, unit / c.kv_heads);
  if (part.parts == 0u) return;
  const uint32_t seq = part.seq;
  const uint32_t count = brought(a.counts, seq, a.tokens), length = held(c, seq);
  const uint32_t rows = a.tokens * a.group;
  if (unit % c.kv_heads == 0u && tile == 0u && part.index == 0u && tid == 0u &&
      (uint64_t)c.lengths[seq] + count > c.capacity && count != 0u)
    report_device_error(a.report, kDevErrCacheFull);

  // ---- the rows' queries, as B operands, into LDS
  u32x4* q_lds = reinterpret_cast<u32x4*>(shared);
  const auto query = [&](uint32_t r) {
    const uint32_t t = r / a.group, h = kv * a.group + (r - t * a.group);
    return a.q + ((size_t)seq * a.tokens + t) * a.q_token_stride + h * a.q_head_stride;
  };
  const float scale = a.scale * kLog2e;
  if constexpr (T::kShift != 0.0f) {
    // the rows' powers of two: 16 threads a row
    const uint32_t r = tile * 16u + tid / 16u;
    float top = 0.0f;
    bool finite = true;
    if (r < rows && r / a.group < count) {
      const float* x = query(r);
      for (uint32_t d = tid & 15u; d < dim; d += 16u) {
        const float v = fabsf(x[d] * scale);
        finite &= v < INFINITY;
        top = fmaxf(top, v);
      }
    }
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) {
      top = fmaxf(top, __shfl_xor(top, s, 64));
      finite &= __shfl_xor((int)finite, s, 64) != 0;
    }
    const uint32_t e = max(__float_as_uint(top) >> 23, 16u);
    if ((tid & 15u) == 0u)
      row_scale[tid / 16u] = finite ? __uint_as_float((268u - e) << 23) : 1.0f;
    __syncthreads();
  }
  for (uint32_t i = tid; i < S::kSteps * 64u; i += kThreads) {
    const uint32_t step = i / 64u, l = i & 63u, r = tile * 16u + (l & 15u);
    constexpr uint32_t kValues = S::kWide ? 4 : 8;
    const uint32_t d0 = (step * 4u + (l >> 4)) * kValues;
    float x[kValues];
    const bool there = r < rows && r / a.group < count && d0 < dim;
#pragma unroll
    for (uint32_t v = 0; v < kValues; ++v) x[v] = 0.0f;
    if (there) {
      const float* src = query(r) + d0;
#pragma unroll
      for (uint32_t v = 0; v < kValues; ++v) x[v] = src[v] * scale;
    }
    if constexpr (S::kWide) {
      u32x4 w;
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) w[v] = __float_as_uint(x[v]);
      q_lds[i] = w;
    } else {
      u32x4 w[T::kPieces];
      const float s = T::kShift != 0.0f ? row_scale[l & 15u] : 1.0f;
#pragma unroll
      for (uint32_t v = 0; v < 8; v += 2) {
        uint32_t p[T::kPieces];
        T::split(x[v] * s, x[v + 1] * s, p);
#pragma unroll
        for (uint32_t k = 0; k < T::kPieces; ++k) w[k][v / 2] = p[k];
      }
#pragma unroll
      for (uint32_t k = 0; k < T::kPieces; ++k) q_lds[k * S::kSteps * 64u + i] = w[k];
    }
  }
  __syncthreads();

  // ---- the lane's row, and its slots
  const uint32_t r = tile * 16u + n, t = r / a.group;
  uint32_t begin = 0u, end = 0u;
  if (r < rows && t < count) seen_slots(length, t, c.capacity, a.window, begin, end);
  float unscale = 1.0f;
  if constexpr (T::kShift != 0.0f)
    unscale = __uint_as_float((254u << 23) - __float_as_uint(row_scale[n]));
  // the tile's tokens, and the slots that all of their rows see, or any
  const uint32_t t_first = min(tile * 16u / a.group, count);
  const uint32_t t_last = min((min(tile * 16u + 16u, rows) - 1u) / a.group + 1u, count);
  uint32_t any_lo = 0u, any_hi = 0u, all_lo = 0u, all_hi = 0u;
  if (t_first < t_last) {
    seen_slots(length, t_first, c.capacity, a.window, any_lo, all_hi);
    seen_slots(length, t_last - 1u, c.capacity, a.window, all_lo, any_hi);
  }
  const size_t row_at = ((size_t)seq * c.kv_heads + kv) * rows + r;
  float* score_row = o.scores && r < rows && t < count ? o.scores + row_at * o.score_stride : nullptr;

  const uint8_t* keys = static_cast<const uint8_t*>(c.keys);
  const uint8_t* values = static_cast<const uint8_t*>(c.values);
  const uint32_t row_bytes = dim * T::kBytes;
  const uint32_t hi = min(part.c1, any_hi);
  const uint32_t stride = T::kSlots * kWaves;
  const uint32_t first = part.c0 + wave * T::kSlots;

  // A tile's rows in two steps, so that the page numbers are there before the
  // rows are wanted: lane l has slot l % kSlots.
  const auto page_of = [&](uint32_t base) {
    const uint32_t slot = base + (lane & (T::kSlots - 1u));
    return slot < hi ? c.table[(size_t)seq * c.max_pages + divided(slot, c.div_mul, c.div_shift)]
                     : kNone;
  };
  uint32_t bad = 0u;
  const auto row_of = [&](uint32_t base, uint32_t page) {
    const uint32_t slot = base + (lane & (T::kSlots - 1u));
    if (slot >= hi) return kNone;
    if (page >= c.pages) {
      bad = 1u;
      return kNone;
    }
    return (page * c.kv_heads + kv) * c.page_tokens +
           (slot - divided(slot, c.div_mul, c.div_shift) * c.page_tokens);
  };
  // (a slot without a row reads the pool's first one, and is masked)
  const auto pointer = [&](const uint8_t* base, uint32_t row, uint32_t from) {
    const uint32_t at = __shfl(row, from, 64);
    return base + (size_t)(at == kNone ? 0u : at) * row_bytes;
  };
  u32x4 key[S::kSubs][S::kSteps];
  const auto load_keys = [&](uint32_t row) {
#pragma unroll
    for (uint32_t s = 0; s < S::kSubs; ++s) {
      const uint8_t* p = pointer(keys, row, s * 16u + n);
#pragma unroll
      for (uint32_t k = 0; k < S::kSteps; ++k) {
        uint32_t at = (k * 4u + j) * 16u;
        if (!FULL) at = min(at, row_bytes - 16u);  // (its query values are 0)
        key[s][k] = *reinterpret_cast<const u32x4*>(p + at);
      }
    }
  };
  uint32_t value[S::kRows][S::kPasses][S::kWords];
  const auto load_values = [&](uint32_t row) {
#pragma unroll
    for (uint32_t i = 0; i < S::kRows; ++i) {
      const uint8_t* p = pointer(values, row, i / 4u * 16u + j * 4u + i % 4u);
#pragma unroll
      for (uint32_t u = 0; u < S::kPasses; ++u) {
        uint32_t at = (u * 16u + n) * (S::kWords * 4u);
        if (!FULL) at = min(at, row_bytes - S::kWords * 4u);  // (its outputs are not stored)
        if constexpr (S::kWords == 4) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(p + at);
#pragma unroll
          for (uint32_t x = 0; x < 4; ++x) value[i][u][x] = w[x];
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(p + at);
          value[i][u][0] = w.x;
          value[i][u][1] = w.y;
        }
      }
    }
  };

  constexpr uint32_t kTiles = DC / 16;
  f32x4 out[kTiles];
#pragma unroll
  for (uint32_t i = 0; i < kTiles; ++i) out[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  bool any = false;  // the row sees a slot of the lane's

  // out^T += V^T p^T with the values in `value`
  const auto add_values = [&](const float (&p)[S::kRows]) {
    if constexpr (S::kWide) {
#pragma unroll
      for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
        for (uint32_t d = 0; d < S::kEach; ++d) {
          f32x4 acc = out[u * S::kEach + d];
#pragma unroll
          for (uint32_t i = 0; i < S::kRows; ++i)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(value[i][u][d]), p[i], acc,
                                                       0, 0, 0);
          out[u * S::kEach + d] = acc;
        }
    } else {
      u32x4 b[T::kPieces];
#pragma unroll
      for (uint32_t i = 0; i < 8; i += 2) {
        uint32_t w[T::kPieces];
        T::split(p[i], p[i + 1], w);
#pragma unroll
        for (uint32_t k = 0; k < T::kPieces; ++k) b[k][i / 2] = w[k];
      }
#pragma unroll
      for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
        for (uint32_t d = 0; d < S::kEach; ++d) {
          u32x4 v;
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            v[i] = perm(value[2 * i + 1][u][d / 2], value[2 * i][u][d / 2], d & 1 ? kHighs : kLows);
          f32x4 acc = out[u * S::kEach + d];
#pragma unroll
          for (uint32_t k = 0; k < T::kPieces; ++k) acc = T::mfma(v, b[k], acc);
          out[u * S::kEach + d] = acc;
        }
    }
  };

  uint32_t row = first < hi ? row_of(first, page_of(first)) : kNone;
  uint32_t page = first + stride < hi ? page_of(first + stride) : kNone;
  if (first < hi) load_keys(row);
  for (uint32_t base = first; base < hi; base += stride) {
    const uint32_t there = (uint32_t)__builtin_amdgcn_ballot_w64(row != kNone);
    const uint32_t next_page = base + 2u * stride < hi ? page_of(base + 2u * stride) : kNone;
    load_values(row);
    // ---- scores
    // (the queries are read each time: kept across tiles, they would not leave registers for
    // the tile)
    uint32_t q_at = lane;
    asm volatile("" : "+v"(q_at));
    f32x4 sum[S::kSubs];
    if constexpr (S::kWide) {
      f32x4 part_sum[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
      for (uint32_t k = 0; k < S::kSteps; ++k) {
        const u32x4 q = q_lds[k * 64u + q_at];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
          part_sum[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(
              __uint_as_float(key[0][k][e]), __uint_as_float(q[e]), part_sum[e & 1], 0, 0, 0);
      }
      sum[0] = part_sum[0] + part_sum[1];
    } else {
      f32x4 piece[S::kSubs][T::kPieces];
#pragma unroll
      for (uint32_t s = 0; s < S::kSubs; ++s)
#pragma unroll
        for (uint32_t k = 0; k < T::kPieces; ++k) piece[s][k] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (uint32_t k = 0; k < S::kSteps; ++k)
#pragma unroll
        for (uint32_t w = 0; w < T::kPieces; ++w) {
          const u32x4 q = q_lds[(w * S::kSteps + k) * 64u + q_at];
#pragma unroll
          for (uint32_t s = 0; s < S::kSubs; ++s)
            piece[s][w] = T::mfma(key[s][k], q, piece[s][w]);
        }
#pragma unroll
      for (uint32_t s = 0; s < S::kSubs; ++s) {
        sum[s] = piece[s][T::kPieces - 1];
#pragma unroll
        for (int k = (int)T::kPieces - 2; k >= 0; --k) sum[s] += piece[s][k];
        sum[s] *= unscale;
      }
    }
    // ---- the next tile's keys
    row = base + stride < hi ? row_of(base + stride, page) : kNone;
    page = next_page;
    if (base + stride < hi) load_keys(row);
    // ---- p
    float p[S::kRows], top = -INFINITY;
    bool seen[S::kRows];
#pragma unroll
    for (uint32_t i = 0; i < S::kRows; ++i) {
      const uint32_t at = i / 4u * 16u + j * 4u + i % 4u, slot = base + at;
      seen[i] = slot >= begin && slot < end && (there >> at & 1u) != 0u;
      any |= seen[i];
      p[i] = seen[i] ? sum[i / 4u][i % 4u] : -INFINITY;
      top = fmaxf(top, p[i]);
    }
    if (score_row) {
#pragma unroll
      for (uint32_t s = 0; s < S::kSubs; ++s) {
        const uint32_t slot = base + s * 16u + j * 4u;
        if (slot < o.score_stride)
          *reinterpret_cast<float4*>(score_row + slot) =
              make_float4(p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float now = fmaxf(m, top);
    const float from = now == -INFINITY ? 0.0f : now - T::kShift;
    if (__builtin_amdgcn_ballot_w64(now > m)) {
      const float keep = m == -INFINITY ? 0.0f : exp2_of(m - now);
      l *= keep;
#pragma unroll
      for (uint32_t i = 0; i < kTiles; ++i) out[i] *= keep;
      m = now;
    }
#pragma unroll
    for (uint32_t i = 0; i < S::kRows; ++i) {
      p[i] = seen[i] ? exp2_of(p[i] - from) : 0.0f;
      l += p[i];
    }
    // ---- out
    // A slot that no row sees may hold anything: its values are taken as 0.  So
    // are those of a slot with a value that is no finite number, where not all
    // rows see it, for 0 times that would reach the others; the rows that do
    // see it are none from then on.
    const bool inside = base >= all_lo && base + T::kSlots <= all_hi &&
                        there == (T::kSlots == 32u ? 0xffffffffu : 0xffffu | there);
    if (!inside) {
      bool lost = false;
#pragma unroll
      for (uint32_t i = 0; i < S::kRows; ++i) {
        const uint32_t at = i / 4u * 16u + j * 4u + i % 4u, slot = base + at;
        bool use = slot >= any_lo && slot < any_hi && (there >> at & 1u) != 0u;
        uint32_t odd = 0u;
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t x = 0; x < S::kWords; ++x)
            odd |= (value[i][u][x] & T::kExponent) + T::kUnit;
        const uint64_t odds = __builtin_amdgcn_ballot_w64((odd & T::kCarry) != 0u);
        if ((odds >> (16u * j) & 0xffffu) != 0u) {  // (16 lanes have the slot's values)
          lost |= seen[i];
          use = false;
        }
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t x = 0; x < S::kWords; ++x) value[i][u][x] = use ? value[i][u][x] : 0u;
      }
      const uint64_t losts = __builtin_amdgcn_ballot_w64(lost);
      if (losts != 0u && (losts >> n & 0x0001000100010001u) != 0u) {
#pragma unroll
        for (uint32_t i = 0; i < kTiles; ++i) out[i] = f32x4{NAN, NAN, NAN, NAN};
      }
    }
    add_values(p);
  }
  if (bad) report_device_error(a.report, kDevErrCachePage);

  // ---- the waves join
  // A row with slots whose scores are all -inf (0 / 0 in the end) has l = -1
  // until it meets one that is not; a row without slots has l = 0.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  const uint64_t anys = __builtin_amdgcn_ballot_w64(any);
  if (l == 0.0f && m == -INFINITY && (anys >> n & 0x0001000100010001u) != 0u) l = -1.0f;
  if (j == 0u) {
    row_m[wave][n] = m;
    row_l[wave][n] = l;
  }
  __syncthreads();  // (and the queries are no longer read)
  float top = -INFINITY;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, row_m[w][n]);
  const float mine = m == -INFINITY ? 0.0f : exp2_of(m - top);
  float* join = reinterpret_cast<float*>(shared) + (wave * 16u + n) * S::kOutStride;
#pragma unroll
  for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x)
#pragma unroll
      for (uint32_t d = 0; d < S::kEach; d += 4) {
        float4 v;
        v.x = out[u * S::kEach + d][x] * mine;
        v.y = out[u * S::kEach + d + 1][x] * mine;
        v.z = out[u * S::kEach + d + 2][x] * mine;
        v.w = out[u * S::kEach + d + 3][x] * mine;
        *reinterpret_cast<float4*>(join + (u * 16u + j * 4u + x) * S::kEach + d) = v;
      }
  __syncthreads();
  // sixteen threads a row
  const uint32_t jr = tid / 16u, jn = tid & 15u, out_row = tile * 16u + jr;
  if (out_row >= rows) return;
  float2 st = make_float2(-INFINITY, 0.0f);
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) st = joined(st, make_float2(row_m[w][jr], row_l[w][jr]));
  const bool alone = part.parts == 1u;
  const size_t part_row =
      (((size_t)(part.first + part.index) * c.kv_heads + kv) * o.tiles + tile) * 16u + jr;
  const uint32_t jt = out_row / a.group, jh = kv * a.group + (out_row - jt * a.group);
  if (jn == 0u) {
    if (!alone) o.part_stats[part_row] = st;
    else if (o.stats)
      o.stats[((size_t)seq * c.kv_heads + kv) * rows + out_row] = row_stats<T>(st);
  }
  float* to = alone ? a.out + (((size_t)seq * a.tokens + jt) * a.heads + jh) * dim
                    : o.part_out + part_row * dim;
  const float times = alone ? row_times(st) : 1.0f;
  for (uint32_t d = jn * 4u; d < dim; d += 64u) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (st.y != 0.0f) {  // (a row that sees nothing has no part in what its columns hold)
#pragma unroll
      for (uint32_t w = 0; w < kWaves; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(shared) +
                                                          (w * 16u + jr) * S::kOutStride + d);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      v.x *= times, v.y *= times, v.z *= times, v.w *= times;
    }
    *reinterpret_cast<float4*>(to + d) = v;
  }
}

// ---- the parts of a sequence ---------------------------------------------------------
// grid (kv_heads * rows, sequences): threads take four values of the row each,
// in groups that take every so-manieth part.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_join(AttentionArgs a, Outputs o) {
  __shared__ float4 shared[kThreads];
  const CacheView& c = a.cache;
  const uint32_t rows = a.tokens * a.group, kv = blockIdx.x / rows, r = blockIdx.x - kv * rows;
  const uint32_t seq = blockIdx.y, tid = threadIdx.x, lane = tid & 63u;
  const Part part = find_part<true>(a, T::kSlots, o.wanted, seq);
  if (part.parts <= 1u) return;  // written already
  const auto at = [&](uint32_t p) {
    return (((size_t)(part.first + p) * c.kv_heads + kv) * o.tiles + r / 16u) * 16u + r % 16u;
  };
  float2 st = make_float2(-INFINITY, 0.0f);
  for (uint32_t p = lane; p < part.parts; p += 64u) st = joined(st, o.part_stats[at(p)]);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1)
    st = joined(st, make_float2(__shfl_xor(st.x, s, 64), __shfl_xor(st.y, s, 64)));
  const uint32_t dim = c.head_dim, width = dim / 4u, groups = kThreads / width;
  const uint32_t group = tid / width, d = (tid - group * width) * 4u;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (group < groups) {
#pragma unroll 4
    for (uint32_t p = group; p < part.parts; p += groups) {
      const size_t row = at(p);
      const float m = o.part_stats[row].x;
      const float w = m == -INFINITY ? 0.0f : exp2_of(m - st.x);
      const float4 x = *reinterpret_cast<const float4*>(o.part_out + row * dim + d);
      sum.x = fmaf(w, x.x, sum.x);
      sum.y = fmaf(w, x.y, sum.y);
      sum.z = fmaf(w, x.z, sum.z);
      sum.w = fmaf(w, x.w, sum.w);
    }
    shared[group * width + d / 4u] = sum;
  }
  __syncthreads();
  if (group != 0u) return;
  for (uint32_t g = 1; g < groups; ++g) {
    const float4 x = shared[g * width + d / 4u];
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  const float times = row_times(st);
  const uint32_t t = r / a.group, h = kv * a.group + (r - t * a.group);
  float* to = a.out + (((size_t)seq * a.tokens + t) * a.heads + h) * dim + d;
  if (st.y != 0.0f)
    sum = make_float4(sum.x * times, sum.y * times, sum.z * times, sum.w * times);
  else
    sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  *reinterpret_cast<float4*>(to) = sum;
  if (o.stats && tid == 0u) o.stats[((size_t)seq * c.kv_heads + kv) * rows + r] = row_stats<T>(st);
}

template <typename T, uint32_t DC, bool FULL>
hipError_t launch(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  const uint32_t blocks = o.tiles == 1u ? o.units : (o.units + 7u) / 8u * 8u * o.tiles;
  attention_mfma<T, DC, FULL><<<blocks, kThreads, 0, s>>>(a, o);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || o.wanted == 1u) return e;
  attention_join<T><<<dim3(a.cache.kv_heads * a.tokens * a.group, a.cache.sequences), kThreads, 0,
                      s>>>(a, o);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  switch (a.cache.head_dim) {
    case 64: return launch<T, 64, true>(a, o, s);
    case 128: return launch<T, 128, true>(a, o, s);
    case 256: return launch<T, 256, true>(a, o, s);
    default: break;
  }
  if (a.cache.head_dim < 64u) return launch<T, 64, false>(a, o, s);
  if (a.cache.head_dim < 128u) return launch<T, 128, false>(a, o, s);
  return launch<T, 256, false>(a, o, s);
}

}  // namespace

hipError_t launch_attention_mfma(const AttentionArgs& a, const Space& sp, bool* taken,
                                 hipStream_t s) {
  const CacheView& c = a.cache;
  // sixteen-byte loads of keys and values, and stores of the output
  const uint32_t row = c.head_dim * (c.type == kKvF32 ? 4u : 2u);
  *taken = row % 16u == 0u && ((uintptr_t)c.keys | (uintptr_t)c.values | (uintptr_t)a.out) % 16u == 0u;
  if (!*taken) return hipSuccess;
  uint8_t* w = static_cast<uint8_t*>(a.workspace);
  Outputs o{};
  o.part_stats = reinterpret_cast<float2*>(w + sp.part_stats);
  o.part_out = reinterpret_cast<float*>(w + sp.part_out);
  o.stats = a.weights ? reinterpret_cast<float2*>(w + sp.stats) : nullptr;
  o.scores = a.weights ? reinterpret_cast<float*>(w + sp.scores) : nullptr;
  o.score_stride = sp.score_stride;
  o.wanted = parts_wanted(c, a.tokens, a.group);
  o.tiles = row_tiles(a.tokens, a.group);
  o.units = parts_most(c, a.tokens, a.group) * c.kv_heads;
  if (c.type == kKvF32) return launch_type<F32>(a, o, s);
  if (c.type == kKvF16) return launch_type<F16>(a, o, s);
  return launch_type<Bf16>(a, o, s);
}

}  // namespace sihip
