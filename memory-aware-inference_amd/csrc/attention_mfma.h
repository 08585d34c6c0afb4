// Attention over a paged cache on the matrix cores: the kernel, for the three
// types of cache (kernels_attention_{f32,f16,bf16}.hip).
//
// A wave takes tiles of slots (32 of a 16-bit cache, 16 of an f32 one) with RT
// tiles of 16 rows (a row is one query head of one new token) and keeps the
// running maximum, sum and output of each row in registers:
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
// The slots of all sequences, in rounds of one tile for each wave of a
// workgroup, are dealt to the workgroups of a kv head in equal shares, one
// after another: a share may end one sequence and begin others.  A sequence
// inside one share is written at once; the sums of one that lies in several
// are joined in the order of the shares.
#pragma once

#include "attention_common.h"

namespace sihip {
namespace attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}
constexpr uint32_t kLows = 0x05040100u, kHighs = 0x07060302u;  // of two words: (lo, hi) halves

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

template <typename T, uint32_t DC, uint32_t RT, uint32_t WAVES>
struct Shape {
  static constexpr bool kWide = T::kBytes == 4;               // f32 instructions
  static constexpr uint32_t kSubs = T::kSlots / 16;           // score tiles of 16 slots
  static constexpr uint32_t kSteps = DC / (kWide ? 16 : 32);  // 16-byte pieces of a key a lane
  static constexpr uint32_t kRows = kWide ? 4 : 8;            // value rows a lane
  // values of a row that a lane loads at once, and how often
  static constexpr uint32_t kEach = kWide ? 4 : DC >= 128 ? 8 : 4;
  static constexpr uint32_t kPasses = DC / (16 * kEach);
  static constexpr uint32_t kWords = kEach * T::kBytes / 4;
  static constexpr uint32_t kTiles = DC / 16;  // of the output
  static constexpr uint32_t kItems = RT * kSteps * 64;  // 16-byte pieces of the queries
  static constexpr uint32_t kQueryBytes = T::kPieces * kItems * 16;
  static constexpr uint32_t kOutStride = DC + 4;  // words of a row of the join
  static constexpr uint32_t kOutBytes = WAVES / 2 * 16 * kOutStride * 4;  // half the waves'
  static constexpr uint32_t kShared = kQueryBytes > kOutBytes ? kQueryBytes : kOutBytes;
};

// Blocks of the row tiles of one share and head follow each other on one XCD
// (blocks are dealt to the eight in turn), so its L2 serves them the same rows.
__device__ __forceinline__ void block_work(const Outputs& o, uint32_t& unit, uint32_t& tile) {
  const uint32_t b = blockIdx.x;
  if (o.tile_groups == 1u) {
    unit = b;
    tile = 0u;
    return;
  }
  const uint32_t xcd = b & 7u, i = b >> 3, row = uniform(i / o.tile_groups);
  tile = i - row * o.tile_groups;
  unit = row * 8u + xcd;
}

template <typename T, uint32_t DC, bool FULL, uint32_t RT, uint32_t WAVES, uint32_t PER_SIMD>
__global__ __launch_bounds__(64 * WAVES, PER_SIMD) void attention_mfma(AttentionArgs a, Outputs o) {
  using S = Shape<T, DC, RT, WAVES>;
  constexpr uint32_t kThreads = 64 * WAVES, kRound = T::kSlots * WAVES;
  extern __shared__ __attribute__((aligned(16))) uint8_t shared[];
  __shared__ float row_m[WAVES][RT * 16], row_l[WAVES][RT * 16];
  __shared__ uint32_t row_top[RT * 16];
  __shared__ uint32_t last_share;
  const CacheView& c = a.cache;
  const uint32_t wave = uniform(threadIdx.x / 64u);
  const uint32_t dim = FULL ? DC : c.head_dim;
  const uint32_t row_bytes = dim * T::kBytes;
  const uint32_t rows = a.tokens * a.group;
  const uint8_t* keys = static_cast<const uint8_t*>(c.keys);
  const uint8_t* values = static_cast<const uint8_t*>(c.values);
  u32x4* q_lds = reinterpret_cast<u32x4*>(shared);

  uint32_t unit, group_at;
  block_work(o, unit, group_at);
  if (unit >= o.shares * c.kv_heads) return;
  const uint32_t share = uniform(unit / c.kv_heads), kv = unit - share * c.kv_heads;
  const uint32_t row0 = group_at * (RT * 16u);
  Walk walk = first_walk(a, kRound, o.shares, share);

  while (walk.at < walk.end) {
  // (afresh for each sequence: what follows from the thread's number would
  // otherwise stay in registers through the tiles)
  uint32_t tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const uint32_t lane = tid & 63u, n = lane & 15u, j = lane >> 4;
  const uint32_t seq = walk.seq;
  const uint32_t count = walk.count, length = walk.length;
  const uint32_t c0 = walk.start + (walk.at - walk.first) * kRound;
  const uint32_t c1 = min(c0 + (min(walk.end, walk.first + walk.rounds) - walk.at) * kRound,
                          walk.start + walk.slots);
  if (kv == 0u && group_at == 0u && walk.at == walk.first && tid == 0u && count != 0u &&
      (uint64_t)c.lengths[seq] + count > c.capacity)
    report_device_error(a.report, kDevErrCacheFull);

  // ---- the slots that the rows see: any of them, and all
  const uint32_t t_first = min(uniform(row0 / a.group), count);
  const uint32_t t_last = min(uniform((min(row0 + RT * 16u, rows) - 1u) / a.group) + 1u, count);
  uint32_t any_lo = 0u, any_hi = 0u, all_lo = 0u, all_hi = 0u;
  if (t_first < t_last) {
    seen_slots(length, t_first, c.capacity, a.window, any_lo, all_hi);
    seen_slots(length, t_last - 1u, c.capacity, a.window, all_lo, any_hi);
  }
  const uint32_t hi = min(c1, any_hi);
  const uint32_t first = c0 + wave * T::kSlots;

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

  // ---- the rows' queries, as B operands, into LDS; the first keys are under
  // way meanwhile (loads return in order, so the queries' go first)
  uint32_t page = page_of(first);
  uint32_t next_page = page_of(first + kRound);
  constexpr uint32_t kValues = S::kWide ? 4 : 8;
  constexpr uint32_t kMine = (S::kItems + kThreads - 1) / kThreads;
  float x[kMine][kValues];
  const float scale = a.scale * kLog2e;
#pragma unroll
  for (uint32_t k = 0; k < kMine; ++k) {
    const uint32_t i = tid + k * kThreads, l = i & 63u;
    const uint32_t r = row0 + i / (S::kSteps * 64u) * 16u + (l & 15u), t = r / a.group;
    const uint32_t d0 = (i / 64u % S::kSteps * 4u + (l >> 4)) * kValues;
    const bool there = i < S::kItems && r < rows && t < count && d0 < dim;
    const float* src = a.q + ((size_t)seq * a.tokens + t) * a.q_token_stride +
                       (kv * a.group + (r - t * a.group)) * a.q_head_stride + d0;
#pragma unroll
    for (uint32_t v = 0; v < kValues; ++v) x[k][v] = there ? src[v] : 0.0f;
  }
  uint32_t row = row_of(first, page);
  load_keys(row);
  page = next_page;
  if constexpr (T::kShift != 0.0f) {
    if (tid < RT * 16u) row_top[tid] = 0u;
    __syncthreads();
  }
#pragma unroll
  for (uint32_t k = 0; k < kMine; ++k) {
    float top = 0.0f;
#pragma unroll
    for (uint32_t v = 0; v < kValues; ++v) {
      x[k][v] *= scale;
      // (as integers, what is no number is the largest of them)
      if (T::kShift != 0.0f)
        top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(x[k][v]) & 0x7fffffffu));
    }
    if constexpr (T::kShift != 0.0f) {
      const uint32_t i = tid + k * kThreads;
      if (i < S::kItems)
        atomicMax(&row_top[i / (S::kSteps * 64u) * 16u + (i & 15u)], __float_as_uint(top));
    }
  }
  // the rows' powers of two, 2^14 at the largest value; 1 where it is no number
  const auto power = [&](uint32_t r) {
    const uint32_t e = row_top[r] >> 23;
    return e == 255u ? 1.0f : __uint_as_float((268u - max(e, 16u)) << 23);
  };
  if constexpr (T::kShift != 0.0f) __syncthreads();
#pragma unroll
  for (uint32_t k = 0; k < kMine; ++k) {
    const uint32_t i = tid + k * kThreads;
    if (i >= S::kItems) break;
    if constexpr (S::kWide) {
      u32x4 w;
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v) w[v] = __float_as_uint(x[k][v]);
      q_lds[i] = w;
    } else {
      u32x4 w[T::kPieces];
      const float s = T::kShift != 0.0f ? power(i / (S::kSteps * 64u) * 16u + (i & 15u)) : 1.0f;
#pragma unroll
      for (uint32_t v = 0; v < 8; v += 2) {
        uint32_t p[T::kPieces];
        T::split(x[k][v] * s, x[k][v + 1] * s, p);
#pragma unroll
        for (uint32_t q = 0; q < T::kPieces; ++q) w[q][v / 2] = p[q];
      }
#pragma unroll
      for (uint32_t q = 0; q < T::kPieces; ++q) q_lds[q * S::kItems + i] = w[q];
    }
  }
  __syncthreads();

  // ---- the lane's rows, and their slots
  uint32_t begin[RT], end[RT];
  float unscale[RT], m[RT], l[RT];
  float* score_row[RT];
  uint32_t any = 0u;  // bit i: row i sees a slot of the lane's
  f32x4 out[RT][S::kTiles];
#pragma unroll
  for (uint32_t i = 0; i < RT; ++i) {
    const uint32_t r = row0 + i * 16u + n, t = r / a.group;
    begin[i] = end[i] = 0u;
    score_row[i] = nullptr;
    if (r < rows && t < count) {
      seen_slots(length, t, c.capacity, a.window, begin[i], end[i]);
      if (o.scores)
        score_row[i] = o.scores + (((size_t)seq * c.kv_heads + kv) * rows + r) * o.score_stride;
    }
    unscale[i] = 1.0f;
    if constexpr (T::kShift != 0.0f)
      unscale[i] = __uint_as_float((254u << 23) - __float_as_uint(power(i * 16u + n)));
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (uint32_t d = 0; d < S::kTiles; ++d) out[i][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // out^T += V^T p^T with the values in `value`
  const auto add_values = [&](const float (&p)[RT][S::kRows]) {
    if constexpr (S::kWide) {
#pragma unroll
      for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
        for (uint32_t i = 0; i < S::kRows; ++i)
#pragma unroll
          for (uint32_t d = 0; d < S::kEach; ++d)
#pragma unroll
            for (uint32_t r = 0; r < RT; ++r)
              out[r][u * S::kEach + d] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __uint_as_float(value[i][u][d]), p[r][i], out[r][u * S::kEach + d], 0, 0, 0);
    } else {
      u32x4 b[RT][T::kPieces];
#pragma unroll
      for (uint32_t r = 0; r < RT; ++r)
#pragma unroll
        for (uint32_t i = 0; i < 8; i += 2) {
          uint32_t w[T::kPieces];
          T::split(p[r][i], p[r][i + 1], w);
#pragma unroll
          for (uint32_t k = 0; k < T::kPieces; ++k) b[r][k][i / 2] = w[k];
        }
#pragma unroll
      for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
        for (uint32_t d = 0; d < S::kEach; ++d) {
          u32x4 v;
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            v[i] = perm(value[2 * i + 1][u][d / 2], value[2 * i][u][d / 2], d & 1 ? kHighs : kLows);
#pragma unroll
          for (uint32_t k = 0; k < T::kPieces; ++k)
#pragma unroll
            for (uint32_t r = 0; r < RT; ++r)
              out[r][u * S::kEach + d] = T::mfma(v, b[r][k], out[r][u * S::kEach + d]);
        }
    }
  };

  for (uint32_t base = first; base < hi; base += kRound) {
    const uint32_t there = (uint32_t)__builtin_amdgcn_ballot_w64(row != kNone);
    next_page = page_of(base + 2u * kRound);
    load_values(row);
    __builtin_amdgcn_sched_barrier(0);
    // ---- scores
    // (the queries are read each time: kept across tiles, they would not leave registers for
    // the tile)
    uint32_t q_at = lane;
    asm volatile("" : "+v"(q_at));
    f32x4 sum[RT][S::kSubs];
#pragma unroll
    for (uint32_t r = 0; r < RT; ++r) {
      if constexpr (S::kWide) {
        f32x4 even{0, 0, 0, 0}, odd{0, 0, 0, 0};
#pragma unroll
        for (uint32_t k = 0; k < S::kSteps; ++k) {
          const u32x4 q = q_lds[(r * S::kSteps + k) * 64u + q_at];
#pragma unroll
          for (uint32_t e = 0; e < 4; e += 2) {
            even = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(key[0][k][e]),
                                                        __uint_as_float(q[e]), even, 0, 0, 0);
            odd = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(key[0][k][e + 1]),
                                                       __uint_as_float(q[e + 1]), odd, 0, 0, 0);
          }
        }
        sum[r][0] = even + odd;
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
            const u32x4 q = q_lds[w * S::kItems + (r * S::kSteps + k) * 64u + q_at];
#pragma unroll
            for (uint32_t s = 0; s < S::kSubs; ++s)
              piece[s][w] = T::mfma(key[s][k], q, piece[s][w]);
          }
#pragma unroll
        for (uint32_t s = 0; s < S::kSubs; ++s) {
          sum[r][s] = piece[s][T::kPieces - 1];
#pragma unroll
          for (int k = (int)T::kPieces - 2; k >= 0; --k) sum[r][s] += piece[s][k];
          sum[r][s] *= unscale[r];
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- the next tile's keys
    row = row_of(base + kRound, page);
    page = next_page;
    load_keys(row);  // (behind the last tile too: a condition would hold both sets of registers)
    __builtin_amdgcn_sched_barrier(0);
    // ---- p
    float p[RT][S::kRows];
    uint32_t seen[RT];  // bits 0..3 and 16..19: the row sees the lane's slots
#pragma unroll
    for (uint32_t r = 0; r < RT; ++r) {
      float top = -INFINITY;
      seen[r] = (slot_bits(begin[r], end[r], base) & there) >> (4u * j) &
                (T::kSlots == 32u ? 0x000f000fu : 0xfu);
#pragma unroll
      for (uint32_t i = 0; i < S::kRows; ++i) {
        p[r][i] = seen[r] >> (i / 4u * 16u + i % 4u) & 1u ? sum[r][i / 4u][i % 4u] : -INFINITY;
        top = fmaxf(top, p[r][i]);
      }
      any |= seen[r] ? 1u << r : 0u;
      if (score_row[r]) {
#pragma unroll
        for (uint32_t s = 0; s < S::kSubs; ++s) {
          const uint32_t slot = base + s * 16u + j * 4u;
          if (slot < o.score_stride)
            *reinterpret_cast<float4*>(score_row[r] + slot) =
                make_float4(p[r][4 * s], p[r][4 * s + 1], p[r][4 * s + 2], p[r][4 * s + 3]);
        }
      }
      const float now = fmaxf(m[r], columns_max(top));
      const float from = now == -INFINITY ? 0.0f : now - T::kShift;
      if (__builtin_amdgcn_ballot_w64(now > m[r])) {
        const float keep = m[r] == -INFINITY ? 0.0f : exp2_of(m[r] - now);
        l[r] *= keep;
#pragma unroll
        for (uint32_t d = 0; d < S::kTiles; ++d) out[r][d] *= keep;
        m[r] = now;
      }
#pragma unroll
      for (uint32_t i = 0; i < S::kRows; ++i) {
        p[r][i] = exp2_of(p[r][i] - from);  // (0 where not seen)
        l[r] += p[r][i];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- out
    // A slot that no row sees may hold anything: its values are taken as 0.  So
    // are those of a slot with a value that is no finite number, where not all
    // rows see it, for 0 times that would reach the others; the rows that do
    // see it are none from then on.
    constexpr uint32_t kAll = T::kSlots == 32u ? 0xffffffffu : 0xffffu;
    if ((slot_bits(all_lo, all_hi, base) & there & kAll) != kAll) {
      const uint32_t used = (slot_bits(any_lo, any_hi, base) & there) >> (4u * j);
      uint32_t lost = 0u;
#pragma unroll
      for (uint32_t i = 0; i < S::kRows; ++i) {
        const uint32_t at = i / 4u * 16u + i % 4u;
        bool use = (used >> at & 1u) != 0u;
        uint32_t odd = 0u;
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t w = 0; w < S::kWords; ++w)
            odd |= (value[i][u][w] & T::kExponent) + T::kUnit;
        const uint64_t odds = __builtin_amdgcn_ballot_w64((odd & T::kCarry) != 0u);
        if ((odds >> (16u * j) & 0xffffu) != 0u) {  // (16 lanes have the slot's values)
#pragma unroll
          for (uint32_t r = 0; r < RT; ++r) lost |= (seen[r] >> at & 1u) << r;
          use = false;
        }
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t w = 0; w < S::kWords; ++w) value[i][u][w] = use ? value[i][u][w] : 0u;
      }
      if (__builtin_amdgcn_ballot_w64(lost != 0u)) {
        lost |= __shfl_xor(lost, 16, 64);
        lost |= __shfl_xor(lost, 32, 64);
#pragma unroll
        for (uint32_t r = 0; r < RT; ++r) {
          const float none = lost >> r & 1u ? NAN : 0.0f;
#pragma unroll
          for (uint32_t d = 0; d < S::kTiles; ++d) out[r][d] += none;
        }
      }
    }
    add_values(p);
  }
  if (bad) report_device_error(a.report, kDevErrCachePage);

  // ---- the waves join
  // A row with slots whose scores are all -inf (0 / 0 in the end) has l = -1
  // until it meets one that is not; a row without slots has l = 0.
  any |= __shfl_xor(any, 16, 64);
  any |= __shfl_xor(any, 32, 64);
#pragma unroll
  for (uint32_t r = 0; r < RT; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
    if (l[r] == 0.0f && m[r] == -INFINITY && (any >> r & 1u) != 0u) l[r] = -1.0f;
    if (j == 0u) {
      row_m[wave][r * 16u + n] = m[r];
      row_l[wave][r * 16u + n] = l[r];
    }
  }
  // the sequence's shares, and this one among them
  const uint32_t shares =
      uniform((walk.first + walk.rounds - 1u) / walk.each) - uniform(walk.first / walk.each) + 1u;
  float* join = reinterpret_cast<float*>(shared) + ((wave % (WAVES / 2u)) * 16u + n) * S::kOutStride;
  const auto place = [&](uint32_t u, uint32_t w) {
    return reinterpret_cast<float4*>(join + (u * 16u + j * 4u + w) * S::kEach);
  };
#pragma unroll
  for (uint32_t r = 0; r < RT; ++r) {
    __syncthreads();  // (the queries, or the last tile's outputs, are no longer read)
    float top = -INFINITY;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) top = fmaxf(top, row_m[w][r * 16u + n]);
    const float mine = m[r] == -INFINITY ? 0.0f : exp2_of(m[r] - top);
#pragma unroll
    for (uint32_t d = 0; d < S::kTiles; ++d) out[r][d] *= mine;
    // the second half of the waves hands its outputs to the first, which hands its sums to all
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half) {
      if ((wave >= WAVES / 2u) == (half == 0u)) {
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t w = 0; w < 4; ++w)
#pragma unroll
            for (uint32_t d = 0; d < S::kEach; d += 4) {
              f32x4* t = &out[r][u * S::kEach + d];
              float4* to = place(u, w) + d / 4u;
              if (half == 1u) {
                const float4 v = *to;
                t[0][w] += v.x, t[1][w] += v.y, t[2][w] += v.z, t[3][w] += v.w;
              }
              *to = make_float4(t[0][w], t[1][w], t[2][w], t[3][w]);
            }
      }
      __syncthreads();
    }
    constexpr uint32_t kRowThreads = kThreads / 16u;
    const uint32_t jr = tid / kRowThreads, jn = tid % kRowThreads, out_row = row0 + r * 16u + jr;
    if (out_row < rows) {
      float2 st = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (uint32_t w = 0; w < WAVES; ++w)
        st = joined(st, make_float2(row_m[w][r * 16u + jr], row_l[w][r * 16u + jr]));
      const size_t head = (size_t)kv * rows + out_row;
      const size_t part_row = (size_t)(share + seq) * c.kv_heads * rows + head;
      const uint32_t t = out_row / a.group, h = kv * a.group + (out_row - t * a.group);
      if (jn == 0u) {
        if (shares != 1u) o.part_stats[part_row] = st;
        else if (o.stats) o.stats[(size_t)seq * c.kv_heads * rows + head] = row_stats(st, T::kShift);
      }
      float* to = shares == 1u ? a.out + (((size_t)seq * a.tokens + t) * a.heads + h) * dim
                               : o.part_out + part_row * dim;
      const float times = shares == 1u ? row_times(st) : 1.0f;
      for (uint32_t d = jn * 4u; d < dim; d += 4u * kRowThreads) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (st.y != 0.0f) {  // (a row that sees nothing has no part in what its columns hold)
#pragma unroll
          for (uint32_t w = 0; w < WAVES / 2u; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(
                reinterpret_cast<const float*>(shared) + (w * 16u + jr) * S::kOutStride + d);
            v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
          }
          v.x *= times, v.y *= times, v.z *= times, v.w *= times;
        }
        *reinterpret_cast<float4*>(to + d) = v;
      }
    }
  }
  (void)last_share;
  next_walk(a, kRound, walk);
  if (walk.at < walk.end) __syncthreads();  // (the outputs are no longer read)
  }
}

template <typename T, uint32_t DC, bool FULL, uint32_t RT, uint32_t WAVES, uint32_t PER_SIMD>
hipError_t launch_mfma(const AttentionArgs& a, Outputs o, hipStream_t s) {
  using S = Shape<T, DC, RT, WAVES>;
  static const hipError_t attr = hipFuncSetAttribute(
      reinterpret_cast<const void*>(&attention_mfma<T, DC, FULL, RT, WAVES, PER_SIMD>),
      hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::kShared);
  if (attr != hipSuccess) return attr;
  const uint32_t tiles = row_tiles(a.tokens, a.group);
  o.tile_groups = (tiles + RT - 1u) / RT;
  o.round = T::kSlots * WAVES;
  o.shift = T::kShift;
  o.shares = shares_for(a.cache, o.tile_groups, PER_SIMD * 4u / WAVES, o.round);
  const uint32_t units = o.shares * a.cache.kv_heads;
  const uint32_t blocks = o.tile_groups == 1u ? units : (units + 7u) / 8u * 8u * o.tile_groups;
  attention_mfma<T, DC, FULL, RT, WAVES, PER_SIMD><<<blocks, 64 * WAVES, S::kShared, s>>>(a, o);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || o.shares == 1u) return e;
  return launch_attention_join(a, o, s);
}

// The row tiles a wave takes, so that the cache is read for several at once:
// as many as leave registers for two waves a SIMD beside the tile; two of the
// largest heads, as one wave of twice the registers.
template <typename T, uint32_t DC, bool FULL>
hipError_t launch_rows(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  const uint32_t tiles = row_tiles(a.tokens, a.group);
  if (tiles == 1u) return launch_mfma<T, DC, FULL, 1, 8, 2>(a, o, s);
  if constexpr (DC == 256) return launch_mfma<T, DC, FULL, 1, 8, 2>(a, o, s);
  if constexpr (DC == 64)
    if (tiles == 3u || tiles > 4u) return launch_mfma<T, DC, FULL, 3, 8, 2>(a, o, s);
  return launch_mfma<T, DC, FULL, 2, 8, 2>(a, o, s);
}

template <typename T>
hipError_t launch_type(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  switch (a.cache.head_dim) {
    case 64: return launch_rows<T, 64, true>(a, o, s);
    case 128: return launch_rows<T, 128, true>(a, o, s);
    case 256: return launch_rows<T, 256, true>(a, o, s);
    default: break;
  }
  if (a.cache.head_dim < 64u) return launch_mfma<T, 64, false, 1, 8, 2>(a, o, s);
  if (a.cache.head_dim < 128u) return launch_mfma<T, 128, false, 1, 8, 2>(a, o, s);
  return launch_mfma<T, 256, false, 1, 8, 2>(a, o, s);
}

}  // namespace attn
}  // namespace sihip
