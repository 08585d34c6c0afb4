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
// and the last 8 (exact); for F16 two of 11 bits, 22 of the 24, for a third
// would cost half as many products again.  F16's least step, 2^-24, sets how far
// these reach: q is scaled by a power of two that puts its row's largest value at
// 2^14, and its second piece, whose sum is one of its own, by 2^12 more, so that
// values down to 2^-28 of the largest have their 22 bits, and smaller ones are
// good to 2^-51 of it; p is taken times 2^14, both pieces, for they share their sum:
// 22 bits down to 2^-17, and smaller ones good to 2^-39 of the row's largest.  An
// f32 cache takes the f32 instructions.  Products and sums are f32.
//
// A wave has up to 128 values of a head.  Larger heads are a team's.  For one
// row tile two waves take a half each, of the keys and of the values: they add
// their halves' scores through LDS, and both go on with the sums.  For several
// (kBySlots) the p of a row would be worked out by every wave of the team: so
// four waves take a sixteen of slots each, with whole keys, agree on the rows'
// maxima, put their p, in pieces, into LDS, and take a quarter of the values of
// all their slots.  The queries of one row tile stay in registers; those of
// several are in LDS.
//
// The slots of all sequences, in rounds of the tiles of a workgroup's teams,
// are dealt to the workgroups of a kv head in equal shares, one after another:
// a share may end one sequence and begin others.  A sequence inside one share is
// written at once; the sums of one that lies in several are joined in the order
// of the shares.
//
// Measured, calls back to back over caches that are not in the L2: one token
// over 131,071 slots of 4 heads of 256 in BF16 95 us for 537 MB, 5.7 TB/s
// (6.1 in this kernel), bound by memory; one token a sequence of 24 in F32,
// 427 MB, 102 us with the weights, of which this kernel has 89; eight drafted
// tokens a sequence of four, 183 MB, 58 us, bound by the arithmetic of a round
// and by what comes before its loads and behind the last (4 us each); one
// token over 1021 slots of 8 heads of 128, 4.2 MB, 12.5 us: the launch and a
// chain of dependent reads (lengths, page numbers, rows, other shares' sums).
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
  static constexpr float kQueryRest = 1.0f;  // what a query's last piece is held times
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  // The pieces of x and y, in the halves of one word each.  What is no number
  // is its first piece alone.
  template <bool QUERY>
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
  static constexpr float kQueryRest = 0x1p12f;  // (a rest of at most 2^3)
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  template <bool QUERY>
  static __device__ __forceinline__ void split(float x, float y, uint32_t (&w)[kPieces]) {
    const float rest = QUERY ? kQueryRest : 1.0f;
    const _Float16 a = (_Float16)x, b = (_Float16)y;
    const _Float16 c = (_Float16)((x - (float)a) * rest), d = (_Float16)((y - (float)b) * rest);
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
  static constexpr float kShift = 0.0f, kQueryRest = 1.0f;
  static constexpr uint32_t kExponent = 0x7f800000u, kUnit = 0x00800000u, kCarry = 0x80000000u;
};

// DW: values of a head that a wave has; VS: waves of a team, which have a head
// together; RT: row tiles a wave.
template <typename T, uint32_t DW, uint32_t VS, uint32_t RT>
struct Shape {
  static constexpr uint32_t kWaves = 8, kTeams = kWaves / VS;
  static constexpr bool kWide = T::kBytes == 4;               // f32 instructions
  static constexpr uint32_t kSubs = T::kSlots / 16;           // score tiles of 16 slots
  static constexpr uint32_t kSteps = DW / (kWide ? 16 : 32);  // 16-byte pieces of a key a lane
  static constexpr uint32_t kValues = kWide ? 4 : 8;          // values of such a piece
  static constexpr uint32_t kRows = kWide ? 4 : 8;            // value rows a lane
  // values of a row that a lane loads at once, and how often
  static constexpr uint32_t kEach = kWide ? 4 : DW >= 128 ? 8 : 4;
  static constexpr uint32_t kPasses = DW / (16 * kEach);
  static constexpr uint32_t kWords = kEach * T::kBytes / 4;
  static constexpr uint32_t kTiles = DW / 16;  // of the wave's output
  static constexpr bool kInRegisters = RT == 1;  // the queries
  // how a team shares the scores: a sixteen of its slots a wave, or a part of the head
  static constexpr bool kBySlots = VS == 4;
  static constexpr uint32_t kOwnSubs = kBySlots ? 1 : kSubs;  // score tiles of a wave
  static constexpr uint32_t kOwnRows = 4 * kOwnSubs;          // and a lane's slots in them
  static constexpr uint32_t kKeySteps = kBySlots ? VS * kSteps : kSteps;
  static constexpr uint32_t kTeamTiles = kBySlots ? VS / kSubs : 1;
  static constexpr uint32_t kTeamSlots = kTeamTiles * T::kSlots, kRound = kTeams * kTeamSlots;
  static constexpr uint32_t kSets = kBySlots ? kWaves : kTeams;  // of maxima and sums
  static constexpr uint32_t kItems = VS * RT * kSteps * 64;  // 16-byte pieces of the queries
  static constexpr uint32_t kQueryBytes = kInRegisters ? 0 : T::kPieces * kItems * 16;
  // what the waves of a team exchange: p, or halves of scores
  static constexpr uint32_t kHalves = kWaves * kSubs * 64 * 16;
  static constexpr uint32_t kExchangeBytes =
      VS == 1 ? 0 : kBySlots ? kTeams * kTeamTiles * RT * T::kPieces * 64 * 16 : 2 * kHalves;
  static constexpr uint32_t kOutStride = DW * VS + 4;  // words of a row of the join
  // row tiles joined at once
  static constexpr uint32_t kOutTiles = RT * kTeams * 16 * kOutStride * 4 <= 144 * 1024 ? RT : 1;
  static constexpr uint32_t kOutBytes = kOutTiles * kTeams * 16 * kOutStride * 4;
  static constexpr uint32_t kTileBytes = kQueryBytes + kExchangeBytes;
  static constexpr uint32_t kShared = kTileBytes > kOutBytes ? kTileBytes : kOutBytes;
};

// The workgroup's waves meet, what they wrote to LDS in place.  Loads from
// memory go on.
__device__ __forceinline__ void exchange_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Blocks of the row tiles of one share and head follow each other on one XCD
// (blocks are dealt to the eight in turn), so its L2 serves them the same rows.
__device__ __forceinline__ void block_work(const Outputs& o, uint32_t& unit, uint32_t& tile) {
  const uint32_t b = blockIdx.x;
  if (o.tile_groups == 1u) {
    unit = b;
    tile = 0u;
    return;
  }
  const uint32_t xcd = b & 7u, i = b >> 3, row = o.by_tiles.of(i);
  tile = i - row * o.tile_groups;
  unit = row * 8u + xcd;
}

// FAST: heads of DW * VS values on pages of whole sixteens of slots, so that the
// slots of a score tile lie one after another and addresses are scalars.
// ONCE: no other workgroup reads the values, which then pass the caches by.
template <typename T, uint32_t DW, uint32_t VS, bool FAST, uint32_t RT, bool ONCE>
__global__ __launch_bounds__(512, 2) void attention_mfma(AttentionArgs a, Outputs o) {
  using S = Shape<T, DW, VS, RT>;
  constexpr uint32_t kThreads = 64 * S::kWaves, kRound = S::kRound;
  extern __shared__ __attribute__((aligned(16))) uint8_t shared[];
  __shared__ float row_m[S::kSets][RT * 16], row_l[S::kSets][RT * 16];
  __shared__ float2 row_sum[RT * 16];
  __shared__ uint32_t row_top[RT * 16], last_share;
  const CacheView& c = a.cache;
  const uint32_t wave = uniform(threadIdx.x / 64u), team = wave / VS, half = wave % VS;
  const uint32_t dim = FAST ? DW * VS : c.head_dim;
  const uint32_t row_bytes = dim * T::kBytes;
  const uint32_t rows = a.tokens * a.group;
  const uint8_t* keys = static_cast<const uint8_t*>(c.keys);
  const uint8_t* values = static_cast<const uint8_t*>(c.values);
  u32x4* q_lds = reinterpret_cast<u32x4*>(shared);

  uint32_t unit, group_at;
  block_work(o, unit, group_at);
  if (unit >= o.shares * c.kv_heads) return;
  const uint32_t share = o.by_heads.of(unit), kv = unit - share * c.kv_heads;
  const uint32_t row0 = group_at * (RT * 16u);
  Walk walk = first_walk<kRound>(a, o, share);

  while (walk.at < walk.end) {
    // (afresh for each sequence: what follows from the thread's number would
    // otherwise stay in registers through the tiles)
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const uint32_t lane = tid & 63u, n = lane & 15u, j = lane >> 4;
    const uint32_t seq = walk.seq, count = walk.span.count, length = walk.span.length;
    const uint32_t c0 = walk.span.start + (walk.at - walk.first) * kRound;
    const uint32_t c1 = min(c0 + (min(walk.end, walk.first + walk.span.rounds) - walk.at) * kRound,
                            walk.span.start + walk.span.slots);
    // the sequence lies in this share
    const bool alone = walk.first >= walk.begin && walk.first + walk.span.rounds <= walk.limit;

    if (kv == 0u && group_at == 0u && walk.at == walk.first && tid == 0u && count != 0u &&
        (uint64_t)c.lengths[seq] + count > c.capacity)
      report_device_error(a.report, kDevErrCacheFull);

    // ---- the slots that the rows see: any of them, and all
    const uint32_t t_first = min(o.by_group.of(row0), count);
    const uint32_t t_last = min(o.by_group.of(min(row0 + RT * 16u, rows) - 1u) + 1u, count);
    uint32_t any_lo = 0u, any_hi = 0u, all_lo = 0u, all_hi = 0u;
    if (t_first < t_last) {
      seen_slots(length, t_first, c.capacity, a.window, any_lo, all_hi);
      seen_slots(length, t_last - 1u, c.capacity, a.window, all_lo, any_hi);
    }
    const uint32_t hi = min(c1, any_hi);
    const uint32_t first = c0 + team * S::kTeamSlots;

    // Where a tile's rows lie, in two steps, so that the page numbers are there
    // before the rows are wanted.  FAST: of each score tile; else lane l has slot
    // l % kSlots.
    constexpr uint32_t kPlaces = FAST ? S::kTeamTiles * S::kSubs : 1;
    struct Place {
      uint32_t at[kPlaces];
    };
    const uint32_t* table = c.table + (size_t)seq * c.max_pages;
    uint32_t bad = 0u;  // the end of the last slots whose page lies beyond the pool
    const auto pages_of = [&](uint32_t base) {
      Place p;
      if constexpr (FAST) {
#pragma unroll
        for (uint32_t s = 0; s < kPlaces; ++s) {
          const uint32_t slot = base + s * 16u;
          p.at[s] = slot < hi ? table[divided(slot, c.div_mul, c.div_shift)] : kNone;
        }
      } else {
        const uint32_t slot = base + (lane & (T::kSlots - 1u));
        p.at[0] = slot < hi ? table[divided(slot, c.div_mul, c.div_shift)] : kNone;
      }
      return p;
    };
    const auto rows_of = [&](uint32_t base, const Place& page) {
      Place p;
#pragma unroll
      for (uint32_t s = 0; s < kPlaces; ++s) {
        const uint32_t slot = base + (FAST ? s * 16u : lane & (T::kSlots - 1u));
        p.at[s] = kNone;
        if (slot < hi) {
          if (page.at[s] < c.pages)
            p.at[s] = (page.at[s] * c.kv_heads + kv) * c.page_tokens +
                      (slot - divided(slot, c.div_mul, c.div_shift) * c.page_tokens);
          else
            bad = slot + (FAST ? 16u : 1u);
        }
      }
      return p;
    };
    // The slots of tile `tile` that have a row, a bit each.  (FAST: and those behind
    // the last on its page, which no row of the queries sees.)
    const auto slots_there = [&](const Place& p, uint32_t tile) {
      if constexpr (!FAST) return (uint32_t)__builtin_amdgcn_ballot_w64(p.at[0] != kNone);
      uint32_t bits = 0u;
#pragma unroll
      for (uint32_t s = 0; s < (FAST ? S::kSubs : 1u); ++s)
        bits |= p.at[tile * S::kSubs + s] != kNone ? 0xffffu << (16u * s) : 0u;
      return bits;
    };
    // Row `from` of score tile `sub`; a slot without a row reads the pool's first
    // page, or first row, and is masked.
    const auto pointer = [&](const uint8_t* base, const Place& p, uint32_t sub, uint32_t from) {
      if constexpr (FAST) {
        const uint32_t at = p.at[sub];
        return base + (size_t)(at == kNone ? 0u : at) * row_bytes + from * row_bytes;
      } else {
        const uint32_t at = __shfl(p.at[0], sub * 16u + from, 64);
        return base + (size_t)(at == kNone ? 0u : at) * row_bytes;
      }
    };
    // (by slots: the wave's score tile in place of the first)
    const auto own_place = [&](const Place& p) {
      Place r = p;
      if constexpr (S::kBySlots)
#pragma unroll
        for (uint32_t u = 1; u < VS; ++u)
          if (half == u) r.at[0] = p.at[u];
      return r;
    };
    u32x4 key[S::kOwnSubs][S::kKeySteps];
    const auto load_keys = [&](const Place& row) {
      const Place own = own_place(row);
#pragma unroll
      for (uint32_t s = 0; s < S::kOwnSubs; ++s) {
        const uint8_t* p = pointer(keys, own, s, n);
#pragma unroll
        for (uint32_t k = 0; k < S::kKeySteps; ++k) {
          uint32_t at = (((S::kBySlots ? 0u : half * S::kSteps) + k) * 4u + j) * 16u;
          if (!FAST) at = min(at, row_bytes - 16u);  // (its query values are 0)
          key[s][k] = *reinterpret_cast<const Words4*>(p + at);
        }
      }
    };
    uint32_t value[S::kTeamTiles][S::kRows][S::kPasses][S::kWords];
    const auto load_values = [&](const Place& row, uint32_t tile) {
#pragma unroll
      for (uint32_t i = 0; i < S::kRows; ++i) {
        const uint8_t* p = pointer(values, row, tile * S::kSubs + i / 4u, j * 4u + i % 4u);
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u) {
          uint32_t at = ((half * S::kPasses + u) * 16u + n) * (S::kWords * 4u);
          if (!FAST) at = min(at, row_bytes - S::kWords * 4u);  // (its outputs are not stored)
          if constexpr (S::kWords == 4) {
            const Words4* from = reinterpret_cast<const Words4*>(p + at);
            const u32x4 w = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x) value[tile][i][u][x] = w[x];
          } else {
            const Words2* from = reinterpret_cast<const Words2*>(p + at);
            const Words2 w = ONCE ? __builtin_nontemporal_load(from) : *from;
            value[tile][i][u][0] = w.x;
            value[tile][i][u][1] = w.y;
          }
        }
      }
    };

    // ---- the rows' queries, as B operands; the first keys are under way meanwhile
    // (loads return in order, so the queries' go first)
    Place page = pages_of(first), next_page = pages_of(first + kRound);
    const float scale = a.scale * kLog2e;
    // Sixteen-byte pieces of the operands: those of the wave's half where they
    // stay in registers, else the thread's share of all.
    constexpr uint32_t kMine = S::kInRegisters ? S::kSteps : (S::kItems + kThreads - 1) / kThreads;
    const auto item = [&](uint32_t k) {  // row tile, half, step, lane: the piece's place in LDS
      return S::kInRegisters ? (half * S::kSteps + k) * 64u + lane : tid + k * kThreads;
    };
    const auto item_row = [&](uint32_t i) { return i / (VS * S::kSteps * 64u) * 16u + (i & 15u); };
    float x[kMine][S::kValues];
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
      const uint32_t i = item(k), r = row0 + item_row(i), t = o.by_group.of(r);
      const uint32_t d0 = (i / 64u % (VS * S::kSteps) * 4u + ((i & 63u) >> 4)) * S::kValues;
      const bool there = i < S::kItems && r < rows && t < count && d0 < dim;
      const float* src = a.q + ((size_t)seq * a.tokens + t) * a.q_token_stride +
                         (kv * a.group + (r - t * a.group)) * a.q_head_stride + d0;
#pragma unroll
      for (uint32_t v = 0; v < S::kValues; v += 4) {
        Floats4 f{0.0f, 0.0f, 0.0f, 0.0f};
        if (there) f = *reinterpret_cast<const Floats4*>(src + v);
        x[k][v] = f.x, x[k][v + 1] = f.y, x[k][v + 2] = f.z, x[k][v + 3] = f.w;
      }
    }
    Place row = rows_of(first, page);
    load_keys(row);
    page = next_page;
    // The largest of a row's values, as an integer (what is no number is larger
    // than all): in LDS, or of the wave's half over the lanes that have it.
    uint32_t largest = 0u;
    if (!S::kInRegisters && T::kShift != 0.0f) {
      if (tid < RT * 16u) row_top[tid] = 0u;
      exchange_barrier();
    }
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
      uint32_t top = 0u;
#pragma unroll
      for (uint32_t v = 0; v < S::kValues; ++v) {
        x[k][v] *= scale;
        top = max(top, __float_as_uint(x[k][v]) & 0x7fffffffu);
      }
      if (T::kShift != 0.0f) {
        if (S::kInRegisters) largest = max(largest, top);
        else if (item(k) < S::kItems) atomicMax(&row_top[item_row(item(k))], top);
      }
    }
    if (T::kShift != 0.0f) {
      if (S::kInRegisters) {
        largest = max(largest, (uint32_t)__shfl_xor(largest, 16, 64));
        largest = max(largest, (uint32_t)__shfl_xor(largest, 32, 64));
      } else {
        exchange_barrier();
      }
    }
    // the row's power of two, 2^14 at the largest value; 1 where that is no number
    const auto power = [&](uint32_t r) {
      const uint32_t e = (S::kInRegisters ? largest : row_top[r]) >> 23;
      return e == 255u ? 1.0f : __uint_as_float((268u - max(e, 16u)) << 23);
    };
    u32x4 query[S::kInRegisters ? S::kSteps : 1][T::kPieces];
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
      const uint32_t i = item(k);
      if (i >= S::kItems) break;
      u32x4 w[T::kPieces];
      if constexpr (S::kWide) {
#pragma unroll
        for (uint32_t v = 0; v < 4; ++v) w[0][v] = __float_as_uint(x[k][v]);
      } else {
        const float s = T::kShift != 0.0f ? power(item_row(i)) : 1.0f;
#pragma unroll
        for (uint32_t v = 0; v < 8; v += 2) {
          uint32_t p[T::kPieces];
          T::template split<true>(x[k][v] * s, x[k][v + 1] * s, p);
#pragma unroll
          for (uint32_t q = 0; q < T::kPieces; ++q) w[q][v / 2] = p[q];
        }
      }
#pragma unroll
      for (uint32_t q = 0; q < T::kPieces; ++q) {
        if constexpr (S::kInRegisters) query[k][q] = w[q];
        else q_lds[q * S::kItems + i] = w[q];
      }
    }
    if (!S::kInRegisters) exchange_barrier();
#pragma unroll
    for (uint32_t u = 0; u < S::kTeamTiles; ++u) load_values(row, u);

    // ---- the lane's rows, and their slots
    uint32_t begin[RT], end[RT];
    float unscale[RT], m[RT], l[RT];
    float* score_row[RT];
    uint32_t any = 0u;  // bit i: row i sees a slot of the lane's
    f32x4 out[RT][S::kTiles];
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
      const uint32_t r = row0 + i * 16u + n, t = o.by_group.of(r);
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

    // out^T += V^T p^T with a tile's values
    const auto add_values = [&](uint32_t tile, const u32x4 (&b)[RT][T::kPieces]) {
      const auto& v = value[tile];
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
                    __uint_as_float(v[i][u][d]), __uint_as_float(b[r][0][i]),
                    out[r][u * S::kEach + d], 0, 0, 0);
      } else {
        // (four sums at a time, so that none waits for the one before)
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t d = 0; d < S::kEach; d += 4) {
            u32x4 x[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i)
                x[e][i] = perm(v[2 * i + 1][u][(d + e) / 2], v[2 * i][u][(d + e) / 2],
                               e & 1 ? kHighs : kLows);
#pragma unroll
            for (uint32_t r = 0; r < RT; ++r)
#pragma unroll
              for (uint32_t k = 0; k < T::kPieces; ++k)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                  f32x4& acc = out[r][u * S::kEach + d + e];
                  acc = T::mfma(x[e], b[r][k], acc);
                }
          }
      }
    };
    // p of a lane's slots, as the words of the B operands that they make
    const auto operands = [&](const float (&p)[S::kOwnRows], uint32_t (&b)[T::kPieces][4]) {
      if constexpr (S::kWide) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) b[0][i] = __float_as_uint(p[i]);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < S::kOwnRows; i += 2) {
          uint32_t w[T::kPieces];
          T::template split<false>(p[i], p[i + 1], w);
#pragma unroll
          for (uint32_t k = 0; k < T::kPieces; ++k) b[k][i / 2] = w[k];
        }
      }
    };
    // A slot that no row sees may hold anything: its values are taken as 0.  So
    // are those of a slot with a value that is no finite number, where not all
    // rows see it, for 0 times that would reach the others; the rows that do
    // see it are none from then on.
    const auto clear_unseen = [&](uint32_t tile, uint32_t base, uint32_t there) {
      constexpr uint32_t kAll = T::kSlots == 32u ? 0xffffffffu : 0xffffu;
      if ((slot_bits(all_lo, all_hi, base) & there & kAll) == kAll) return;
      auto& v = value[tile];
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
          for (uint32_t w = 0; w < S::kWords; ++w) odd |= (v[i][u][w] & T::kExponent) + T::kUnit;
        const uint64_t odds = __builtin_amdgcn_ballot_w64((odd & T::kCarry) != 0u);
        if ((odds >> (16u * j) & 0xffffu) != 0u) {  // (16 lanes have the slot's values)
#pragma unroll
          for (uint32_t r = 0; r < RT; ++r) {
            const uint32_t seen = (slot_bits(begin[r], end[r], base) & there) >> (4u * j);
            lost |= (seen >> at & 1u) << r;
          }
          use = false;
        }
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t w = 0; w < S::kWords; ++w) v[i][u][w] = use ? v[i][u][w] : 0u;
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
    };

    // (a team without slots in the last round goes through it: its waves, and the
    // others', meet at the exchange)
    uint32_t turn = 0u;
    for (uint32_t at = c0; at < hi; at += kRound) {
      const uint32_t team_base = at + team * S::kTeamSlots;
      const uint32_t base = team_base + (S::kBySlots ? half * 16u : 0u);  // of the wave's scores
      uint32_t there[S::kTeamTiles];
#pragma unroll
      for (uint32_t u = 0; u < S::kTeamTiles; ++u) there[u] = slots_there(row, u);
      uint32_t own_there = there[0];
      if constexpr (S::kBySlots) own_there = own_place(row).at[0] != kNone ? 0xffffu : 0u;
      next_page = pages_of(team_base + 2u * kRound);
      // ---- scores
      f32x4 sum[RT][S::kOwnSubs];
      // (queries in LDS are read for each tile: kept across tiles, they would not leave
      // registers for it; a step's are under way while the one before is multiplied)
      uint32_t q_at = (S::kBySlots ? 0u : half * S::kSteps * 64u) + lane;
      asm volatile("" : "+v"(q_at));
      const auto read_query = [&](uint32_t i, u32x4(&q)[T::kPieces]) {
        if constexpr (!S::kInRegisters)
#pragma unroll
          for (uint32_t w = 0; w < T::kPieces; ++w) q[w] = q_lds[w * S::kItems + i * 64u + q_at];
        else
#pragma unroll
          for (uint32_t w = 0; w < T::kPieces; ++w) q[w] = query[i][w];
      };
      u32x4 q[2][T::kPieces];
      read_query(0u, q[0]);
#pragma unroll
      for (uint32_t r = 0; r < RT; ++r) {
        // sums that do not wait for each other: two of the f32 instructions, one a piece else
        constexpr uint32_t kSums = S::kWide ? 2 : T::kPieces;
        f32x4 piece[S::kOwnSubs][kSums];
#pragma unroll
        for (uint32_t s = 0; s < S::kOwnSubs; ++s)
#pragma unroll
          for (uint32_t k = 0; k < kSums; ++k) piece[s][k] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (uint32_t k = 0; k < S::kKeySteps; ++k) {
          const uint32_t i = r * S::kKeySteps + k;
          if (i + 1u < RT * S::kKeySteps) read_query(i + 1u, q[(i + 1u) & 1u]);
          if (!S::kInRegisters) __builtin_amdgcn_sched_barrier(0);
          const auto& now = q[i & 1u];
          if constexpr (S::kWide) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
              piece[0][e & 1u] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __uint_as_float(key[0][k][e]), __uint_as_float(now[0][e]), piece[0][e & 1u], 0,
                  0, 0);
          } else {
#pragma unroll
            for (uint32_t w = 0; w < T::kPieces; ++w)
#pragma unroll
              for (uint32_t s = 0; s < S::kOwnSubs; ++s)
                piece[s][w] = T::mfma(key[s][k], now[w], piece[s][w]);
          }
        }
#pragma unroll
        for (uint32_t s = 0; s < S::kOwnSubs; ++s) {
          sum[r][s] = piece[s][kSums - 1];
          if (T::kQueryRest != 1.0f) sum[r][s] *= 1.0f / T::kQueryRest;
#pragma unroll
          for (int k = (int)kSums - 2; k >= 0; --k) sum[r][s] += piece[s][k];
          if (T::kShift != 0.0f) sum[r][s] *= unscale[r];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // ---- the next tile's keys
      row = rows_of(team_base + kRound, page);
      page = next_page;
      load_keys(row);  // (behind the last tile too: a condition would hold both sets of registers)
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (VS > 1 && !S::kBySlots) {
        // ---- the other half's scores: both waves add the first half's to the second's
        f32x4* place = reinterpret_cast<f32x4*>(shared + S::kQueryBytes) +
                       (turn & 1u) * (S::kHalves / 16u);
#pragma unroll
        for (uint32_t s = 0; s < S::kSubs; ++s)
          place[(wave * S::kSubs + s) * 64u + lane] = sum[0][s];
        exchange_barrier();
#pragma unroll
        for (uint32_t s = 0; s < S::kSubs; ++s)
          sum[0][s] += place[((wave ^ 1u) * S::kSubs + s) * 64u + lane];
        ++turn;
      }
      // ---- p
      float p[RT][S::kOwnRows], now[RT];
#pragma unroll
      for (uint32_t r = 0; r < RT; ++r) {
        // bits 0..3 and 16..19: the row sees the lane's slots
        const uint32_t seen = (slot_bits(begin[r], end[r], base) & own_there) >> (4u * j) &
                              (S::kOwnSubs == 2u ? 0x000f000fu : 0xfu);
        float top = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < S::kOwnRows; ++i) {
          p[r][i] = seen >> (i / 4u * 16u + i % 4u) & 1u ? sum[r][i / 4u][i % 4u] : -INFINITY;
          top = fmaxf(top, p[r][i]);
        }
        any |= seen ? 1u << r : 0u;
        if (score_row[r] && (S::kBySlots || half == 0u)) {
#pragma unroll
          for (uint32_t s = 0; s < S::kOwnSubs; ++s) {
            const uint32_t slot = base + s * 16u + j * 4u;
            if (slot < o.score_stride)
              *reinterpret_cast<float4*>(score_row[r] + slot) =
                  make_float4(p[r][4 * s], p[r][4 * s + 1], p[r][4 * s + 2], p[r][4 * s + 3]);
          }
        }
        now[r] = columns_max(top);
        if (S::kBySlots && j == 0u) row_m[wave][r * 16u + n] = now[r];
      }
      if constexpr (S::kBySlots) {  // the team's maxima (and the last round's p is read)
        exchange_barrier();
#pragma unroll
        for (uint32_t r = 0; r < RT; ++r)
#pragma unroll
          for (uint32_t u = 0; u < VS; ++u)
            now[r] = fmaxf(now[r], row_m[team * VS + u][r * 16u + n]);
      }
#pragma unroll
      for (uint32_t r = 0; r < RT; ++r) {
        now[r] = fmaxf(m[r], now[r]);
        const float from = now[r] == -INFINITY ? 0.0f : now[r] - T::kShift;
        if (__builtin_amdgcn_ballot_w64(now[r] > m[r])) {
          const float keep = m[r] == -INFINITY ? 0.0f : exp2_of(m[r] - now[r]);
          l[r] *= keep;
#pragma unroll
          for (uint32_t d = 0; d < S::kTiles; ++d) out[r][d] *= keep;
          m[r] = now[r];
        }
#pragma unroll
        for (uint32_t i = 0; i < S::kOwnRows; ++i) {
          p[r][i] = exp2_of(p[r][i] - from);  // (0 where not seen)
          l[r] += p[r][i];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // ---- out
      if constexpr (S::kBySlots) {
        // each wave's p into the team's operands: a tile's slots are those of one or two waves
        constexpr uint32_t kPart = 4u / S::kSubs;  // words
        uint32_t* place = reinterpret_cast<uint32_t*>(shared + S::kQueryBytes);
#pragma unroll
        for (uint32_t r = 0; r < RT; ++r) {
          uint32_t b[T::kPieces][4];
          operands(p[r], b);
#pragma unroll
          for (uint32_t k = 0; k < T::kPieces; ++k) {
            const uint32_t tile = team * S::kTeamTiles + half / S::kSubs;
            uint32_t* to = place + (((tile * RT + r) * T::kPieces + k) * 64u + lane) * 4u +
                           half % S::kSubs * kPart;
            if constexpr (kPart == 4u)
              *reinterpret_cast<uint4*>(to) = make_uint4(b[k][0], b[k][1], b[k][2], b[k][3]);
            else
              *reinterpret_cast<uint2*>(to) = make_uint2(b[k][0], b[k][1]);
          }
        }
        exchange_barrier();
#pragma unroll
        for (uint32_t u = 0; u < S::kTeamTiles; ++u) {
          u32x4 b[RT][T::kPieces];
#pragma unroll
          for (uint32_t r = 0; r < RT; ++r)
#pragma unroll
            for (uint32_t k = 0; k < T::kPieces; ++k)
              b[r][k] = reinterpret_cast<const u32x4*>(
                  place)[(((team * S::kTeamTiles + u) * RT + r) * T::kPieces + k) * 64u + lane];
          clear_unseen(u, team_base + u * T::kSlots, there[u]);
          add_values(u, b);
          __builtin_amdgcn_sched_barrier(0);
          load_values(row, u);  // the next tile's
        }
      } else {
        u32x4 b[RT][T::kPieces];
#pragma unroll
        for (uint32_t r = 0; r < RT; ++r) {
          uint32_t w[T::kPieces][4];
          operands(p[r], w);
#pragma unroll
          for (uint32_t k = 0; k < T::kPieces; ++k)
            b[r][k] = u32x4{w[k][0], w[k][1], w[k][2], w[k][3]};
        }
        clear_unseen(0u, base, own_there);
        add_values(0u, b);
        __builtin_amdgcn_sched_barrier(0);
        load_values(row, 0u);  // the next tile's
      }
    }
    // (slots before the window need no page)
    if (bad > any_lo) report_device_error(a.report, kDevErrCachePage);

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
      if (j == 0u && (S::kBySlots || half == 0u)) {
        row_m[S::kBySlots ? wave : team][r * 16u + n] = m[r];
        row_l[S::kBySlots ? wave : team][r * 16u + n] = l[r];
      }
    }
    float* join = reinterpret_cast<float*>(shared) + (team * 16u + n) * S::kOutStride;
    constexpr uint32_t kTileWords = S::kTeams * 16u * S::kOutStride;
#pragma unroll
    for (uint32_t r0 = 0; r0 < RT; r0 += S::kOutTiles) {
      exchange_barrier();  // (queries and scores, or the last tiles' outputs, are no longer read)
#pragma unroll
      for (uint32_t r = r0; r < r0 + S::kOutTiles; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < S::kSets; ++w) top = fmaxf(top, row_m[w][r * 16u + n]);
        if (wave == r % S::kWaves) {
          Joined sum_l;
#pragma unroll
          for (uint32_t w = 0; w < S::kSets; ++w)
            sum_l.add(make_float2(row_m[w][r * 16u + n], row_l[w][r * 16u + n]), top);
          if (j == 0u) row_sum[r * 16u + n] = sum_l.result(top);
        }
        const float mine = Joined::times(m[r], top);
#pragma unroll
        for (uint32_t u = 0; u < S::kPasses; ++u)
#pragma unroll
          for (uint32_t w = 0; w < 4; ++w)
#pragma unroll
            for (uint32_t d = 0; d < S::kEach; d += 4) {
              const f32x4* t = &out[r][u * S::kEach + d];
              *reinterpret_cast<float4*>(
                  join + (r - r0) * kTileWords +
                  ((half * S::kPasses + u) * 16u + j * 4u + w) * S::kEach + d) =
                  make_float4(t[0][w] * mine, t[1][w] * mine, t[2][w] * mine, t[3][w] * mine);
            }
      }
      exchange_barrier();
      constexpr uint32_t kRowThreads = kThreads / 16u;
      const uint32_t jr = tid / kRowThreads, jn = tid % kRowThreads;
#pragma unroll
      for (uint32_t r = r0; r < r0 + S::kOutTiles; ++r) {
        const uint32_t out_row = row0 + r * 16u + jr;
        if (out_row >= rows) continue;
        const float2 st = row_sum[r * 16u + jr];
        const size_t head = (size_t)kv * rows + out_row;
        const size_t part_row = (size_t)(share + seq) * c.kv_heads * rows + head;
        const uint32_t t = o.by_group.of(out_row), h = kv * a.group + (out_row - t * a.group);
        if (jn == 0u) {
          if (!alone)
            o.part_stats[part_row] = st;
          else if (o.stats)
            o.stats[(size_t)seq * c.kv_heads * rows + head] = row_stats(st, T::kShift);
        }
        float* to = alone ? a.out + (((size_t)seq * a.tokens + t) * a.heads + h) * dim
                          : o.part_out + part_row * dim;
        const float times = alone ? row_times(st) : 1.0f;
        for (uint32_t d = jn * 4u; d < dim; d += 4u * kRowThreads) {
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (st.y != 0.0f) {  // (a row that sees nothing has no part in what its columns hold)
#pragma unroll
            for (uint32_t w = 0; w < S::kTeams; ++w) {
              const float4 y = *reinterpret_cast<const float4*>(
                  reinterpret_cast<const float*>(shared) + (r - r0) * kTileWords +
                  (w * 16u + jr) * S::kOutStride + d);
              v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
            }
            v.x *= times, v.y *= times, v.z *= times, v.w *= times;
          }
          *reinterpret_cast<Floats4*>(to + d) = Floats4{v.x, v.y, v.z, v.w};
        }
      }
    }
    if (o.counters && !alone) {
      // The last of the sequence's shares joins them.  Each wave waits for its
      // stores; then one thread's release and acquire make this share's outputs
      // known to the other XCDs, and theirs to this workgroup.
      const uint32_t share0 = uniform(walk.first / walk.each);
      const uint32_t last = uniform((walk.first + walk.span.rounds - 1u) / walk.each);
      const uint32_t shares = last - share0 + 1u;
      uint32_t* counter = o.counters + ((size_t)seq * c.kv_heads + kv) * o.tile_groups + group_at;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      exchange_barrier();
      if (tid == 0u)
        last_share = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_ACQ_REL,
                                            __HIP_MEMORY_SCOPE_AGENT) == shares - 1u;
      exchange_barrier();
      if (last_share) {
        if (tid == 0u)
          __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        constexpr uint32_t kRowThreads = kThreads / 16u;
        for (uint32_t out_row = row0 + tid / kRowThreads; out_row < min(row0 + RT * 16u, rows);
             out_row += 16u) {
          const size_t head = (size_t)kv * rows + out_row;
          const auto at = [&](uint32_t p) {
            return (size_t)(share0 + p + seq) * c.kv_heads * rows + head;
          };
          // (all of it under way at once)
          constexpr uint32_t kOuts = (DW * VS + 4u * kRowThreads - 1u) / (4u * kRowThreads);
          float2 set[kSharesJoinedInside];
          float4 x[kSharesJoinedInside][kOuts];
#pragma unroll
          for (uint32_t p = 0; p < kSharesJoinedInside; ++p) {
            set[p] = make_float2(-INFINITY, 0.0f);
            if (p < shares) set[p] = o.part_stats[at(p)];
#pragma unroll
            for (uint32_t k = 0; k < kOuts; ++k) {
              const uint32_t d = (tid % kRowThreads + k * kRowThreads) * 4u;
              x[p][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (p < shares && d < dim)
                x[p][k] = *reinterpret_cast<const float4*>(o.part_out + at(p) * dim + d);
            }
          }
          float top = -INFINITY;
#pragma unroll
          for (uint32_t p = 0; p < kSharesJoinedInside; ++p) top = fmaxf(top, set[p].x);
          Joined sum_l;
          float4 v[kOuts];
#pragma unroll
          for (uint32_t k = 0; k < kOuts; ++k) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (uint32_t p = 0; p < kSharesJoinedInside; ++p) {
            sum_l.add(set[p], top);
#pragma unroll
            for (uint32_t k = 0; k < kOuts; ++k) add_share(set[p].x, top, x[p][k], v[k]);
          }
          const float2 st = sum_l.result(top);
          const uint32_t t = o.by_group.of(out_row), h = kv * a.group + (out_row - t * a.group);
          float* to = a.out + (((size_t)seq * a.tokens + t) * a.heads + h) * dim;
          if (o.stats && tid % kRowThreads == 0u)
            o.stats[(size_t)seq * c.kv_heads * rows + head] = row_stats(st, T::kShift);
#pragma unroll
          for (uint32_t k = 0; k < kOuts; ++k) {
            const uint32_t d = (tid % kRowThreads + k * kRowThreads) * 4u;
            const float4 f = finished(v[k], st);
            if (d < dim) *reinterpret_cast<Floats4*>(to + d) = Floats4{f.x, f.y, f.z, f.w};
          }
        }
      }
    }
    next_sequence<kRound>(a, walk);
    if (walk.at < walk.end) exchange_barrier();  // (the outputs are no longer read)
  }
}

template <typename T, uint32_t DW, uint32_t VS, bool FAST, uint32_t RT, bool ONCE>
hipError_t launch_mfma(const AttentionArgs& a, Outputs o, hipStream_t s) {
  using S = Shape<T, DW, VS, RT>;
  static const hipError_t attr = hipFuncSetAttribute(
      reinterpret_cast<const void*>(&attention_mfma<T, DW, VS, FAST, RT, ONCE>),
      hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::kShared);
  if (attr != hipSuccess) return attr;
  const uint32_t tiles = row_tiles(a.tokens, a.group);
  o.tile_groups = (tiles + RT - 1u) / RT;
  o.round = S::kRound;
  o.shift = T::kShift;
  o.shares = shares_for(a.cache, o.tile_groups, o.round);
  o.by_shares = divisor_of(o.shares);
  o.by_tiles = divisor_of(o.tile_groups);
  // A few shares are joined by the last of them; many, whose join is more than
  // one workgroup's work, by a kernel of their own.  (1021 slots of 8 heads of
  // 128, four shares: 1.9 us less inside than with the second kernel, 12.5 in
  // all.  131,071 slots of 4 heads of 256, 64 shares: the second kernel takes
  // 5.5 of 95 us.)
  const size_t counters = (size_t)a.cache.sequences * a.cache.kv_heads * o.tile_groups;
  if (o.shares > kSharesJoinedInside || counters * 4u + 64u > kWorkspaceCounterBytes)
    o.counters = nullptr;
  const uint32_t units = o.shares * a.cache.kv_heads;
  const uint32_t blocks = o.tile_groups == 1u ? units : (units + 7u) / 8u * 8u * o.tile_groups;
  attention_mfma<T, DW, VS, FAST, RT, ONCE><<<blocks, 64 * S::kWaves, S::kShared, s>>>(a, o);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || o.shares == 1u || o.counters) return e;
  return launch_attention_join(a, o, s);
}

// The row tiles a workgroup takes, so that the cache is read for several at
// once: two, or three where two would leave the last group one of its two; of
// heads of 128 in 16 bits two, for three of them do not fit the registers (80
// us instead of 59 for 44 rows over 44,236 slots of 8 heads).  Heads of 256
// are shared by slots: 48 rows over 44,236 slots of 4 heads, three tiles at
// once, took 54 us where two waves with half of the head each and two tiles at
// once took 64.  (All four with plain loads of the values, the calls back to
// back.  Three tiles of F32 heads of 256 spill 30 registers, two none.)
//
// Where that is all of the rows, the values' loads are nontemporal (their lines
// are whole ones; the keys' come in two halves, and measured slower so).  Over
// caches that other memory's traffic has driven out of the 256 MB cache
// 131,071 slots of 4 heads of 256 in BF16 take 94.9 us so and 100.7 without, 48
// rows over 44,236 slots 57.7 and 60.5, 24 sequences in F32 102.3 and 103.6; over
// one that it still holds (8 x 4000 slots, 131 MB) 31.9 and 30.8.
template <typename T, uint32_t DW, uint32_t VS, bool FAST, uint32_t RT>
hipError_t launch_tiles(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  if (row_tiles(a.tokens, a.group) <= RT) return launch_mfma<T, DW, VS, FAST, RT, true>(a, o, s);
  return launch_mfma<T, DW, VS, FAST, RT, false>(a, o, s);
}
template <typename T, uint32_t DIM>
hipError_t launch_rows(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  const uint32_t tiles = row_tiles(a.tokens, a.group);
  if (tiles == 1u)
    return launch_mfma<T, (DIM < 128 ? DIM : 128), (DIM + 127) / 128, true, 1, true>(a, o, s);
  constexpr uint32_t kDw = DIM == 256 ? 64 : DIM, kVs = DIM / kDw;
  if constexpr (DIM != 128 || T::kBytes == 4)
    if (tiles == 3u || tiles > 4u) return launch_tiles<T, kDw, kVs, true, 3>(a, o, s);
  return launch_tiles<T, kDw, kVs, true, 2>(a, o, s);
}

// Heads of 64, 128 and 256 on pages of whole sixteens take scalar addresses: only
// they leave the registers for several row tiles.  (For one it is the same:
// 131,071 slots of 4 heads of 256 94.5 us, 92.7 on pages of 24; 8 sequences of 4000
// slots of 8 heads of 128 in F16 31.0 and 30.5.)  Others take one row tile at a time,
// in the next larger shape (those 8 sequences: 80 values 24.3 us, 96 26.3, 128 31.0).
template <typename T>
hipError_t launch_type(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  const uint32_t dim = a.cache.head_dim;
  if (a.cache.page_tokens % 16u == 0u) {
    if (dim == 64u) return launch_rows<T, 64>(a, o, s);
    if (dim == 128u) return launch_rows<T, 128>(a, o, s);
    if (dim == 256u) return launch_rows<T, 256>(a, o, s);
  }
  if (dim <= 64u) return launch_tiles<T, 64, 1, false, 1>(a, o, s);
  if (dim <= 128u) return launch_tiles<T, 128, 1, false, 1>(a, o, s);
  return launch_tiles<T, 128, 2, false, 1>(a, o, s);
}

}  // namespace attn
}  // namespace sihip
