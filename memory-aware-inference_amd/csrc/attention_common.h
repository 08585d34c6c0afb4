// What the attention kernels share: the workspace's layout and which slots a
// row sees.
#pragma once

#include <algorithm>

#include "decode_internal.h"

namespace sihip {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

// Row tiles of 16 rows that a kv head's tokens * group rows make.
__host__ __device__ inline uint32_t row_tiles(uint32_t tokens, uint32_t group) {
  return (tokens * group + 15u) / 16u;
}

// Shares that the rounds of all sequences are dealt to: as many workgroups as
// the card's 8 XCDs of 32 CUs hold at once, one a CU, over the kv heads.  The
// groups of row tiles of one share and head go to one XCD; one workgroup more
// than an XCD has CUs would wait for a whole share (verified drafts of three
// groups: 113 us for 33 workgroups on some XCDs, 94 us for 30).  No more than
// there can be rounds.
constexpr uint32_t kXcds = 8, kXcdCus = 32;
inline uint32_t shares_for(const CacheView& c, uint32_t tile_groups, uint32_t round) {
  const uint64_t rounds = (uint64_t)c.sequences * ((c.capacity + 31u) / round + 2u);
  const uint32_t units = kXcds * std::max(1u, kXcdCus / tile_groups);
  return (uint32_t)std::min<uint64_t>(std::max(1u, units / c.kv_heads), rounds);
}
inline uint32_t shares_most(const CacheView& c) {
  return std::max(1u, kXcds * kXcdCus / c.kv_heads);
}

// The workspace: (m, l) and the outputs before the division of the rows of
// every (share, sequence) pair (Outputs); with weights (m, 1 / l) of every row
// and its scores of all slots, [sequences][kv_heads][rows].  A share of a later
// sequence is the same or a later one, so that share + sequence numbers the pairs.
struct Space {
  size_t part_stats, part_out, stats, scores, bytes;
  uint32_t score_stride;
};
inline Space space_of(const CacheView& c, uint32_t heads, uint32_t tokens, bool weights) {
  const auto whole = [](size_t n) { return (n + 255u) / 256u * 256u; };
  Space s{};
  const size_t part_rows = (size_t)(shares_most(c) + c.sequences - 1u) * heads * tokens;
  s.part_stats = 0;
  s.part_out = whole(part_rows * 8u);
  s.bytes = s.part_out + whole(part_rows * c.head_dim * 4u);
  s.score_stride = (c.capacity + 3u) / 4u * 4u;
  if (weights) {
    const size_t rows = (size_t)c.sequences * heads * tokens;
    s.stats = s.bytes;
    s.scores = s.stats + whole(rows * 8u);
    s.bytes = s.scores + rows * s.score_stride * 4u;
  }
  return s;
}

// The slots that token t of a sequence of `length` tokens sees: [begin, end).
__device__ __forceinline__ void seen_slots(uint32_t length, uint32_t t, uint32_t capacity,
                                           uint32_t window, uint32_t& begin, uint32_t& end) {
  const uint32_t n = length + t + 1u;
  end = min(n, capacity);
  begin = window != 0u && n > window ? n - window : 0u;
}

// ---- how the work is dealt ----------------------------------------------------------
struct Outputs {
  float2* part_stats;  // (m, l) of a share's rows, [shares + sequences - 1][kv_heads][rows]
  float* part_out;     // and their outputs before the division
  float2* stats;       // with weights: (m, 1 / l) of every row, [sequences][kv_heads][rows]
  float* scores;
  uint32_t* counters;  // of shares that are done, zeroed; null: a second kernel joins
  uint32_t score_stride, shares, tile_groups, round;
  float shift;  // p is held times 2^shift
  Divisor by_group, by_heads, by_shares, by_tiles;  // group, kv_heads, shares, tile_groups
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Maximum over the lanes that share lane % 16: the second halves of the
// wave, then its odd rows of 16, are put beside the first.
__device__ __forceinline__ float columns_max(float v) {
  const uint32_t b = __float_as_uint(v);
  auto x = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t c = __float_as_uint(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
  x = __builtin_amdgcn_permlane16_swap(c, c, false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

// Bits [lo, hi) of a tile's 32 slots from `base` on.
__device__ __forceinline__ uint32_t slot_bits(uint32_t lo, uint32_t hi, uint32_t base) {
  const uint32_t a = lo > base ? min(lo - base, 32u) : 0u, b = hi > base ? min(hi - base, 32u) : 0u;
  return (uint32_t)((1ull << b) - 1ull) & ~(uint32_t)((1ull << a) - 1ull);
}

// One sequence's new tokens and the slots that any row of it sees, from a
// multiple of the tile on, in rounds (one at least, so that every sequence is
// somebody's).
struct Span {
  uint32_t count, length, start, slots, rounds;
};

// A value that all lanes hold, in a scalar register.
__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return __builtin_amdgcn_readfirstlane(v);
}

// Running sums of the first `count` lanes' values.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t lane, uint32_t count) {
  for (uint32_t o = 1; o < min(count, 64u); o <<= 1) {
    const uint32_t w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  return v;
}

// Rounds a share.  Going over to a next sequence takes a workgroup about as long
// as a round, so a sequence counts for one more, but for the first, where that
// makes the shares no more than an eighth longer.  (When it was taken, verified
// drafts of four sequences 74.5 us without it, 70.2 with it, 74.1 with two rounds; 24
// sequences of an f32 cache 110.7, 107.4, 108.2.  But four of 4000 slots, whose 32 shares
// of two rounds end where the sequences do, 16.4 without and 20.0 with it.)
struct Deal {
  uint32_t each, start;
};
__device__ __forceinline__ Deal deal_of(uint32_t total, uint32_t sequences, const Outputs& o) {
  const uint32_t none = o.by_shares.of(total + o.shares - 1u);
  const uint32_t one = o.by_shares.of(total + sequences - 1u + o.shares - 1u);
  return one - none <= none / 8u ? Deal{one, 1u} : Deal{none, 0u};
}

// A workgroup's walk through its share of the rounds of all sequences, the
// rounds [begin, limit) of [0, total).  Up to 64 sequences' lengths are read
// once, a lane each.
struct Walk {
  uint32_t lengths, counts, upto;  // the lane's sequence, and the rounds up to its last
  uint32_t start, each, begin, limit, at, end;  // the rounds that are left: [at, end)
  uint32_t seq, first;             // the present sequence, its first round
  Span span;
};
__device__ __forceinline__ Span span_of(const AttentionArgs& a, uint32_t count, uint32_t length,
                                        uint32_t round) {
  Span s{count, length, 0u, 0u, 1u};
  if (count == 0u) return s;
  uint32_t begin, end, other;
  seen_slots(length, 0u, a.cache.capacity, a.window, begin, other);
  seen_slots(length, count - 1u, a.cache.capacity, a.window, other, end);
  s.start = begin & ~31u;
  s.slots = end > s.start ? end - s.start : 0u;
  s.rounds = max(1u, (s.slots + round - 1u) / round);
  return s;
}
__device__ __forceinline__ Span span_of(const AttentionArgs& a, uint32_t seq, uint32_t round) {
  return span_of(a, brought(a.counts, seq, a.tokens), held(a.cache, seq), round);
}

// The present sequence's span.
template <uint32_t ROUND>
__device__ __forceinline__ void take_sequence(const AttentionArgs& a, Walk& w) {
  uint32_t count, length;
  if (a.cache.sequences <= 64u) {
    count = __builtin_amdgcn_readlane(w.counts, w.seq);
    length = __builtin_amdgcn_readlane(w.lengths, w.seq);
  } else {
    count = uniform(brought(a.counts, w.seq, a.tokens));
    length = uniform(held(a.cache, w.seq));
  }
  w.span = span_of(a, count, length, ROUND);
}
template <uint32_t ROUND>
__device__ __forceinline__ Walk first_walk(const AttentionArgs& a, const Outputs& o,
                                           uint32_t share) {
  const uint32_t lane = threadIdx.x & 63u, sequences = a.cache.sequences;
  Walk w{};
  uint32_t total = 0u;
  for (uint32_t base = 0; base < sequences; base += 64u) {
    uint32_t rounds = 0u;
    if (base + lane < sequences) {
      w.counts = brought(a.counts, base + lane, a.tokens);
      w.lengths = held(a.cache, base + lane);
      rounds = span_of(a, w.counts, w.lengths, ROUND).rounds;
    }
    w.upto = total + wave_scan(rounds, lane, sequences - base);
    total = __builtin_amdgcn_readlane(w.upto, min(sequences - base, 64u) - 1u);
  }
  const Deal deal = deal_of(total, sequences, o);
  w.each = deal.each;
  w.start = deal.start;
  w.upto += w.start * lane;
  total += w.start * (sequences - 1u);
  w.begin = w.at = min(share * w.each, total);
  w.end = min(w.begin + w.each, total);
  w.limit = w.begin + w.each;
  if (w.at >= w.end) return w;
  if (sequences <= 64u) {
    w.seq = (uint32_t)__builtin_ctzll(__builtin_amdgcn_ballot_w64(w.at < w.upto));
  } else {  // the first whose last round is not before `at`
    uint32_t before = 0u;
    for (uint32_t base = 0;; base += 64u) {
      const uint32_t rounds = base + lane < sequences ? span_of(a, base + lane, ROUND).rounds : 0u;
      const uint32_t sum = before + wave_scan(rounds, lane, 64u);
      const uint32_t upto = sum + w.start * (base + lane);
      const uint64_t here = __builtin_amdgcn_ballot_w64(w.at < upto);
      if (here) {
        const uint32_t at = (uint32_t)__builtin_ctzll(here);
        w.seq = base + at;
        w.first = __builtin_amdgcn_readlane(upto - rounds, at);
        break;
      }
      before = __builtin_amdgcn_readlane(sum, 63);
    }
  }
  take_sequence<ROUND>(a, w);
  if (sequences <= 64u) w.first = __builtin_amdgcn_readlane(w.upto, w.seq) - w.span.rounds;
  w.at = max(w.at, w.first);
  return w;
}
template <uint32_t ROUND>
__device__ __forceinline__ void next_sequence(const AttentionArgs& a, Walk& w) {
  w.at = w.first = w.first + w.span.rounds + w.start;
  if (w.at >= w.end) return;
  ++w.seq;
  take_sequence<ROUND>(a, w);
}

// ---- running maxima and sums -------------------------------------------------------
// (m, l) of sets of a row's slots, joined to those of all of them.  l < 0: there
// are slots, and all scores are -inf, which says nothing beside a set that has
// others.  A set's sum is taken times 2^(its m - the joint one).
struct Joined {
  float m = -INFINITY, l = 0.0f;
  bool minus = false;
  __device__ __forceinline__ static float times(float m, float top) {
    return m == -INFINITY ? 1.0f : exp2_of(m - top);  // (l is 0, -1 or no number)
  }
  // with `top` the joint maximum
  __device__ __forceinline__ void add(float2 set, float top) {
    minus |= set.y < 0.0f;
    l = fmaf(set.y < 0.0f ? 0.0f : set.y, times(set.x, top), l);
  }
  __device__ __forceinline__ float2 result(float top) const {
    return make_float2(top, minus && top == -INFINITY && l == 0.0f ? -1.0f : l);
  }
};
// What a row's sums are taken times in the end, and its (m, 1 / l) for the
// weights: 0 / 0 where every score is -inf.
__device__ __forceinline__ float row_times(float2 st) {
  return st.y < 0.0f ? NAN : 1.0f / st.y;
}
__device__ __forceinline__ float2 row_stats(float2 st, float shift) {
  if (st.y == 0.0f) return make_float2(0.0f, 0.0f);
  return make_float2(st.x == -INFINITY ? 0.0f : st.x - shift, row_times(st));
}

// Four values of a share's output added at the share's weight, and what becomes
// of the sum.
__device__ __forceinline__ void add_share(float m, float top, const float4& x, float4& sum) {
  const float w = m == -INFINITY ? 0.0f : exp2_of(m - top);
  sum.x = fmaf(w, x.x, sum.x);
  sum.y = fmaf(w, x.y, sum.y);
  sum.z = fmaf(w, x.z, sum.z);
  sum.w = fmaf(w, x.w, sum.w);
}
__device__ __forceinline__ float4 finished(float4 sum, float2 st) {
  if (st.y == 0.0f) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const float t = row_times(st);
  return make_float4(sum.x * t, sum.y * t, sum.z * t, sum.w * t);
}

constexpr uint32_t kSharesJoinedInside = 8;

}  // namespace attn

// kernels_attention_{f32,f16,bf16}.hip: the kernels of one type of cache
hipError_t launch_attention_f32(const AttentionArgs& a, const attn::Outputs& o, hipStream_t s);
hipError_t launch_attention_f16(const AttentionArgs& a, const attn::Outputs& o, hipStream_t s);
hipError_t launch_attention_bf16(const AttentionArgs& a, const attn::Outputs& o, hipStream_t s);
// kernels_attention_mfma.hip: the sequences that lie in several shares
hipError_t launch_attention_join(const AttentionArgs& a, const attn::Outputs& o, hipStream_t s);

// kernels_attention_mfma.hip: the output, and with `scores` every row's (m, 1 / l) and scores,
// where the matrix-core kernels take the call (*taken).
hipError_t launch_attention_mfma(const AttentionArgs& a, const attn::Space& sp, bool* taken,
                                 hipStream_t s);

}  // namespace sihip
