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

// Shares that the rounds of all sequences are dealt to: the workgroups that
// 256 CUs hold at once, over the kv heads and groups of row tiles; no more
// than there can be rounds.
constexpr uint32_t kCus = 256;
inline uint32_t shares_for(const CacheView& c, uint32_t tile_groups, uint32_t per_cu,
                           uint32_t round) {
  const uint64_t rounds = (uint64_t)c.sequences * ((c.capacity + 31u) / round + 1u);
  const uint32_t wanted = std::max(1u, kCus * per_cu / (c.kv_heads * tile_groups));
  return (uint32_t)std::min<uint64_t>(wanted, rounds);
}
// At most, whatever the kernel: two workgroups a CU.
inline uint32_t shares_most(const CacheView& c) { return std::max(1u, 2u * kCus / c.kv_heads); }

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
  uint32_t score_stride, shares, tile_groups, round;
  float shift;  // p is held times 2^shift
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Maximum or sum over the lanes that share lane % 16: the second halves of the
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
__device__ __forceinline__ Span span_of(const AttentionArgs& a, uint32_t seq, uint32_t round) {
  Span s{brought(a.counts, seq, a.tokens), held(a.cache, seq), 0u, 0u, 1u};
  if (s.count == 0u) return s;
  uint32_t begin, end, other;
  seen_slots(s.length, 0u, a.cache.capacity, a.window, begin, other);
  seen_slots(s.length, s.count - 1u, a.cache.capacity, a.window, other, end);
  s.start = begin / 32u * 32u;
  s.slots = end > s.start ? end - s.start : 0u;
  s.rounds = max(1u, (s.slots + round - 1u) / round);
  return s;
}

// A value that all lanes hold, in a scalar register.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t lane) {
#pragma unroll
  for (uint32_t o = 1; o < 64u; o <<= 1) {
    const uint32_t w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  return v;
}

// All sequences' rounds, by a wave.
__device__ __forceinline__ uint32_t all_rounds(const AttentionArgs& a, uint32_t round) {
  const uint32_t lane = threadIdx.x & 63u, sequences = a.cache.sequences;
  if (sequences == 1u) return span_of(a, 0u, round).rounds;
  uint32_t total = 0u;
  for (uint32_t base = lane; base < sequences; base += 64u) total += span_of(a, base, round).rounds;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
  return uniform(total);
}

// A workgroup's walk through the rounds of its share [at, end), `each` of them
// or fewer: sequence `seq` has the rounds [first, first + rounds).
struct Walk : Span {
  uint32_t seq, first, at, end, each;
};
__device__ __forceinline__ void take(Walk& w, const Span& s) {
  w.count = uniform(s.count), w.length = uniform(s.length), w.start = uniform(s.start);
  w.slots = uniform(s.slots), w.rounds = uniform(s.rounds);
}

// The walk's sequence: the one with round `w.at`.  Every lane of a wave takes part.
__device__ __forceinline__ void find_sequence(const AttentionArgs& a, uint32_t round, Walk& w) {
  const uint32_t lane = threadIdx.x & 63u, sequences = a.cache.sequences;
  w.seq = w.first = 0u;
  if (sequences == 1u) return take(w, span_of(a, 0u, round));
  uint32_t before = 0u;
  for (uint32_t base = 0; base < sequences; base += 64u) {
    const uint32_t mine =
        base + lane < sequences ? span_of(a, base + lane, round).rounds : 0u;
    const uint32_t upto = wave_scan(mine, lane);
    const uint64_t here = __builtin_amdgcn_ballot_w64(mine != 0u && w.at < before + upto);
    if (here) {
      const uint32_t at = (uint32_t)__builtin_ctzll(here);
      w.seq = base + at;
      w.first = before + __builtin_amdgcn_readlane(upto - mine, at);
      return take(w, span_of(a, w.seq, round));
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
}
__device__ __forceinline__ Walk first_walk(const AttentionArgs& a, uint32_t round, uint32_t shares,
                                           uint32_t share) {
  Walk w{};
  const uint32_t total = all_rounds(a, round);
  w.each = uniform((total + shares - 1u) / shares);
  const uint64_t at = (uint64_t)share * w.each;
  w.at = uniform((uint32_t)min(at, (uint64_t)total));
  w.end = uniform((uint32_t)min(at + w.each, (uint64_t)total));
  if (w.at < w.end) find_sequence(a, round, w);
  return w;
}
__device__ __forceinline__ void next_walk(const AttentionArgs& a, uint32_t round, Walk& w) {
  w.at = w.first = w.first + w.rounds;
  if (w.at >= w.end) return;
  ++w.seq;
  take(w, span_of(a, w.seq, round));
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
__device__ __forceinline__ float2 row_stats(float2 st, float shift) {
  if (st.y == 0.0f) return make_float2(0.0f, 0.0f);
  return make_float2(st.x == -INFINITY ? 0.0f : st.x - shift, row_times(st));
}

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
