// What the attention kernels share: the workspace's layout and which slots a
// row sees.
#pragma once

#include <algorithm>

#include "decode_internal.h"

namespace sihip {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

// Workgroups that the split of the caches' lengths aims at: two for each of
// 256 CUs, what the registers of the largest heads leave room for.
constexpr uint32_t kTargetGroups = 512;

// Row tiles of 16 rows that a kv head's tokens * group rows make.
__host__ __device__ inline uint32_t row_tiles(uint32_t tokens, uint32_t group) {
  return (tokens * group + 15u) / 16u;
}

// Parts that all sequences' slots together are dealt to.  A sequence's last
// part may be short, so that up to `sequences` more are in use.
inline uint32_t parts_wanted(const CacheView& c, uint32_t tokens, uint32_t group) {
  return std::max(1u, kTargetGroups / (c.kv_heads * row_tiles(tokens, group)));
}
inline uint32_t parts_most(const CacheView& c, uint32_t tokens, uint32_t group) {
  const uint32_t wanted = parts_wanted(c, tokens, group);
  return wanted == 1u ? c.sequences : wanted + c.sequences;
}

// The workspace: (m, l) and the unscaled output of every part's rows,
// [parts][kv_heads][row tiles][16]; with weights (m, 1 / l) of every row, and
// its scores of all slots, [sequences][kv_heads][tokens * group].
struct Space {
  size_t part_stats, part_out, stats, scores, bytes;
  uint32_t score_stride;
};
inline Space space_of(const CacheView& c, uint32_t heads, uint32_t tokens, bool weights) {
  const uint32_t group = heads / c.kv_heads;
  const auto whole = [](size_t n) { return (n + 255u) / 256u * 256u; };
  Space s{};
  const size_t part_rows =
      (size_t)parts_most(c, tokens, group) * c.kv_heads * row_tiles(tokens, group) * 16u;
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

}  // namespace attn

// kernels_attention_mfma.hip: the output, and with `scores` every row's (m, 1 / l) and scores,
// where the matrix-core kernels take the call (*taken).
hipError_t launch_attention_mfma(const AttentionArgs& a, const attn::Space& sp, bool* taken,
                                 hipStream_t s);

}  // namespace sihip
