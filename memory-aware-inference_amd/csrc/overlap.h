// Whether two arguments of a call have memory in common, for the checks of
// calls whose outputs may not be read by them. Host only.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace sihip {

// `blocks` blocks of `rows` rows of `size` bytes, block_stride and row_stride bytes apart; the rows of a block lie
// within its stride. Null: no memory. What would pass the address space ends at its end.
struct Region {
  uintptr_t at = 0, end = 0;
  size_t blocks = 0, block_stride = 0, rows = 0, row_stride = 0, size = 0;

  Region() = default;
  Region(const void* p, size_t size_) : Region(p, 1, 0, 1, 0, size_) {}
  Region(const void* p, size_t rows_, size_t stride, size_t size_)
      : Region(p, rows_, stride, 1, 0, size_) {}
  Region(const void* p, size_t blocks_, size_t block_stride_, size_t rows_, size_t row_stride_,
         size_t size_)
      : at((uintptr_t)p), blocks(blocks_), block_stride(block_stride_), rows(rows_),
        row_stride(row_stride_), size(size_) {
    if (!p || !blocks || !rows || !size) {
      at = end = 0;
      return;
    }
    const unsigned __int128 last = (unsigned __int128)at + span() +
                                   (unsigned __int128)(blocks - 1) * block_stride;
    end = last > UINTPTR_MAX ? UINTPTR_MAX : (uintptr_t)last;
  }
  unsigned __int128 span() const { return (unsigned __int128)(rows - 1) * row_stride + size; }
};

namespace overlap_detail {
using Wide = __int128;

inline Wide floor_div(Wide a, Wide b) {  // b > 0
  const Wide q = a / b;
  return q * b > a ? q - 1 : q;
}

// n_a pieces of l_a bytes s_a apart from 0 on, n_b of l_b bytes s_b apart from d on: f(d of a piece of b
// less the other's place) for pairs that have bytes in common, one of each distance at least, until it is true.
// A stride is at least its piece.
template <class F>
bool any_pair(Wide n_a, Wide s_a, Wide l_a, Wide d, Wide n_b, Wide s_b, Wide l_b, F f) {
  if (n_a == 1) s_a = s_b;
  if (n_b == 1) s_b = s_a;
  if (n_a == 1 && n_b == 1) return d < l_a && -l_b < d && f(d);
  if (s_a == s_b) {  // piece j of b against piece i of a: what counts is j - i
    Wide k = std::max(floor_div(-l_b - d, s_a) + 1, -(n_a - 1));
    for (; k < n_b && d + k * s_a < l_a; ++k)
      if (f(d + k * s_a)) return true;
    return false;
  }
  for (Wide i = 0; i < n_a; ++i) {
    Wide j = std::max(floor_div(i * s_a - l_b - d, s_b) + 1, Wide(0));
    for (; j < n_b && d + j * s_b < i * s_a + l_a; ++j)
      if (f(d + j * s_b - i * s_a)) return true;
  }
  return false;
}
}  // namespace overlap_detail

// Exact: what lies between another one's rows is apart from them. Regions that do not reach into
// one another's extent, or have equal strides, are told apart at once, others row by row.
inline bool overlap(const Region& a, const Region& b) {
  using overlap_detail::Wide;
  if (a.at >= b.end || b.at >= a.end) return false;
  if (a.blocks > b.blocks) return overlap(b, a);  // (the loop is over the fewer)
  return overlap_detail::any_pair(
      a.blocks, a.block_stride, a.span(), (Wide)b.at - (Wide)a.at, b.blocks, b.block_stride,
      b.span(), [&](Wide d) {
        return overlap_detail::any_pair(a.rows, a.row_stride, a.size, d, b.rows, b.row_stride,
                                        b.size, [](Wide) { return true; });
      });
}

// Whether an output has memory in common with one of the inputs.
template <size_t N>
bool overlaps_any(const Region& out, const Region (&in)[N]) {
  for (const Region& x : in)
    if (overlap(out, x)) return true;
  return false;
}

}  // namespace sihip
