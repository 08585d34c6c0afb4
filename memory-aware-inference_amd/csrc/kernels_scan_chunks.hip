// The state scan of prompts: 32 tokens at a time on the matrix cores.
//
// With G_i the sum of the log decays up to token i of a chunk and S the state before
// it, the chunk's inputs u (rows u_i) solve a triangular system and the rest is
// products:
//   (I + L) U = R,  R_i = w_i (v_i - e^{G_i} S^T k_i),  L_ij = w_i (k_i . k_j) e^{G_i - G_j}, j < i
//   o_i = e^{G_i} S^T q_i + sum_{j <= i} P_ij u_j,  P_ij = (q_i . k_j) e^{G_i - G_j}
//   S'  = e^{G} S + sum_j e^{G - G_j} k_j u_j^T
// (without the correction U is w v).  Of U the first sixteen rows are T00 R0, T00 the inverse of (I + L)'s
// first diagonal block, the others T11 (R1 - L10 U0).
// Every column of v, S and o goes through this by
// itself, so a wave takes sixteen columns through all chunks and keeps their state in
// its registers: the layout that the matrix cores leave sums in is, up to the order of
// the summed index, the one that they take right operands in, and nothing
// but the operands that all columns share goes through LDS.  Those are made by four or six
// further waves, up to two chunks ahead, so that a chunk has one barrier.
//
// The matrix cores take 16-bit operands, f32 values as sums of pieces.  Products of whole columns,
// whose errors count against a column's size, are of two f16 each (22 bits of keys and queries,
// to their largest value, of a state's column and of what it gains, both to the larger of their largest
// values; three products of pieces).  R, U and what they are multiplied by are three bf16 each (8
// bits of each, cut off, so that their sum is the value; six products): a loud token that is
// forgotten within its chunk costs the quiet ones behind it nothing.  The sums G are 64 bits wide, of
// log decays of no less than -256: they stay below 2^14 and good to 2^-38, so that the difference of two of them is as
// exact as the gates.
//
// A chunk of one workgroup by itself is a chain: products with the state, the system's three products,
// P's, the units, the state's own; a taker's wave, alone on its SIMD, issues or waits for one of
// them at a time (4093 tokens of 48 heads of 128: 128 chunks in 295 us, 5 thousand cycles each; its
// matrix instructions are 1.6 thousand of them).  With eight takers a SIMD has three waves and a chunk 1.6 thousand
// vector instructions of four cycles and more and 230 matrix instructions of 16: 9 thousand cycles.
//
// What is no finite number stays where it belongs: a zero of L or P times a later token's NaN
// would not, so a wave that finds one in U takes the chunk token by token.  So do all of them where a key or query is
// so short beside eps's root that its pieces, held over its length, would lose bits: its row is raised
// by a power of two that is kept beside it.
#include "scan_common.h"

namespace sihip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kChunk = 32;
constexpr uint32_t kPieces = 3;       // bf16
constexpr uint32_t kHalves = 2;       // f16
// What keys and queries are held times: far enough above f16's least numbers for their low pieces, and what is
// added to a state as far, which is held in its units over this (2^14 left those 2^-22 to 2^-21 of the
// largest, and states of the selective form 2.3e-7 to 2.7e-7 off where now 1.4e-7).
constexpr float kUp = 0x1p10f;
constexpr float kForgotten = -256.0f; // the least log decay of a token
// The waves of a workgroup: `takers` that take sixteen columns each through the chunks, two or four that
// make the rows of K and Q, and two that make what is left of a chunk's operands.  Four makers of
// rows where two takers leave registers for eight waves: theirs is the longest course without the
// correction (two sequences of 3001 tokens of 64 heads of 128 x 64: 208 us with two, 186 with four), and close
// to it with it (4093 tokens of 48 heads of 128: 303 and 293).
constexpr uint32_t row_makers(uint32_t steps, uint32_t takers) {
  return steps > 2 && takers == 2 ? 4 : 2;
}
constexpr uint32_t waves_of(uint32_t steps, uint32_t takers) {
  return takers + 2u + row_makers(steps, takers);
}
constexpr uint32_t kRow = 20;     // floats between rows of the 16 x 16 blocks of f32

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The bf16 pieces of x and y, in the halves of one word each.
__device__ __forceinline__ void split(float x, float y, uint32_t (&w)[kPieces]) {
#pragma unroll
  for (uint32_t i = 0; i < kPieces; ++i) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    w[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    x -= __uint_as_float(a & 0xffff0000u);
    y -= __uint_as_float(b & 0xffff0000u);
  }
}
__device__ __forceinline__ void split8(const f32x4& lo, const f32x4& hi, u32x4 (&p)[kPieces]) {
  uint32_t w[4][kPieces];
  split(lo[0], lo[1], w[0]);
  split(lo[2], lo[3], w[1]);
  split(hi[0], hi[1], w[2]);
  split(hi[2], hi[3], w[3]);
#pragma unroll
  for (uint32_t i = 0; i < kPieces; ++i) p[i] = u32x4{w[0][i], w[1][i], w[2][i], w[3][i]};
}
// The f16 pieces, of values of at most 2^15.
__device__ __forceinline__ void halve(float x, float y, uint32_t (&w)[kHalves]) {
  const f16x2 a = __builtin_convertvector((f32x2{x, y}), f16x2);
  const f16x2 b = __builtin_convertvector(
      (f32x2{__builtin_fmaf((float)a.x, -1.0f, x), __builtin_fmaf((float)a.y, -1.0f, y)}), f16x2);
  w[0] = __builtin_bit_cast(uint32_t, a);
  w[1] = __builtin_bit_cast(uint32_t, b);
}
__device__ __forceinline__ void halve8(const f32x4& lo, const f32x4& hi, u32x4 (&p)[kHalves]) {
  uint32_t w[4][kHalves];
  halve(lo[0], lo[1], w[0]);
  halve(lo[2], lo[3], w[1]);
  halve(hi[0], hi[1], w[2]);
  halve(hi[2], hi[3], w[3]);
#pragma unroll
  for (uint32_t i = 0; i < kHalves; ++i) p[i] = u32x4{w[0][i], w[1][i], w[2][i], w[3][i]};
}
// The power of two that takes a largest value m (of at least 2^-119) into [2^7, 2^8), and its inverse.
__device__ __forceinline__ float scale_of(float m, float* inverse) {
  const uint32_t e = min(max(__float_as_uint(m) >> 23, 8u), 254u);
  *inverse = __uint_as_float((e - 7u) << 23);
  return __uint_as_float((261u - e) << 23);
}
__device__ __forceinline__ int32_t exponent(float x) {  // of x >= 0, biased
  return (int32_t)(__float_as_uint(x) >> 23);
}
// (NaNs count as nothing)
__device__ __forceinline__ float largest(const f32x4& x, float m) {
  asm("v_max3_f32 %0, %0, |%1|, |%2|\n\tv_max3_f32 %0, %0, |%3|, |%4|"
      : "+&v"(m)
      : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]));
  return m;
}
// Maximum over the lanes of a column.
__device__ __forceinline__ float columns_max(float v) {
  const uint32_t b = __float_as_uint(v);
  auto x = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t c = __float_as_uint(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
  x = __builtin_amdgcn_permlane16_swap(c, c, false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
// The products of pieces, the least first.
constexpr uint32_t kPairs = 6;
constexpr uint32_t kLeft[kPairs] = {0, 2, 1, 0, 1, 0}, kRight[kPairs] = {2, 0, 1, 1, 0, 0};
constexpr uint32_t kHalfPairs = 3;  // of f16
constexpr uint32_t kHalfLeft[kHalfPairs] = {0, 1, 0}, kHalfRight[kHalfPairs] = {1, 0, 0};

// 2^x, the card's
__device__ __forceinline__ float power_of_two(double x) {
  return __builtin_amdgcn_exp2f((float)x);
}

// LDS writes are done, and everybody's; loads from memory stay under way.
__device__ __forceinline__ void exchange_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Operands of 16 rows by 32 columns lie as the matrix cores take them: lane (p, row) = p * 16 + row
// has columns 16 a + 4 p + i, a = 0, 1, i = 0..3, in sixteen bytes, one such fragment a piece.
// The rows' places are permuted by p and the column step, so that writes of neighbouring
// columns and the transposing reads meet different banks.
__device__ __forceinline__ uint32_t place(uint32_t p, uint32_t row, uint32_t step) {
  return p * 16u + (row ^ ((16u - 4u * p) % 16u) ^ step);
}

// Rows of a chunk by way of a buffer whose length ends behind the last token: what is read behind it
// is zero, and what is written there goes nowhere, without a branch.  Offsets are bytes from the chunk's first
// row; kOutside is behind any of them.
constexpr uint32_t kOutside = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const float* first, uint32_t bytes) {
  // (all lanes' are the same: in scalar registers)
  const uint64_t at = (uint64_t)first;
  const uint32_t low = __builtin_amdgcn_readfirstlane((uint32_t)at);
  const uint32_t high = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
  const uint64_t base = (uint64_t)high << 32 | low;
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, __builtin_amdgcn_readfirstlane(bytes),
                                           0x00027000);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const float* first, size_t stride,
                                                          uint32_t left) {
  return buffer_of(first, min(left, kChunk) * (uint32_t)stride * 4u);
}

constexpr uint32_t kRaised = 1u, kZeros = 2u;  // short rows that are raised, keys that are zeros
struct alignas(16) Gated {  // of a chunk's tokens (four of them are read at once)
  float grow[kChunk];   // e^{G_i}
  float fade[kChunk];   // e^{G - G_i}
  float write[kChunk];  // w_i
  float keep[kChunk];   // a_i
  float key[kChunk], query[kChunk];  // what the rows of the operands are to be multiplied by
  float total;          // e^{G}
  // of eight rows each (delta rule): kRaised, kZeros, or nothing; rows beside these have key[], query[]
  alignas(4) uint8_t raised[4];
};

// Keys of more than 128 values leave room for fewer chunks: rows of two, blocks of one.  Then a chunk's
// blocks are made when the one before it has been taken, behind a barrier of their own.
template <uint32_t STEPS>
struct ChunkShared {
  static constexpr bool kTight = STEPS > 4;
  static constexpr uint32_t kRowSets = kTight ? 2 : 3, kBlockSets = kTight ? 1 : 2;
  u32x4 key[kRowSets][2 * STEPS * kHalves * 64];  // [tile of 16 tokens][step of 32 keys][piece][place]
  u32x4 query[kRowSets][2 * STEPS * kHalves * 64];
  u32x4 solve[kBlockSets][3 * kPieces * 64];      // T00, T11 and -L10, beside blocks of zeros
  u32x4 mix[kBlockSets][2 * kPieces * 64];        // P
  Gated gated[3];
  double sum[2][kChunk];                     // G_i / ln 2
  alignas(16) float scratch[2][16 * kRow];   // blocks on their way from one layout to the other
};

template <uint32_t STEPS>
__device__ __forceinline__ uint32_t half_fragment(uint32_t tile, uint32_t step, uint32_t piece) {
  return ((tile * STEPS + step) * kHalves + piece) * 64u;
}
__device__ __forceinline__ uint32_t fragment(uint32_t tile, uint32_t piece) {
  return (tile * kPieces + piece) * 64u;
}

// ---- the makers -------------------------------------------------------------------
// A chunk's rows of keys and queries on their way: a lane has four values of `kLoads` rows.
template <uint32_t STEPS, uint32_t MAKERS>
struct Raw {
  static constexpr uint32_t kLanes = STEPS > 4 ? 64 : STEPS > 2 ? 32 : STEPS * 8;  // a row's
  static constexpr uint32_t kRows = 64 / kLanes;                  // rows a load
  static constexpr uint32_t kParts = STEPS > 4 && MAKERS < 4 ? 2 : 1;  // in which a maker takes its rows
  static constexpr uint32_t kPartRows = kChunk / MAKERS / kParts;
  static constexpr uint32_t kLoads = kPartRows / kRows;
  f32x4 k[kLoads], q[kLoads];
};

// The lane's share of part `part` (of a maker after the other) of the rows from `k` and `q` on; `left` tokens of the
// sequence are there.
template <uint32_t STEPS, uint32_t MAKERS>
__device__ __forceinline__ void fetch(Raw<STEPS, MAKERS>& r, const ScanArgs& a, const float* k,
                                      const float* q, uint32_t part, uint32_t lane,
                                      uint32_t left) {
  using W = Raw<STEPS, MAKERS>;
  const __amdgpu_buffer_rsrc_t keys = rows_of(k, a.k_stride, left);
  const __amdgpu_buffer_rsrc_t queries = rows_of(q, a.q_stride, a.out ? left : 0u);
  const uint32_t at = 4u * (lane % W::kLanes), t0 = part * W::kPartRows + lane / W::kLanes;
  const uint32_t k_step = 4u * (uint32_t)a.k_stride, q_step = 4u * (uint32_t)a.q_stride;
  if (a.key_dim % 4u == 0u) {
    // (a lane behind the row's end reads behind the buffer's)
    const uint32_t in = at < a.key_dim ? 4u * at : kOutside;
#pragma unroll
    for (uint32_t l = 0; l < W::kLoads; ++l) {
      const uint32_t t = t0 + l * W::kRows;
      r.k[l] = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(keys, in + t * k_step, 0, 0));
      r.q[l] = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(queries, in + t * q_step, 0, 0));
    }
    return;
  }
#pragma unroll
  for (uint32_t l = 0; l < W::kLoads; ++l)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t t = t0 + l * W::kRows, in = at + i < a.key_dim ? 4u * (at + i) : kOutside;
      r.k[l][i] =
          __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(keys, in + t * k_step, 0, 0));
      r.q[l][i] =
          __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(queries, in + t * q_step, 0, 0));
    }
}

// Value v of V, reduced by `f` over LANES neighbouring lanes, in lanes v + a multiple of V: of two
// values one goes on in the lanes whose bit is clear, the other in those whose bit is set.
template <uint32_t LANES, uint32_t V, class F>
__device__ __forceinline__ float reduced(float (&x)[V], uint32_t lane, F f) {
  auto moved = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value,
                                                      0xf, 0xf, true));
  };
  auto half = [&](uint32_t values, uint32_t bit, auto ctrl) {
    const bool odd = lane & bit;
#pragma unroll
    for (uint32_t i = 0; i < V / 2; ++i)
      if (i < values / 2) x[i] = f(odd ? x[2 * i + 1] : x[2 * i], moved(odd ? x[2 * i] : x[2 * i + 1], ctrl));
  };
  using std::integral_constant;
  half(V, 1u, integral_constant<int, 0xb1>{});       // neighbours of a pair
  half(V / 2, 2u, integral_constant<int, 0x4e>{});   // pairs of four
  if (V >= 8) half(V / 4, 4u, integral_constant<int, 0x124>{});  // fours, round the sixteen
  if (V >= 16) half(V / 8, 8u, integral_constant<int, 0x128>{});
  if (LANES == 8) x[0] = f(x[0], __shfl_xor(x[0], 4));
  if (LANES >= 16 && V == 8) x[0] = f(x[0], moved(x[0], integral_constant<int, 0x128>{}));
  if (LANES >= 32) {  // the odd rows of sixteen are put beside the even ones
    const uint32_t b = __float_as_uint(x[0]);
    auto y = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    x[0] = f(__uint_as_float(y[0]), __uint_as_float(y[1]));
  }
  if (LANES == 64) {
    const uint32_t b = __float_as_uint(x[0]);
    auto y = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    x[0] = f(__uint_as_float(y[0]), __uint_as_float(y[1]));
  }
  return x[0];
}
// Value v of them again, in all of the lanes.
template <uint32_t LANES, uint32_t V>
__device__ __forceinline__ float spread(float x, uint32_t lane) {
  if (LANES == 8) return __shfl(x, (lane & ~7u) + V);
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + V, 0xf, 0xf, true));
}

template <uint32_t N, class F>
__device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<uint32_t, N - 1>{});
  }
}

// Keys and queries in pieces: under the delta rule over their length, else to a power of two that
// is kept beside them.  Over its length a row of the length l is l / sqrt(l^2 + eps) long: where that is 2^-8 and
// more, its largest value is held as 2^-2 at least, and f16's least step, 2^-24, is 22 bits of it.  Shorter
// rows are raised.
template <uint32_t STEPS, bool DELTA, uint32_t MAKERS>
__device__ __forceinline__ void make_rows(ChunkShared<STEPS>& sh, uint32_t chunk,
                                          const Raw<STEPS, MAKERS>& r, const ScanArgs& a, uint32_t part,
                                          uint32_t lane, uint32_t left) {
  using W = Raw<STEPS, MAKERS>;
  constexpr uint32_t V = 2 * W::kLoads;  // the loads' keys and queries in turn
  const uint32_t in = lane % W::kLanes, row = part * W::kPartRows + lane / W::kLanes;
  const uint32_t at = 4u * in, step = at / 32u, half = at / 16u % 2u, p = at / 4u % 4u;
  const bool held = at < 32u * STEPS;
  float x[V], scale;
  Gated& g = sh.gated[chunk % 3u];
  auto sizes = [&] {
#pragma unroll
    for (uint32_t l = 0; l < W::kLoads; ++l) {
      x[2 * l] = largest(r.k[l], 0.0f);
      x[2 * l + 1] = largest(r.q[l], 0.0f);
    }
    return reduced<W::kLanes>(x, lane, [](float y, float z) { return fmaxf(y, z); });
  };
  const uint32_t token = row + in % V / 2u * W::kRows;  // of the value that comes to this lane
  if (DELTA) {
#pragma unroll
    for (uint32_t l = 0; l < W::kLoads; ++l) {
      auto squares = [](const f32x4& y) {
        return __builtin_fmaf(y[3], y[3], __builtin_fmaf(y[2], y[2], __builtin_fmaf(y[1], y[1], y[0] * y[0])));
      };
      x[2 * l] = squares(r.k[l]);
      x[2 * l + 1] = squares(r.q[l]);
    }
    const float sum = reduced<W::kLanes>(x, lane, [](float y, float z) { return y + z; });
    // (rows behind the last token are zeros whatever eps is)
    scale = kUp * inverse_root(sum + (token < left ? a.eps : 1.0f));
    // (queries that are not read are zeros)
    bool small = token < left && sum < a.eps * 0x1p-16f && (a.out || in % 2u == 0u);
    uint32_t some = 0u;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(small) != 0u, 0)) {
      const float most = sizes();
      const bool none = small && !(most > 0.0f);  // (zeros are held as they are)
      small = small && !none;
      some = (__builtin_amdgcn_ballot_w64(small) ? kRaised : 0u) |
             (__builtin_amdgcn_ballot_w64(none && in % 2u == 0u) ? kZeros : 0u);
      // (the largest into [2^8, 2^10); what is below 2^-118 has fewer bits)
      const int32_t e = exponent(scale);
      const int32_t up = small ? max(min(min(262 - exponent(most) - e, 253 - e), 126), 0) : 0;
      scale *= __uint_as_float((uint32_t)(127 + up) << 23);
      const float down = none ? 0.0f : __uint_as_float((uint32_t)(127 - up) << 23);
      if (in < V) (in % 2u ? g.query : g.key)[token] = down;
    }
#pragma unroll
    for (uint32_t i = 0; i < W::kPartRows / 8u; ++i) g.raised[part * (W::kPartRows / 8u) + i] = some;
  } else {
    float down;
    scale = scale_of(sizes(), &down);
    if (in < V) (in % 2u ? g.query : g.key)[token] = in % 2u ? a.scale * down : down;
  }
  auto put = [&](u32x4* to, const f32x4& y, uint32_t t) {
    uint32_t lo[kHalves], hi[kHalves];
    halve(y[0], y[1], lo);
    halve(y[2], y[3], hi);
    if (held)
#pragma unroll
      for (uint32_t i = 0; i < kHalves; ++i)
        reinterpret_cast<u32x2*>(to + half_fragment<STEPS>(t / 16u, step, i) +
                                 place(p, t % 16u, step))[half] = u32x2{lo[i], hi[i]};
  };
  each<W::kLoads>([&](auto l) {
    constexpr uint32_t L = decltype(l)::value;
    put(sh.key[chunk % sh.kRowSets], r.k[L] * spread<W::kLanes, 2 * L>(scale, lane), row + L * W::kRows);
    put(sh.query[chunk % sh.kRowSets], r.q[L] * spread<W::kLanes, 2 * L + 1>(scale, lane),
        row + L * W::kRows);
  });
}

// A chunk's gates, by one wave, a token a lane; rows behind the last token change nothing.
template <uint32_t STEPS, bool DELTA>
__device__ __forceinline__ void make_gates(ChunkShared<STEPS>& sh, uint32_t n, const ScanArgs& a,
                                           uint32_t lane, float gate, float beta, float decay,
                                           float bias, uint32_t left) {
  float log_keep = 0.0f, write = 0.0f;
  if (lane < left && lane < kChunk) {
    const float s = softplus(gate + bias);
    log_keep = decay * s;
    // (e^-256 is zero in f32, and so is every factor across this token; what is larger would cost the
    // sums behind it the bits of their own tokens' decays, an infinite one all of them)
    if (log_keep < kForgotten) log_keep = kForgotten;
    write = DELTA ? sigmoid(beta) : s;
  }
  double sum = log_keep * 1.4426950408889634;
#pragma unroll
  for (uint32_t m = 1; m < kChunk; m *= 2) {
    const double before = __shfl_up(sum, m);
    if (lane % kChunk >= m) sum += before;
  }
  const double all = __shfl(sum, kChunk - 1u);
  if (lane < kChunk) {
    Gated& g = sh.gated[n % 3u];
    sh.sum[n % 2u][lane] = sum;
    g.grow[lane] = power_of_two(sum);
    g.fade[lane] = power_of_two(all - sum);
    g.write[lane] = write;
    g.keep[lane] = expf(log_keep);
    if (lane == 0u) g.total = power_of_two(all);
  }
}

// A 16 x 16 block in the matrix cores' layout of sums (lane (p, n): rows 4 p + r of column n), as
// one with four columns 4 p + r of row n a lane, by way of LDS.
__device__ __forceinline__ f32x4 turned(float* block, const f32x4& x, uint32_t p, uint32_t n) {
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) block[(4u * p + r) * kRow + n] = x[r];
  return *reinterpret_cast<const f32x4*>(block + n * kRow + 4u * p);
}
// Four columns 16 tj + 4 p + r of row 16 ti + n into fragments.
__device__ __forceinline__ void put_pieces(u32x4* to, const f32x4& x, uint32_t p, uint32_t n,
                                           uint32_t ti, uint32_t tj) {
  uint32_t lo[kPieces], hi[kPieces];
  split(x[0], x[1], lo);
  split(x[2], x[3], hi);
#pragma unroll
  for (uint32_t c = 0; c < kPieces; ++c)
    reinterpret_cast<u32x2*>(to + fragment(ti, c) + place(p, n, 0u))[tj] = u32x2{lo[c], hi[c]};
}

// The inverse of I + L, L strictly lower, 16 x 16, in the layout of sums; `low` has columns
// 4 p + r of row n.  Four rows are solved in the lanes that have them, and taken off the rows
// below by matrix products of four columns.
__device__ __forceinline__ f32x4 inverted(const f32x4& low, uint32_t p, uint32_t n) {
  f32x4 x;
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) x[r] = 4u * p + r == n ? 1.0f : 0.0f;
#pragma unroll
  for (uint32_t c = 0; c < 4; ++c) {
    const bool here = p == c, below = n >= 4u * (c + 1u);
    auto l = [&](uint32_t i, uint32_t j) {
      return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(low[j]), 20u * c + i));
    };
    const f32x4 y = x;
    const float x1 = __builtin_fmaf(-l(1, 0), y[0], y[1]);
    const float x2 = __builtin_fmaf(-l(2, 1), x1, __builtin_fmaf(-l(2, 0), y[0], y[2]));
    const float x3 = __builtin_fmaf(
        -l(3, 2), x2, __builtin_fmaf(-l(3, 1), x1, __builtin_fmaf(-l(3, 0), y[0], y[3])));
    x[1] = here ? x1 : y[1];
    x[2] = here ? x2 : y[2];
    x[3] = here ? x3 : y[3];
    if (c == 3u) break;
    f32x4 solved, off = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) solved[r] = here ? x[r] : 0.0f;
#pragma unroll
    for (uint32_t r = 0; r < 4; r += 2) {
      x = __builtin_amdgcn_mfma_f32_16x16x4f32(below ? -low[r] : 0.0f, solved[r], x, 0, 0, 0);
      off = __builtin_amdgcn_mfma_f32_16x16x4f32(below ? -low[r + 1] : 0.0f, solved[r + 1], off, 0,
                                                 0, 0);
    }
    x += off;
  }
  return x;
}

// Sixteen rows' fragments, all steps.
template <uint32_t STEPS>
struct Tile {
  u32x4 x[STEPS][kHalves];

  __device__ __forceinline__ void read(const u32x4* from, uint32_t tile, uint32_t p, uint32_t n) {
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s)
#pragma unroll
      for (uint32_t i = 0; i < kHalves; ++i)
        x[s][i] = from[half_fragment<STEPS>(tile, s, i) + place(p, n, s)];
  }
};
// Products of rows `j` with rows `i`: lane (p, n) row n of i with rows 4 p + r of j.
template <uint32_t STEPS>
__device__ __forceinline__ f32x4 products(const Tile<STEPS>& j, const Tile<STEPS>& i) {
  f32x4 sum[2];
  sum[0] = sum[1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (uint32_t s = 0; s < STEPS; ++s)
#pragma unroll
    for (uint32_t k = 0; k < kHalfPairs; ++k)
      sum[(s * kHalfPairs + k) % 2] =
          mfma16(j.x[s][kHalfLeft[k]], i.x[s][kHalfRight[k]], sum[(s * kHalfPairs + k) % 2]);
  return sum[0] + sum[1];
}
// e^{G_i - G_j}, i token 16 ti + n, j tokens 16 tj + 4 p + r
__device__ __forceinline__ f32x4 between(const double* sum, uint32_t ti, uint32_t tj, uint32_t p,
                                         uint32_t n) {
  const double i = sum[16u * ti + n];
  f32x4 d;
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) d[r] = power_of_two(i - sum[16u * tj + 4u * p + r]);
  return d;
}

// A diagonal block of (I + L)^-1 out of products of keys.
template <uint32_t STEPS>
__device__ __forceinline__ void put_solve(ChunkShared<STEPS>& sh, uint32_t chunk, f32x4 x,
                                          const f32x4& decay, uint32_t t, uint32_t p, uint32_t n) {
  const float w = sh.gated[chunk % 3u].write[16u * t + n] * (1.0f / (kUp * kUp));
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) x[r] = n > 4u * p + r ? w * x[r] * decay[r] : 0.0f;
  put_pieces(sh.solve[chunk % sh.kBlockSets], turned(sh.scratch[t], inverted(x, p, n), p, n), p, n, t, t);
}

// A tile of P out of products of keys and queries.
template <uint32_t STEPS, bool DELTA>
__device__ __forceinline__ void put_mix(ChunkShared<STEPS>& sh, uint32_t chunk, const ScanArgs& a,
                                        f32x4 x, const f32x4& decay, uint32_t ti, uint32_t tj,
                                        uint32_t p, uint32_t n) {
  const Gated& g = sh.gated[chunk % 3u];
  const float f = DELTA ? a.scale * (1.0f / (kUp * kUp)) : g.query[16u * ti + n];
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) {
    x[r] *= f * decay[r];
    if (!DELTA) x[r] *= g.key[16u * tj + 4u * p + r];
    if (ti == tj && n < 4u * p + r) x[r] = 0.0f;
  }
  put_pieces(sh.mix[chunk % sh.kBlockSets], x, p, n, ti, tj);
}

// What has the first sixteen tokens for columns: T00, L10 and two tiles of P.
template <uint32_t STEPS, bool DELTA>
__device__ __forceinline__ void make_first(ChunkShared<STEPS>& sh, uint32_t chunk,
                                           const ScanArgs& a, uint32_t lane) {
  const uint32_t p = lane / 16u, n = lane % 16u;
  const u32x4 *keys = sh.key[chunk % sh.kRowSets], *queries = sh.query[chunk % sh.kRowSets];
  const double* sum = sh.sum[chunk % 2u];
  Tile<STEPS> key, other;
  key.read(keys, 0u, p, n);
  const f32x4 near = between(sum, 0u, 0u, p, n), far = between(sum, 1u, 0u, p, n);
  if (DELTA) {
    other.read(keys, 1u, p, n);
    __builtin_amdgcn_sched_barrier(0);
    const f32x4 x = products(key, key);
    f32x4 low = products(key, other);
    other.read(queries, 0u, p, n);
    put_solve(sh, chunk, x, near, 0u, p, n);
    low *= (sh.gated[chunk % 3u].write[16u + n] * (-1.0f / (kUp * kUp))) * far;
    put_pieces(sh.solve[chunk % sh.kBlockSets], low, p, n, 2u, 0u);
  } else {
    other.read(queries, 0u, p, n);
  }
  put_mix<STEPS, DELTA>(sh, chunk, a, products(key, other), near, 0u, 0u, p, n);
  other.read(queries, 1u, p, n);
  put_mix<STEPS, DELTA>(sh, chunk, a, products(key, other), far, 1u, 0u, p, n);
}
// What has the others for columns: T11 and a tile of P.
template <uint32_t STEPS, bool DELTA>
__device__ __forceinline__ void make_second(ChunkShared<STEPS>& sh, uint32_t chunk,
                                            const ScanArgs& a, uint32_t lane) {
  const uint32_t p = lane / 16u, n = lane % 16u;
  Tile<STEPS> key, query;
  key.read(sh.key[chunk % sh.kRowSets], 1u, p, n);
  query.read(sh.query[chunk % sh.kRowSets], 1u, p, n);
  const f32x4 near = between(sh.sum[chunk % 2u], 1u, 1u, p, n);
  __builtin_amdgcn_sched_barrier(0);
  if (DELTA) put_solve(sh, chunk, products(key, key), near, 1u, p, n);
  put_mix<STEPS, DELTA>(sh, chunk, a, products(key, query), near, 1u, 1u, p, n);
}

// ---- the takers --------------------------------------------------------------------
// Sixteen columns' state: tile k has keys 16 k + 4 p + i of column lane % 16.
// It is held in units of a power of two that keep the column's largest value, or what is added to
// it, in [2^11, 2^15): f16 pieces of such columns reach 2^-22 of that and further.
template <uint32_t STEPS>
struct State {
  f32x4 s[2 * STEPS];
  float unit;  // what one unit is worth

  __device__ __forceinline__ void times(float f) {
#pragma unroll
    for (uint32_t k = 0; k < 2 * STEPS; ++k) s[k] *= f;
  }
  // Units in which a largest value of 2^e of them fits, e biased as f32 exponents are: what all
  // that is held in them is to be multiplied by.  (They stay above 2^-122: what is that small has fewer bits.)
  static __device__ __forceinline__ bool fits(int32_t e) { return (uint32_t)(e - 138) <= 3u; }
  __device__ __forceinline__ float fit(int32_t e, int32_t most = 126) {
    const int32_t now = exponent(unit);
    const int32_t up = fits(e) ? 0 : max(min(141 - e, min(now - 5, most)), now - 240);
    unit = __uint_as_float((uint32_t)(now - up) << 23);
    // (what loses more than 126 bits is nothing beside the largest)
    return __uint_as_float((uint32_t)(127 + max(up, -126)) << 23);
  }
};

struct Column {  // a lane's column, and where its rows are
  const float* v;  // the first token's first column
  float* out;      // the same; null: no outputs
  size_t v_stride, out_stride;
  uint32_t v_at, out_at;  // bytes to row 4 p of a chunk in the lane's column
};

// A chunk token by token.
template <uint32_t STEPS, bool DELTA>
__device__ void take_steps(State<STEPS>& st, const ChunkShared<STEPS>& sh, uint32_t chunk,
                           const Column& c, uint32_t t0, uint32_t left, uint32_t lane, float qscale,
                           float skip) {
  const uint32_t p = lane / 16u, buf = chunk % sh.kRowSets;
  const Gated& g = sh.gated[chunk % 3u];
  // keys 16 k + 4 p + 0..3 of token t
  auto value = [&](const u32x4* from, uint32_t t, uint32_t k, float f) {
    f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t i = 0; i < kHalves; ++i) {
      const u32x2 w = reinterpret_cast<const u32x2*>(
          from + half_fragment<STEPS>(t / 16u, k / 2u, kHalves - 1u - i) +
          place(p, t % 16u, k / 2u))[k % 2u];
      typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
      r += __builtin_convertvector(__builtin_bit_cast(f16x4, w), f32x4);
    }
    return r * f;
  };
  auto total = [](float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
  };
  st.times(st.unit);
  const uint32_t v_at = c.v_at - 16u * p * (uint32_t)c.v_stride;
  const uint32_t out_at =
      p == 0u ? c.out_at : kOutside;  // (one of the four lanes that have a column stores)
  const __amdgpu_buffer_rsrc_t from = rows_of(c.v + t0 * c.v_stride, c.v_stride, left);
  const __amdgpu_buffer_rsrc_t to =
      rows_of(c.out + t0 * c.out_stride, c.out_stride, c.out ? left : 0u);
  for (uint32_t t = 0; t < min(left, kChunk); ++t) {
    const float v = __uint_as_float(
        __builtin_amdgcn_raw_buffer_load_b32(from, v_at + t * 4u * (uint32_t)c.v_stride, 0, 0));
    const float keep = g.keep[t], write = g.write[t];
    const bool factors = !DELTA || g.raised[t / 8u];
    const float kf = (factors ? g.key[t] : 1.0f) * (DELTA ? 1.0f / kUp : 1.0f);
    const float qf = (factors ? g.query[t] : 1.0f) * (DELTA ? qscale / kUp : 1.0f);
    float sk = 0.0f, sq = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < 2 * STEPS; ++k) {
      const f32x4 key = value(sh.key[buf], t, k, kf);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) sk = __builtin_fmaf(key[i], st.s[k][i], sk);
    }
    const float u = DELTA ? write * (v - keep * total(sk)) : write * v;
#pragma unroll
    for (uint32_t k = 0; k < 2 * STEPS; ++k) {
      const f32x4 key = value(sh.key[buf], t, k, kf);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        st.s[k][i] = __builtin_fmaf(key[i], u, keep * st.s[k][i]);
    }
    if (c.out) {
#pragma unroll
      for (uint32_t k = 0; k < 2 * STEPS; ++k) {
        const f32x4 q = value(sh.query[buf], t, k, qf);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) sq = __builtin_fmaf(q[i], st.s[k][i], sq);
      }
      __builtin_amdgcn_raw_buffer_store_b32(
          __float_as_uint(__builtin_fmaf(skip, v, total(sq))), to,
          out_at == kOutside ? kOutside : out_at + t * 4u * (uint32_t)c.out_stride, 0, 0);
    }
  }
  st.unit = 1.0f;
}

// A chunk's products; `v` its values of the lane's column, tokens 16 tile + 4 p + i.
template <uint32_t STEPS, bool DELTA, bool DEEP>
__device__ __forceinline__ void take_chunk(State<STEPS>& st, const ChunkShared<STEPS>& sh,
                                           uint32_t chunk, const Column& c, const f32x4 (&v)[2],
                                           uint32_t t0, uint32_t left, uint32_t lane, float qscale,
                                           float skip) {
  if (!DEEP) asm volatile("" : "+v"(lane));
  const uint32_t p = lane / 16u, n = lane % 16u, buf = chunk % sh.kRowSets;
  const Gated& g = sh.gated[chunk % 3u];
  // Reads of a step are under way while the products of the one before it are made: the
  // compiler left alone puts each read right before its use, and a chunk waits forty times.
  struct Operands {
    u32x4 x[2][kHalves], y[2][kHalves];
  };
  auto read = [&](Operands& o, uint32_t s) {
    const uint32_t at = place(p, n, s);
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
      for (uint32_t i = 0; i < kHalves; ++i) {
        if (DELTA) o.x[t][i] = sh.key[buf][half_fragment<STEPS>(t, s, i) + at];
        o.y[t][i] = sh.query[buf][half_fragment<STEPS>(t, s, i) + at];
      }
  };
  Operands ahead;
  if (DEEP) {
    read(ahead, 0u);
    __builtin_amdgcn_sched_barrier(0);
  }
  f32x4 sk[2], sq[2];
#pragma unroll
  for (uint32_t t = 0; t < 2; ++t) sk[t] = sq[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float most = 0.0f, also = 0.0f;
#pragma unroll
  for (uint32_t k = 0; k < 2 * STEPS; k += 2) {
    most = largest(st.s[k], most);
    also = largest(st.s[k + 1], also);
  }
  most = columns_max(fmaxf(most, also));
  if (__builtin_amdgcn_ballot_w64(most > 0.0f && !st.fits(exponent(most)))) {
    const float up = most > 0.0f ? st.fit(exponent(most)) : 1.0f;
    st.times(up);
    most *= up;
  }
  u32x4 solve[3][kPieces], mix[2][kPieces];
  auto read_solve = [&] {
#pragma unroll
    for (uint32_t t = 0; t < 3; ++t)
#pragma unroll
      for (uint32_t i = 0; i < kPieces; ++i)
        if (DELTA) solve[t][i] = sh.solve[chunk % sh.kBlockSets][fragment(t, i) + place(p, n, 0u)];
  };
  auto read_mix = [&] {
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
      for (uint32_t i = 0; i < kPieces; ++i)
        mix[t][i] = sh.mix[chunk % sh.kBlockSets][fragment(t, i) + place(p, n, 0u)];
  };
#pragma unroll
  for (uint32_t s = 0; s < STEPS; ++s) {
    if (!DEEP) read(ahead, s);
    const Operands o = ahead;
    if (DEEP && s + 1u < STEPS) read(ahead, s + 1u);
    if (DEEP && s + 1u == STEPS) read_solve();
    __builtin_amdgcn_sched_barrier(0);
    u32x4 state[kHalves];
    halve8(st.s[2 * s], st.s[2 * s + 1], state);
#pragma unroll
    for (uint32_t i = 0; i < kHalfPairs; ++i)
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t) {
        if (DELTA) sk[t] = mfma16(o.x[t][kHalfLeft[i]], state[kHalfRight[i]], sk[t]);
        sq[t] = mfma16(o.y[t][kHalfLeft[i]], state[kHalfRight[i]], sq[t]);
      }
    __builtin_amdgcn_sched_barrier(0);
  }
  const float down_k = st.unit * (1.0f / kUp), down_q = st.unit * (DELTA ? qscale / kUp : 1.0f);
  f32x4 grow[2], u[2];
#pragma unroll
  for (uint32_t t = 0; t < 2; ++t) {
    grow[t] = *reinterpret_cast<const f32x4*>(g.grow + 16u * t + 4u * p);
    const f32x4 w = *reinterpret_cast<const f32x4*>(g.write + 16u * t + 4u * p);
    u[t] = DELTA ? w * (v[t] - grow[t] * (sk[t] * down_k)) : w * v[t];
  }
  u32x4 right[kPieces];
  // rows 16 a + 4 p + i of the right operand
  auto put = [&](const f32x4& x, uint32_t a) {
    uint32_t lo[kPieces], hi[kPieces];
    split(x[0], x[1], lo);
    split(x[2], x[3], hi);
#pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
      right[i][2 * a] = lo[i];
      right[i][2 * a + 1] = hi[i];
    }
  };
  auto times = [&](const u32x4 (&left)[kPieces], f32x4 sum) {
    f32x4 more = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t i = 0; i < kPairs; i += 2) {
      more = mfma(left[kLeft[i]], right[kRight[i]], more);
      sum = mfma(left[kLeft[i + 1]], right[kRight[i + 1]], sum);
    }
    return sum + more;
  };
  if (DEEP) read_mix();
  if (DELTA) {
    const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!DEEP) read_solve();
    __builtin_amdgcn_sched_barrier(0);
    put(u[0], 0u);
    put(none, 1u);
    u[0] = times(solve[0], none);
    put(u[0], 0u);
    u[1] = times(solve[2], u[1]);
    put(u[1], 1u);
    u[1] = times(solve[1], none);
    put(u[1], 1u);
  } else {
    put(u[0], 0u);
    put(u[1], 1u);
  }
  const uint32_t raised =
      DELTA ? __builtin_amdgcn_readfirstlane(*reinterpret_cast<const uint32_t*>(g.raised)) : 0u;
  bool odd = raised & (0x01010101u * kRaised);
#pragma unroll
  for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) odd |= __builtin_amdgcn_classf(u[t][i], 0x207);  // NaN, infinity
  // (the steps' code goes behind the rest where that leaves registers: 9.85 against 11.0 us for a call of one chunk)
  const bool steps = __builtin_amdgcn_ballot_w64(odd) != 0u;
  if (DELTA && STEPS <= 4 ? __builtin_expect(steps, false) : steps) {
    take_steps<STEPS, DELTA>(st, sh, chunk, c, t0, left, lane, qscale, skip);
    return;
  }
  {
    if (!DEEP) read_mix();
    f32x4 o[2];
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) {
      o[t] = grow[t] * (sq[t] * down_q);
      if (!DELTA) o[t] *= *reinterpret_cast<const f32x4*>(g.query + 16u * t + 4u * p);
    }
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i)
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t) o[t] = mfma(mix[t][kLeft[i]], right[kRight[i]], o[t]);
    // (last: the sums before it are cut to their own size)
    if (__builtin_amdgcn_readfirstlane(__float_as_uint(skip)))
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) o[t][i] = __builtin_fmaf(skip, v[t][i], o[t][i]);
    if (c.out) {
      const __amdgpu_buffer_rsrc_t to = rows_of(c.out + t0 * c.out_stride, c.out_stride, left);
      uint32_t at = c.out_at;
      if (!DEEP) asm volatile("" : "+v"(at));
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          __builtin_amdgcn_raw_buffer_store_b32(
              __float_as_uint(o[t][i]), to,
              at + (16u * t + i) * 4u * (uint32_t)c.out_stride, 0, 0);
    }
  }
  // the transposing read: a lane points at four keys (4 (lane % 4)..) of token 4 p + lane / 4 % 4
  // and gets four tokens (4 p + 0..3) of key lane % 16
  const uint32_t token = 4u * p + n / 4u, quarter = n % 4u;
  auto turn = [&](u32x4 (&x)[kHalves], uint32_t k) {
#pragma unroll
    for (uint32_t i = 0; i < kHalves; ++i) {
      i16x4 part[2];
#pragma unroll
      for (uint32_t t = 0; t < 2; ++t) {
        const u32x4* from = sh.key[buf] + half_fragment<STEPS>(t, k / 2u, i) +
                            place(quarter, token, k / 2u);
        typedef __attribute__((address_space(3))) i16x4 Local;
        part[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (Local*)(reinterpret_cast<const i16x4*>(from) + k % 2u));
      }
      const u32x2 lo = __builtin_bit_cast(u32x2, part[0]), hi = __builtin_bit_cast(u32x2, part[1]);
      x[i] = u32x4{lo.x, lo.y, hi.x, hi.y};
    }
  };
  f32x4 fade[2];
#pragma unroll
  for (uint32_t t = 0; t < 2; ++t) fade[t] = *reinterpret_cast<const f32x4*>(g.fade + 16u * t + 4u * p);
  float all = g.total;
  u32x4 next[2][kHalves];
  if (DEEP) {
    turn(next[0], 0u);
    turn(next[1], 1u);
    __builtin_amdgcn_sched_barrier(0);
  }
  float gained = 0.0f;
  if (__builtin_expect(raised != 0u, false)) {
    // (a key of zeros adds nothing, however large its u: the units are the others')
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t)
      if (raised >> (8u * (2u * t + p / 2u)) & kZeros)
        u[t] *= *reinterpret_cast<const f32x4*>(g.key + 16u * t + 4u * p);
  }
#pragma unroll
  for (uint32_t t = 0; t < 2; ++t) {
    u[t] *= fade[t];
    if (!DELTA) u[t] *= *reinterpret_cast<const f32x4*>(g.key + 16u * t + 4u * p);
    gained = largest(u[t], gained);
  }
  // The larger of what the column gains and what is left of its state has to fit.  (By their
  // exponents: one may be more than f32's largest number times the other.)
  const float rest = all * most;
  gained = columns_max(gained);
  const int32_t size =
      max(exponent(rest), exponent(gained) - exponent(st.unit) + (DELTA ? 127 : 135));
  const bool some = rest > 0.0f || gained > 0.0f;
  if (__builtin_amdgcn_ballot_w64(some && !st.fits(size))) {
    // (the state is multiplied once, by both: what is forgotten may not fit the new units)
    if (some) all *= st.fit(size, min(126, 253 - exponent(all)));
  }
  // (the unit is a power of two, and so is its inverse)
  const float gain =
      __uint_as_float((254u << 23) - __float_as_uint(st.unit)) * (DELTA ? 1.0f / kUp : 1.0f);
  u32x4 gains[kHalves];
  halve8(u[0] * gain, u[1] * gain, gains);
#pragma unroll
  for (uint32_t k = 0; k < 2 * STEPS; k += 2) {
    u32x4 x[2][kHalves];
    if (!DEEP) {
      turn(next[0], k);
      turn(next[1], k + 1u);
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
      for (uint32_t i = 0; i < kHalves; ++i) x[h][i] = next[h][i];
    if (DEEP && k + 2u < 2 * STEPS) {
      turn(next[0], k + 2u);
      turn(next[1], k + 3u);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) st.s[k + h] *= all;
#pragma unroll
    for (uint32_t i = 0; i < kHalfPairs; ++i)
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h)
        st.s[k + h] = mfma16(x[h][kHalfLeft[i]], gains[kHalfRight[i]], st.s[k + h]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A workgroup: 16 TAKERS columns of one head of one sequence; grid (column blocks * heads, sequences).
// At step n of its course chunk n's rows and gates and chunk n - 1's blocks are made, and chunk n - 2 is taken;
// where LDS is tight, chunk n's rows and gates while chunk n - 1 is taken, then chunk n's blocks.
template <uint32_t STEPS, bool DELTA, uint32_t TAKERS>
__global__ __launch_bounds__(64 * waves_of(STEPS, TAKERS))
__attribute__((amdgpu_waves_per_eu(waves_of(STEPS, TAKERS) / 4))) void scan_chunks_kernel(ScanArgs a,
                                                                              uint32_t blocks) {
  __shared__ ChunkShared<STEPS> sh;
  constexpr bool TIGHT = ChunkShared<STEPS>::kTight;
  constexpr bool DEEP = TIGHT ? TAKERS < 4 && !DELTA : TAKERS < 8;  // (registers for reads ahead)
  constexpr uint32_t BEHIND = TIGHT ? 0 : 1;  // chunks from rows to blocks
  const uint32_t lane = threadIdx.x % 64u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
  const uint32_t seq = blockIdx.y, head = blockIdx.x / blocks, block = blockIdx.x % blocks;
  const uint32_t count = __builtin_amdgcn_readfirstlane(tokens_of(a.count, seq));
  const uint32_t chunks = (count + kChunk - 1u) / kChunk;
  const size_t row0 = (size_t)seq * a.count.tokens;
  const uint32_t dk = a.key_dim, dv = a.value_dim;
  if (wave >= TAKERS + 2u) {
    const uint32_t maker = wave - TAKERS - 2u, key_head = key_head_of(a, head);
    constexpr uint32_t MAKERS = row_makers(STEPS, TAKERS);
    using W = Raw<STEPS, MAKERS>;
    W raw;
    const float* k = a.k + row0 * a.k_stride + (size_t)key_head * dk;
    const float* q = a.out ? a.q + row0 * a.q_stride + (size_t)key_head * dk : a.k;
    fetch<STEPS, MAKERS>(raw, a, k, q, maker * W::kParts, lane, count);
    for (uint32_t n = 0; n < chunks + 1u + BEHIND; ++n) {
      const uint32_t left = count - min(count, n * kChunk);
      if (left) {
        make_rows<STEPS, DELTA, MAKERS>(sh, n, raw, a, maker * W::kParts, lane, left);
#pragma unroll
        for (uint32_t part = 1; part < W::kParts; ++part) {
          fetch<STEPS, MAKERS>(raw, a, k, q, maker * W::kParts + part, lane, left);
          make_rows<STEPS, DELTA, MAKERS>(sh, n, raw, a, maker * W::kParts + part, lane, left);
        }
        k += kChunk * a.k_stride;
        if (a.out) q += kChunk * a.q_stride;
        if (left > kChunk) fetch<STEPS, MAKERS>(raw, a, k, q, maker * W::kParts, lane, left - kChunk);
      }
      exchange_barrier();
      if (TIGHT) exchange_barrier();
    }
    return;
  }
  if (wave == TAKERS) {
    // the blocks of zeros stay: the upper ones of P and beside T00, T11 and -L10
#pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i)
#pragma unroll
      for (uint32_t b = 0; b < sh.kBlockSets; ++b) {
        reinterpret_cast<u32x2*>(sh.mix[b] + fragment(0, i) + lane)[1] = u32x2{0u, 0u};
        reinterpret_cast<u32x2*>(sh.solve[b] + fragment(0, i) + lane)[1] = u32x2{0u, 0u};
        reinterpret_cast<u32x2*>(sh.solve[b] + fragment(1, i) + lane)[0] = u32x2{0u, 0u};
        reinterpret_cast<u32x2*>(sh.solve[b] + fragment(2, i) + lane)[1] = u32x2{0u, 0u};
      }
    for (uint32_t n = 0; n < chunks + 1u + BEHIND; ++n) {
      if (TIGHT) exchange_barrier();
      if (n >= BEHIND && n - BEHIND < chunks) make_first<STEPS, DELTA>(sh, n - BEHIND, a, lane);
      exchange_barrier();
    }
    return;
  }
  if (wave == TAKERS + 1u) {
    const float decay = a.decay[head], bias = a.bias ? a.bias[head] : 0.0f;
    const float* gate = a.gate + (row0 + lane) * a.value_heads + head;
    const float* beta = DELTA ? a.beta + (row0 + lane) * a.value_heads + head : nullptr;
    const size_t gate_step = (size_t)kChunk * a.value_heads;
    float gx = 0.0f, bx = 0.0f;  // the next chunk's gates
    auto fetch_gates = [&](uint32_t n) {
      if (lane < kChunk && n * kChunk + lane < count) {
        gx = gate[n * gate_step];
        if (DELTA) bx = beta[n * gate_step];
      }
    };
    fetch_gates(0u);
    for (uint32_t n = 0; n < chunks + 1u + BEHIND; ++n) {
      if (n < chunks) {
        make_gates<STEPS, DELTA>(sh, n, a, lane, gx, bx, decay, bias, count - n * kChunk);
        fetch_gates(n + 1u);
      }
      if (TIGHT) exchange_barrier();
      if (n >= BEHIND && n - BEHIND < chunks) make_second<STEPS, DELTA>(sh, n - BEHIND, a, lane);
      exchange_barrier();
    }
    return;
  }
  __builtin_amdgcn_s_setprio(2);  // (before the makers of their SIMD: 1.5 % of a chunk)
  const uint32_t p = lane / 16u, col = block * 16u * TAKERS + wave * 16u + lane % 16u;
  const bool there = col < dv;
  Column c;
  c.v = a.v + row0 * a.v_stride + (size_t)head * dv;
  c.v_stride = a.v_stride;
  c.out = a.out ? a.out + (row0 * a.value_heads + head) * dv : nullptr;
  c.out_stride = (size_t)a.value_heads * dv;
  // (a column that is not there reads zeros and writes nothing)
  c.v_at = there ? 4u * (4u * p * (uint32_t)c.v_stride + col) : kOutside;
  c.out_at = there ? 4u * (4u * p * (uint32_t)c.out_stride + col) : kOutside;
  // (keys behind the last are behind the state's buffer)
  const size_t state0 = ((size_t)seq * a.value_heads + head) * dk * dv;
  uint32_t state_at = there ? 4u * (4u * p * dv + col) : kOutside;
  State<STEPS> st;
  st.unit = 1.0f;
  {
    const __amdgpu_buffer_rsrc_t from =
        buffer_of(a.state + state0, a.state ? 4u * dk * dv : 0u);
#pragma unroll
    for (uint32_t k = 0; k < 2 * STEPS; ++k)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        st.s[k][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            from, state_at + (16u * k + i) * 4u * dv, 0, 0));
  }
  // (it is there before the first chunk: else every chunk waits for all loads that are under way)
#pragma unroll
  for (uint32_t k = 0; k < 2 * STEPS; ++k) asm volatile("" : "+v"(st.s[k]));
  const float skip = a.skip ? a.skip[head] : 0.0f;
  f32x4 v[2];
  auto values = [&](uint32_t t0) {
    const __amdgpu_buffer_rsrc_t from =
        rows_of(c.v + t0 * c.v_stride, c.v_stride, count - min(count, t0));
    uint32_t at = c.v_at;
    if (!DEEP) asm volatile("" : "+v"(at));  // (offsets anew: no registers held for them)
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        v[t][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            from, at + (16u * t + i) * 4u * (uint32_t)c.v_stride, 0, 0));
  };
  if (DEEP) values(0u);
  exchange_barrier();
  exchange_barrier();
  for (uint32_t n = 0; n < chunks; ++n) {
    const uint32_t t0 = n * kChunk;
    if (!DEEP) values(t0);
    const f32x4 now[2] = {v[0], v[1]};
    if (DEEP) values(t0 + kChunk);
    take_chunk<STEPS, DELTA, DEEP>(st, sh, n, c, now, t0, count - t0, lane, a.scale, skip);
    exchange_barrier();
    if (TIGHT) exchange_barrier();
  }
  if (a.state_out) {
    const __amdgpu_buffer_rsrc_t to = buffer_of(a.state_out + state0, 4u * dk * dv);
    asm volatile("" : "+v"(state_at));  // (offsets anew, as above)
#pragma unroll
    for (uint32_t k = 0; k < 2 * STEPS; ++k)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(st.s[k][i] * st.unit), to,
                                              state_at + (16u * k + i) * 4u * dv, 0, 0);
  }
}

template <uint32_t TAKERS>
hipError_t launch(const ScanArgs& a, hipStream_t s) {
  const uint32_t blocks = (a.value_dim + 16u * TAKERS - 1u) / (16u * TAKERS);
  const dim3 grid(blocks * a.value_heads, a.sequences);
  auto go = [&](auto steps) {
    constexpr uint32_t STEPS = decltype(steps)::value;
    if constexpr (STEPS > 4 && TAKERS == 8)
      return hipErrorInvalidValue;
    else if (a.delta)
      scan_chunks_kernel<STEPS, true, TAKERS>
          <<<grid, 64u * waves_of(STEPS, TAKERS), 0, s>>>(a, blocks);
    else
      scan_chunks_kernel<STEPS, false, TAKERS>
          <<<grid, 64u * waves_of(STEPS, TAKERS), 0, s>>>(a, blocks);
    return hipGetLastError();
  };
  using std::integral_constant;
  switch ((a.key_dim + 31u) / 32u) {
    case 1: return go(integral_constant<uint32_t, 1>{});
    case 2: return go(integral_constant<uint32_t, 2>{});
    case 3: return go(integral_constant<uint32_t, 3>{});
    case 4: return go(integral_constant<uint32_t, 4>{});
    case 5: case 6: return go(integral_constant<uint32_t, 6>{});
    default: return go(integral_constant<uint32_t, 8>{});
  }
}

// Columns a workgroup has: the more, the fewer make the same operands twice, but the longer a chunk takes
// (two, four and eight takers 5, 6 and 9 thousand cycles, key_dim 128) and the fewer workgroups there
// are for the card's 256 CUs, each of which holds one: what takes the fewest cycles in whole rounds.  (Below 33 keys LDS
// has room for two, but 192 workgroups take 61 us and 384 of them 113.)  1024 tokens of 48 heads of 128 x 128, delta rule: one sequence 83 us with two, 90 with four, 125 with
// eight; two of them 153, 92, 125; four 230, 180, 131; eight 458, 302, 268.  The same order within 4 % for keys of
// 32, 64 and 256 and the selective form: four sequences of 32 keys 166, 136, 90, of 64 184, 157, 104, of 256 502,
// 373 (no eight); selective ones 117, 63, 59, 136, 99, 68, 337, 307, of 128 184, 142, 100.
struct Shape {
  uint32_t takers;
  uint64_t rounds;
};
Shape shape_for(const ScanArgs& a) {
  const uint64_t heads = (uint64_t)a.value_heads * a.sequences;
  Shape best{0u, 0u};
  uint64_t least = ~uint64_t(0);
  for (uint32_t takers : {2u, 4u, 8u}) {
    if (takers == 8u && a.key_dim > 128u) continue;  // (their registers would not do)
    const uint64_t groups = heads * ((a.value_dim + 16u * takers - 1u) / (16u * takers));
    const uint64_t rounds = (groups + 255u) / 256u;
    const uint64_t cycles = rounds * (takers == 2u ? 11u : takers == 4u ? 13u : 19u);
    if (cycles < least) {
      least = cycles;
      best = Shape{takers, rounds};
    }
  }
  return best;
}

}  // namespace

// (A chunk's rows lie within the 2^30 bytes that its buffers' offsets reach.)  Where one round of workgroups takes
// them four tokens are faster in a chunk than token by token: 48 heads of 128 x 128, delta rule, chunks /
// steps, 4 tokens of one sequence 7.6 / 11.2 us, of four 10.8 / 13.0; of 64 x 64 6.1 / 7.5, 6.7 / 8.0; of one sequence of 256 x 128
// 10.4 / 14.4.  With more rounds a chunk costs the same for all lengths, steps by the state: 48 sequences of 48
// heads, 8, 12 and 16 tokens, 128 x 128 96 / 95, 96 / 124, 97 / 150; 64 x 128 64 / 44, 63 / 57, 63 / 69;
// 96 x 96 76 / 59, 76 / 79, 76 / 96; 64 x 64 50 / 29, 50 / 38, 51 / 46; 32 x 128 50 / 29, 50 / 40, 50 / 48. 12
// sequences: 128 x 128 32 / 38, 33 / 49, 33 / 59; 64 x 128 21 / 19, 22 / 25, 22 / 30; 64 x 64 17 / 14, 18 / 19, 18 / 23.
// The selective form the same way: 48 sequences 128 x 128 79 / 84, 79 / 105, 80 / 124; 64 x 128 50 / 39, 50 / 48,
// 49 / 56; 64 x 64 41 / 25, 41 / 32, 42 / 38.
bool scan_chunks_take(const ScanArgs& a) {
  constexpr size_t most = size_t(1) << 23;
  const uint32_t state = a.key_dim * a.value_dim;
  const uint32_t enough = state >= 128u * 128u ? 8u : state > 64u * 64u ? 12u : 16u;
  return a.k_stride <= most && a.v_stride <= most &&
         (!a.out || (a.q_stride <= most && (size_t)a.value_heads * a.value_dim <= most)) &&
         (a.count.tokens >= enough || (a.count.tokens >= 4u && shape_for(a).rounds == 1u));
}

hipError_t launch_scan_chunks(const ScanArgs& a, hipStream_t s) {
  const uint32_t takers = shape_for(a).takers;
  return takers == 2u ? launch<2>(a, s) : takers == 4u ? launch<4>(a, s) : launch<8>(a, s);
}

}  // namespace sihip
