// Norms of query and key heads, their rotation by positions of one or several
// axes, and new tokens' rows into the paged cache, in one pass.
//
// A head x becomes y = x (shift + w) / sqrt(mean x^2 + eps); pair (a, b) of y
// turns by p f_i turns as in kernels_rope.hip, p being the row's position on
// pair i's axis.  Memory is all there is to it: each row is read once, held in
// the registers of the 16 lanes that have it (64 where it is no whole sixteen bytes)
// while they add up its squares, and written once.  Prompts of 368 MB take 75.5 us into the
// cache (4.9 TB/s, what a copy reaches), rows of 492 MB by themselves 98 us (5.0 TB/s); a
// single token's heads 5.3 us, a launch and the chain from page number to slot.  (kernels_rope.hip, the
// same without norms and axes, deals a row's pairs to any thread: heads of 72 take 26.2 us there and 27.8 here,
// single tokens 4.8 and 5.2; heads of 128 71.4 and 70.7, of 255 46.8 and 35.3.)
#include "rope_units.h"

namespace sihip {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kTokens = 8;  // tokens a workgroup has at most

// What every row of a call shares.
struct Turns {
  NormArgs norm;
  RopeArgs rope;
  AxesArgs axes;
  const uint32_t* positions;  // [axes][rows]; null: the slots' numbers
  size_t rows;
};

// In LDS: the cosines and sines of a workgroup's tokens, times the magnitude, and
// the two norms' factors.
struct Shared {
  float cs[kTokens][kMaxHeadDim / 2], sn[kTokens][kMaxHeadDim / 2];
  float wq[kMaxHeadDim], wk[kMaxHeadDim];
};

// Fills it for `count` tokens from row `row` on; position_of(t) is a token's where there are none.
template <class F>
__device__ __forceinline__ void fill(Shared& sh, const Turns& a, size_t row, uint32_t count,
                                     uint32_t dim, bool keys, void* ws, F position_of) {
  const uint32_t half = a.rope.rotary_dim / 2u;
  for (uint32_t i = threadIdx.x; i < half * count; i += kThreads) {
    const uint32_t t = i / half, pair = i - t * half;
    uint32_t axis = 0u;
    if (a.axes.axis) {
      axis = a.axes.axis[pair];
      if (axis >= a.axes.axes) {
        report_device_error(ws, kDevErrRopeAxis);
        axis = 0u;
      }
    }
    const uint32_t p = a.positions ? a.positions[axis * a.rows + row + t] : position_of(t);
    const uint64_t phase = a.rope.frequencies[pair] * p;
    float s, c;
    sincospif((float)(int64_t)phase * 0x1p-63f, &s, &c);
    sh.cs[t][pair] = c * a.rope.magnitude;
    sh.sn[t][pair] = s * a.rope.magnitude;
  }
  if (a.norm.on)
    for (uint32_t i = threadIdx.x; i < dim; i += kThreads) {
      sh.wq[i] = a.norm.q ? a.norm.shift + a.norm.q[i] : 1.0f;
      if (keys) sh.wk[i] = a.norm.k ? a.norm.shift + a.norm.k[i] : 1.0f;
    }
  __syncthreads();
}

// One row by the LANES lanes that have it, K units each at most: N = 4: sixteen bytes at a time, N =
// 1: single values (row_units).
template <uint32_t N, uint32_t K, uint32_t LANES, typename T>
__device__ __forceinline__ void norm_row(uint32_t lane, Row<T> r, const Turns& a, uint32_t dim,
                                         uint32_t units, const float* w, const float* cs,
                                         const float* sn) {
  const uint32_t n = a.rope.rotary_dim, half = n / 2u;
  const bool pairs = a.rope.layout == 1u;
  constexpr uint32_t P = N == 4 ? 2u : 1u;  // pairs of a unit of the interleaved layout
  const uint32_t turning = pairs ? half / P : half / N;
  float x[K][2 * N];
  float squares = 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < K; ++j) {
    const uint32_t u = lane + j * LANES;
#pragma unroll
    for (uint32_t i = 0; i < 2 * N; ++i) x[j][i] = 0.0f;
    if (u < units) {
      if (u >= turning) {
        load_units<N>(x[j], r.x + n + N * (u - turning));
      } else if (pairs) {
        load_units<2 * P>(x[j], r.x + 2u * P * u);
      } else {
        load_units<N>(x[j], r.x + N * u);
        load_units<N>(x[j] + N, r.x + half + N * u);
      }
    }
  }
  if (a.norm.on) {
#pragma unroll
    for (uint32_t j = 0; j < K; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 2 * N; ++i) squares = __builtin_fmaf(x[j][i], x[j][i], squares);
#pragma unroll
    for (uint32_t m = 1; m < LANES; m *= 2) squares += __shfl_xor(squares, m);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(squares / (float)dim + a.norm.eps));
#pragma unroll
    for (uint32_t j = 0; j < K; ++j) {
      const uint32_t u = lane + j * LANES;
      if (u >= units) continue;
      float f[2 * N] = {};
      if (u >= turning) {
        load_units<N>(f, w + n + N * (u - turning));
      } else if (pairs) {
        load_units<2 * P>(f, w + 2u * P * u);
      } else {
        load_units<N>(f, w + N * u);
        load_units<N>(f + N, w + half + N * u);
      }
#pragma unroll
      for (uint32_t i = 0; i < 2 * N; ++i) x[j][i] = x[j][i] * inv * f[i];
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < K; ++j) {
    const uint32_t u = lane + j * LANES;
    if (u >= units) continue;
    if (u >= turning) {
      store_units<N>(r.y + n + N * (u - turning), x[j]);
    } else if (pairs) {
      float y[2 * P];
#pragma unroll
      for (uint32_t i = 0; i < P; ++i) {
        const float c = cs[P * u + i], s = sn[P * u + i];
        y[2 * i] = x[j][2 * i] * c - x[j][2 * i + 1] * s;
        y[2 * i + 1] = x[j][2 * i + 1] * c + x[j][2 * i] * s;
      }
      store_units<2 * P>(r.y + 2u * P * u, y);
    } else {
      float y[N], z[N];
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        const float c = cs[N * u + i], s = sn[N * u + i];
        y[i] = x[j][i] * c - x[j][i + N] * s;
        z[i] = x[j][i + N] * c + x[j][i] * s;
      }
      store_units<N>(r.y + N * u, y);
      store_units<N>(r.y + half + N * u, z);
    }
  }
}

constexpr uint32_t lanes_of(uint32_t n) { return n == 4u ? 16u : 64u; }

// grid (groups of `each` tokens, slices): the slice's share of the tokens' heads
template <uint32_t N, uint32_t K>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(Turns a, RopeRows rows,
                                                             uint32_t head_dim, uint32_t tokens,
                                                             uint32_t each, Divisor by_heads,
                                                             void* ws) {
  __shared__ Shared sh;
  constexpr uint32_t L = lanes_of(N);
  const uint32_t t0 = blockIdx.x * each, count = min(each, tokens - t0);
  fill(sh, a, t0, count, head_dim, false, ws, [](uint32_t) { return 0u; });
  const uint32_t units = row_units(a.rope.rotary_dim, head_dim, a.rope.layout, N);
  const uint32_t all = count * rows.heads;
  const uint32_t i0 = (uint32_t)((uint64_t)all * blockIdx.y / gridDim.y);
  const uint32_t i1 = (uint32_t)((uint64_t)all * (blockIdx.y + 1u) / gridDim.y);
  for (uint32_t i = i0 + threadIdx.x / L; i < i1; i += kThreads / L) {
    const uint32_t t = by_heads.of(i), h = i - t * rows.heads;
    const size_t row = t0 + t;
    norm_row<N, K, L>(threadIdx.x % L,
                      Row<float>{rows.x + row * rows.token_stride + h * rows.head_stride,
                                 rows.y + row * rows.y_token_stride + h * rows.y_head_stride},
                      a, head_dim, units, sh.wq, sh.cs[t], sh.sn[t]);
  }
}

// grid (groups of `each` rows from `first` on, slices), of sequences * tokens
template <uint32_t N, uint32_t K, typename T>
__global__ __launch_bounds__(kThreads) void norm_rope_append_kernel(
    CacheView cache, Turns a, uint32_t first, uint32_t rows, uint32_t tokens, uint32_t each,
    Divisor by_heads, const uint32_t* __restrict__ counts, const float* __restrict__ k,
    size_t k_stride, const float* __restrict__ v, size_t v_stride, RopeRows q, void* ws) {
  __shared__ Shared sh;
  __shared__ uint32_t place[kTokens];  // the row's slot in the pool, head 0
  __shared__ uint32_t there[kTokens];
  constexpr uint32_t L = lanes_of(N);
  const uint32_t row0 = first + blockIdx.x * each, count = min(each, rows - blockIdx.x * each);
  auto slot_of = [&](uint32_t t) {
    const uint32_t row = row0 + t, seq = row / tokens;
    return held(cache, seq) + (row - seq * tokens);
  };
  if (threadIdx.x < count) {
    const uint32_t row = row0 + threadIdx.x, seq = row / tokens;
    const bool in = row - seq * tokens < brought(counts, seq, tokens);
    uint32_t at = kNone;
    if (in) {
      const uint32_t slot = slot_of(threadIdx.x);
      if (slot < cache.capacity) at = cache_row(cache, seq, 0u, slot);
      if (at == kNone && blockIdx.y == 0u)
        report_device_error(ws, slot < cache.capacity ? kDevErrCachePage : kDevErrCacheFull);
    }
    place[threadIdx.x] = at;
    there[threadIdx.x] = in;
  }
  fill(sh, a, row0, count, cache.head_dim, true, ws, slot_of);
  const uint32_t dim = cache.head_dim, heads = q.heads + 2u * cache.kv_heads;
  const uint32_t units = row_units(a.rope.rotary_dim, dim, a.rope.layout, N);
  const uint32_t all = count * heads, lane = threadIdx.x % L;
  const uint32_t i0 = (uint32_t)((uint64_t)all * blockIdx.y / gridDim.y);
  const uint32_t i1 = (uint32_t)((uint64_t)all * (blockIdx.y + 1u) / gridDim.y);
  for (uint32_t i = i0 + threadIdx.x / L; i < i1; i += kThreads / L) {
    const uint32_t t = by_heads.of(i), h = i - t * heads;
    if (!there[t]) continue;
    const size_t row = row0 + t;
    const uint32_t at = place[t];
    if (h < q.heads) {
      norm_row<N, K, L>(lane,
                        Row<float>{q.x + row * q.token_stride + h * q.head_stride,
                                   q.y + (row * q.heads + h) * dim},
                        a, dim, units, sh.wq, sh.cs[t], sh.sn[t]);
    } else if (at != kNone) {
      const uint32_t kh = h - q.heads;
      const bool value = kh >= cache.kv_heads;
      const uint32_t kv = value ? kh - cache.kv_heads : kh;
      const size_t to = ((size_t)at + (size_t)kv * cache.page_tokens) * dim;
      if (value) {
        const float* x = v + row * v_stride + (size_t)kv * dim;
        for (uint32_t u = lane; u < dim / N; u += L) {
          float f[N];
          load_units<N>(f, x + N * u);
          store_units<N>((T*)cache.values + to + N * u, f);
        }
      } else {
        norm_row<N, K, L>(lane, Row<T>{k + row * k_stride + (size_t)kv * dim, (T*)cache.keys + to},
                          a, dim, units, sh.wk, sh.cs[t], sh.sn[t]);
      }
    }
  }
}

// Whether sixteen-byte units cover a row: its rotated part is whole units of
// them (half layout: each half), and so is the rest.
bool whole_units(uint32_t n, uint32_t dim, uint32_t layout) {
  return dim % 4u == 0u && n % (layout == 1u ? 4u : 8u) == 0u;
}

// Tokens a workgroup has, so that few heads fill its groups of lanes too, and
// slices of its rows where there are few tokens.
struct Shape {
  uint32_t each, slices;
};
Shape shape_for(uint32_t rows, uint32_t heads) {
  uint32_t each = std::max(1u, std::min(kTokens, 32u / heads));
  while (each > 1u && rows / each < 1024u) each /= 2u;
  const uint32_t groups = (rows + each - 1u) / each;
  const uint32_t want = (1024u + groups - 1u) / groups;
  return {each, std::max(1u, std::min(want, each * heads))};
}

// A launch takes less than 2^32 threads in x: more rows are several.
constexpr uint32_t kMostGroups = 0xffffffffu / kThreads;

// f(N, K) as constants: units of sixteen bytes or of single values, and how many a
// lane has.
template <class F>
hipError_t with_units(bool whole, uint32_t n, uint32_t dim, uint32_t layout, F f) {
  const uint32_t N = whole ? 4u : 1u;
  const uint32_t rotated = N == 4u && layout == 1u ? n / 4u : n / (2u * N);
  const uint32_t units = rotated + (dim - n) / N, lanes = lanes_of(N);
  using std::integral_constant;
  integral_constant<uint32_t, 1> one;
  integral_constant<uint32_t, 2> two;
  integral_constant<uint32_t, 4> four;
  if (whole) return units <= lanes ? f(four, one) : units <= 2u * lanes ? f(four, two) : f(four, four);
  return units <= lanes ? f(one, one) : units <= 2u * lanes ? f(one, two) : f(one, four);
}

}  // namespace

hipError_t launch_norm_rope(const NormArgs& norm, const RopeArgs& rope, const AxesArgs& axes,
                            const RopeRows& rows, uint32_t tokens, uint32_t head_dim,
                            const uint32_t* positions, void* ws, hipStream_t s) {
  const Shape shape = shape_for(tokens, rows.heads);
  const uint32_t most = kMostGroups / kTokens * kTokens;
  return with_units(
      whole_units(rope.rotary_dim, head_dim, rope.layout), rope.rotary_dim, head_dim, rope.layout,
      [&](auto n, auto k) {
        for (uint32_t t0 = 0; t0 < tokens; t0 += std::min(most, tokens - t0)) {
          const uint32_t part_tokens = std::min(most, tokens - t0);
          const Turns a{norm, rope, axes, positions ? positions + t0 : nullptr, tokens};
          RopeRows part = rows;
          part.x += t0 * rows.token_stride;
          part.y += t0 * rows.y_token_stride;
          const dim3 grid((part_tokens + shape.each - 1u) / shape.each, shape.slices);
          norm_rope_kernel<decltype(n)::value, decltype(k)::value><<<grid, kThreads, 0, s>>>(
              a, part, head_dim, part_tokens, shape.each, divisor_of(rows.heads), ws);
          const hipError_t e = hipGetLastError();
          if (e != hipSuccess) return e;
        }
        return hipSuccess;
      });
}

hipError_t launch_norm_rope_append(const CacheView& cache, const NormArgs& norm,
                                   const RopeArgs& rope, const AxesArgs& axes, uint32_t tokens,
                                   const uint32_t* counts, const uint32_t* positions,
                                   const float* k, size_t k_stride, const float* v,
                                   size_t v_stride, const RopeRows* q, void* ws, hipStream_t s) {
  const RopeRows qr = q ? *q : RopeRows{};
  const uint32_t rows = cache.sequences * tokens, heads = qr.heads + 2u * cache.kv_heads;
  const Shape shape = shape_for(rows, heads);
  const Turns a{norm, rope, axes, positions, rows};
  const uint32_t most = kMostGroups / kTokens * kTokens;
  const bool whole = whole_units(rope.rotary_dim, cache.head_dim, rope.layout) &&
                     aligned4(cache.keys) && aligned4(cache.values);
  return with_units(whole, rope.rotary_dim, cache.head_dim, rope.layout, [&](auto n, auto kk) {
    constexpr uint32_t N = decltype(n)::value, K = decltype(kk)::value;
    auto go = [&](auto kernel) {
      for (uint32_t r0 = 0; r0 < rows; r0 += std::min(most, rows - r0)) {
        const uint32_t part = std::min(most, rows - r0);
        const dim3 grid((part + shape.each - 1u) / shape.each, shape.slices);
        kernel<<<grid, kThreads, 0, s>>>(cache, a, r0, part, tokens, shape.each,
                                         divisor_of(heads), counts, k, k_stride, v, v_stride, qr,
                                         ws);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
      }
      return hipSuccess;
    };
    if (cache.type == kKvF32) return go(norm_rope_append_kernel<N, K, float>);
    if (cache.type == kKvF16) return go(norm_rope_append_kernel<N, K, __half>);
    return go(norm_rope_append_kernel<N, K, __hip_bfloat16>);
  });
}

}  // namespace sihip
