// Rotary positions, and new tokens' rows into the paged cache.
//
// Pair (a, b) of a head turns by an angle of p f_i turns: (a cos - b sin,
// b cos + a sin) times the magnitude.  f_i is a 64-bit fraction of a turn, so
// the position's whole turns drop out in one wrapping product and what is
// left, in [-1/2, 1/2), is exact before it is rounded to 32 bits.
//
// Memory is all there is to it: each row is read once and written once.  A
// workgroup takes the rows of one token, or a slice of them where there are
// few tokens, and computes the token's cosines and sines once, in LDS.  Four
// prompts of 2043 tokens of 32 + 8 + 8 heads of 128 into an F16 cache: 71 us
// for 368 MB, 5.2 TB/s; by single pairs 125.  One token of 24 + 4 + 4 heads of
// 256: 5.1 us, of which an empty launch has 3.7.
#include "decode_internal.h"

namespace sihip {
namespace {

constexpr uint32_t kThreads = 256;

template <typename T>
__device__ __forceinline__ T to_type(float v);
template <>
__device__ __forceinline__ float to_type<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half to_type<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __hip_bfloat16 to_type<__hip_bfloat16>(float v) {
  return __float2bfloat16(v);
}

// What a workgroup does with one row: a source, and where it goes.
template <typename T>
struct Row {
  const float* x;
  T* y;
};

template <uint32_t N, typename T>
__device__ __forceinline__ void store_units(T* y, const float* v) {
  if constexpr (N == 4 && sizeof(T) == 2) {
    union { T t[4]; Words2 u; } w;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) w.t[i] = to_type<T>(v[i]);
    *reinterpret_cast<Words2*>(y) = w.u;
  } else if constexpr (N == 4) {
    *reinterpret_cast<Floats4*>(y) = Floats4{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) y[i] = to_type<T>(v[i]);
  }
}
template <uint32_t N>
__device__ __forceinline__ void load_units(float* v, const float* x) {
  if constexpr (N == 4) {
    const Floats4 f = *reinterpret_cast<const Floats4*>(x);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = x[i];
  }
}

// Units of a row that a thread takes one of.  N = 4: sixteen bytes at a time,
// four pairs of the half layout or two of the interleaved; N = 1: one pair, or
// one value behind the rotated ones, for sizes that are no whole units and
// 16-bit pools on odd halves of a word.  A pair is one thread's,
// so a row may be rotated in place.
__device__ __forceinline__ uint32_t row_units(uint32_t n, uint32_t dim, uint32_t layout,
                                              uint32_t N) {
  const uint32_t rotated = N == 4 && layout == 1u ? n / 4u : n / (2u * N);
  return rotated + (dim - n) / N;
}
template <uint32_t N, typename T>
__device__ __forceinline__ void do_unit(uint32_t u, Row<T> r, uint32_t n, uint32_t layout,
                                        const float* cs, const float* sn) {
  const uint32_t half = n / 2u;
  if (layout == 1u) {
    constexpr uint32_t P = N == 4 ? 2u : 1u;  // pairs a unit
    if (u < half / P) {
      float x[2 * P], y[2 * P];
      load_units<2 * P>(x, r.x + 2u * P * u);
#pragma unroll
      for (uint32_t i = 0; i < P; ++i) {
        const float c = cs[P * u + i], s = sn[P * u + i];
        y[2 * i] = x[2 * i] * c - x[2 * i + 1] * s;
        y[2 * i + 1] = x[2 * i + 1] * c + x[2 * i] * s;
      }
      store_units<2 * P>(r.y + 2u * P * u, y);
      return;
    }
    u -= half / P;
  } else {
    if (u < half / N) {
      float a[N], b[N], y[N], z[N];
      load_units<N>(a, r.x + N * u);
      load_units<N>(b, r.x + half + N * u);
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        const float c = cs[N * u + i], s = sn[N * u + i];
        y[i] = a[i] * c - b[i] * s;
        z[i] = b[i] * c + a[i] * s;
      }
      store_units<N>(r.y + N * u, y);
      store_units<N>(r.y + half + N * u, z);
      return;
    }
    u -= half / N;
  }
  float x[N];
  load_units<N>(x, r.x + n + N * u);
  store_units<N>(r.y + n + N * u, x);
}

// The cosines and sines of a position, times the magnitude, into LDS.
__device__ __forceinline__ void fill_turns(const RopeArgs& rope, uint32_t position, float* cs,
                                           float* sn) {
  for (uint32_t i = threadIdx.x; i < rope.rotary_dim / 2u; i += kThreads) {
    const uint64_t phase = rope.frequencies[i] * position;
    float s, c;
    sincospif((float)(int64_t)phase * 0x1p-63f, &s, &c);
    cs[i] = c * rope.magnitude;
    sn[i] = s * rope.magnitude;
  }
  __syncthreads();
}

// grid (tokens, slices): the slice's share of the token's heads
template <uint32_t N>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs rope, RopeRows rows,
                                                        uint32_t head_dim,
                                                        const uint32_t* __restrict__ positions) {
  __shared__ float cs[128], sn[128];
  const uint32_t t = blockIdx.x;
  fill_turns(rope, positions[t], cs, sn);
  const uint32_t units = row_units(rope.rotary_dim, head_dim, rope.layout, N);
  const uint32_t h0 = (uint32_t)((uint64_t)rows.heads * blockIdx.y / gridDim.y);
  const uint32_t h1 = (uint32_t)((uint64_t)rows.heads * (blockIdx.y + 1u) / gridDim.y);
  for (uint32_t i = threadIdx.x; i < (h1 - h0) * units; i += kThreads) {
    const uint32_t h = h0 + i / units;
    do_unit<N>(i % units, Row<float>{rows.x + t * rows.token_stride + h * rows.head_stride,
                                     rows.y + t * rows.y_token_stride + h * rows.y_head_stride},
               rope.rotary_dim, rope.layout, cs, sn);
  }
}

// grid (rows, slices): the slice's share of the query, key and value heads of row
// first + blockIdx.x, of sequences * tokens
template <uint32_t N, typename T>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(
    CacheView cache, RopeArgs rope, uint32_t first, uint32_t tokens,
    const uint32_t* __restrict__ counts, const uint32_t* __restrict__ positions,
    const float* __restrict__ k, size_t k_stride, const float* __restrict__ v, size_t v_stride,
    RopeRows q, void* ws) {
  __shared__ float cs[128], sn[128];
  const uint32_t row = first + blockIdx.x, seq = row / tokens, t = row - seq * tokens;
  if (t >= brought(counts, seq, tokens)) return;
  const uint32_t slot = held(cache, seq) + t;
  uint32_t at = kNone;
  if (slot < cache.capacity) at = cache_row(cache, seq, 0u, slot);
  if (at == kNone && blockIdx.y == 0u && threadIdx.x == 0u)
    report_device_error(ws, slot < cache.capacity ? kDevErrCachePage : kDevErrCacheFull);
  const uint32_t n = rope.rotary_dim, dim = cache.head_dim;
  if (n) fill_turns(rope, positions ? positions[row] : slot, cs, sn);
  const uint32_t units = row_units(n, dim, rope.layout, N);
  const uint32_t heads = q.heads + 2u * cache.kv_heads;
  const uint32_t h0 = (uint32_t)((uint64_t)heads * blockIdx.y / gridDim.y);
  const uint32_t h1 = (uint32_t)((uint64_t)heads * (blockIdx.y + 1u) / gridDim.y);
  // value rows are all plain; their units are counted like the others' so that one division
  // serves, and the left-over ones of a row go beside them
  const uint32_t plain = dim / N;
  for (uint32_t i = threadIdx.x; i < (h1 - h0) * plain; i += kThreads) {
    const uint32_t h = h0 + i / plain, u = i % plain;
    if (h < q.heads) {
      if (u < units)
        do_unit<N>(u, Row<float>{q.x + row * q.token_stride + h * q.head_stride,
                                 q.y + ((size_t)row * q.heads + h) * dim},
                   n, rope.layout, cs, sn);
    } else if (at != kNone) {
      const uint32_t kh = h - q.heads;
      const bool value = kh >= cache.kv_heads;
      const uint32_t kv = value ? kh - cache.kv_heads : kh;
      const size_t to = ((size_t)at + (size_t)kv * cache.page_tokens) * dim;
      if (value)
        do_unit<N>(u, Row<T>{v + row * v_stride + (size_t)kv * dim, (T*)cache.values + to}, 0u, 0u,
                   cs, sn);
      else if (u < units)
        do_unit<N>(u, Row<T>{k + row * k_stride + (size_t)kv * dim, (T*)cache.keys + to}, n,
                   rope.layout, cs, sn);
    }
  }
}

__global__ void kv_advance_kernel(CacheView cache, const uint32_t* __restrict__ counts,
                                  uint32_t more) {
  const uint32_t s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s >= cache.sequences) return;
  const uint64_t n = (uint64_t)held(cache, s) + (counts ? counts[s] : 0u) + more;
  cache.lengths[s] = (uint32_t)(n < cache.capacity ? n : cache.capacity);
}

// Whether sixteen-byte units cover a row: its rotated part is whole units of
// them (half layout: each half), and so is the rest.
bool rope_vectors(uint32_t n, uint32_t dim, uint32_t layout) {
  return dim % 4u == 0u && n % (layout == 1u ? 4u : 8u) == 0u;
}

// Slices a token's heads are dealt to: enough workgroups for the card where
// the tokens are few, and no more than there are heads.
uint32_t slices_for(uint32_t tokens, uint32_t heads) {
  const uint32_t want = (1024u + tokens - 1u) / tokens;
  return std::max(1u, std::min(want, heads));
}

// A launch takes less than 2^32 threads in x, and runs fewer than it was asked
// for, without an error, from there on: more rows are several.
constexpr uint32_t kMostRows = 0xffffffffu / kThreads;

}  // namespace

hipError_t launch_rope(const RopeArgs& rope, const RopeRows& rows, uint32_t tokens,
                       uint32_t head_dim, const uint32_t* positions, hipStream_t s) {
  const bool vec = rope_vectors(rope.rotary_dim, head_dim, rope.layout);
  for (uint32_t t0 = 0; t0 < tokens; t0 += std::min(kMostRows, tokens - t0)) {
    const uint32_t n = std::min(kMostRows, tokens - t0);
    const dim3 grid(n, slices_for(n, rows.heads));
    RopeRows part = rows;
    part.x += t0 * rows.token_stride;
    part.y += t0 * rows.y_token_stride;
    if (vec)
      rope_kernel<4><<<grid, kThreads, 0, s>>>(rope, part, head_dim, positions + t0);
    else
      rope_kernel<1><<<grid, kThreads, 0, s>>>(rope, part, head_dim, positions + t0);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_rope_append(const CacheView& cache, const RopeArgs* rope, uint32_t tokens,
                              const uint32_t* counts, const uint32_t* positions, const float* k,
                              size_t k_stride, const float* v, size_t v_stride, const RopeRows* q,
                              void* ws, hipStream_t s) {
  const RopeArgs r = rope ? *rope : RopeArgs{0u, 0u, 1.0f, nullptr};
  const RopeRows qr = q ? *q : RopeRows{};
  const bool vec = rope_vectors(r.rotary_dim, cache.head_dim, r.layout) && aligned4(cache.keys) &&
                   aligned4(cache.values);
  const uint32_t rows = cache.sequences * tokens;
  auto go = [&](auto kernel) {
    for (uint32_t r0 = 0; r0 < rows; r0 += std::min(kMostRows, rows - r0)) {
      const uint32_t n = std::min(kMostRows, rows - r0);
      const dim3 grid(n, slices_for(n, qr.heads + 2u * cache.kv_heads));
      kernel<<<grid, kThreads, 0, s>>>(cache, r, r0, tokens, counts, positions, k, k_stride, v,
                                       v_stride, qr, ws);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  if (cache.type == kKvF32)
    return vec ? go(rope_append_kernel<4, float>) : go(rope_append_kernel<1, float>);
  if (cache.type == kKvF16)
    return vec ? go(rope_append_kernel<4, __half>) : go(rope_append_kernel<1, __half>);
  return vec ? go(rope_append_kernel<4, __hip_bfloat16>) : go(rope_append_kernel<1, __hip_bfloat16>);
}

hipError_t launch_kv_advance(const CacheView& cache, const uint32_t* counts, uint32_t more,
                             hipStream_t s) {
  kv_advance_kernel<<<(cache.sequences + 255u) / 256u, 256, 0, s>>>(cache, counts, more);
  return hipGetLastError();
}

}  // namespace sihip
