// The short causal convolution of a recurrent layer's channels.
//
// y_t = act(b + sum_j w_j x_{t - W + 1 + j}), each channel by itself.  Memory is
// all there is to it: a thread has four channels and a run of tokens, and the
// W - 1 inputs before a token stay in its registers, so that but for a run's
// first ones each input is read once.  10240 channels of ragged prompts (471 MB, width 4) take 100.6 us,
// 4.7 TB/s, what a copy reaches; a single token of one sequence 4.2 us, a launch.  What a sequence's new state needs of the old one
// is read by the threads that write it, so the two may be one buffer.
#include "mixer_internal.h"

namespace sihip {
namespace {

constexpr uint32_t kThreads = 64;
constexpr uint32_t kStep = 8;  // tokens whose inputs are under way together

// y / (1 + e^-y).  The quotient by the card's reciprocal, good to a unit in the last place, and what it leaves of y taken
// into it: to half a unit, as a division's.  500 tokens of 10240 channels take 10.3 us (without it 9.75, by a division
// 11.3), 2000 29.4 (28.9, 29.3).
__device__ __forceinline__ float silu(float y) {
  const float d = 1.0f + expf(-y), r = __builtin_amdgcn_rcpf(d), q = y * r;
  const float z = __builtin_fmaf(__builtin_fmaf(-q, d, y), r, q);
  return d < __builtin_inff() ? z : q;
}

template <uint32_t N>
struct Channels {
  float v[N];
};
template <uint32_t N>
__device__ __forceinline__ Channels<N> load(const float* p) {
  Channels<N> c;
  if constexpr (N == 4) {
    const Floats4 f = *reinterpret_cast<const Floats4*>(p);
    c.v[0] = f.x, c.v[1] = f.y, c.v[2] = f.z, c.v[3] = f.w;
  } else {
    c.v[0] = *p;
  }
  return c;
}
template <uint32_t N>
__device__ __forceinline__ void store(float* p, const Channels<N>& c) {
  if constexpr (N == 4)
    *reinterpret_cast<Floats4*>(p) = Floats4{c.v[0], c.v[1], c.v[2], c.v[3]};
  else
    *p = c.v[0];
}

// Tokens [t0, t1) of a sequence that has `count`, channels c .. c + N - 1, the loads of STEP tokens
// under way together; x, y and the states at the sequence's first.
template <uint32_t W, uint32_t N, uint32_t STEP>
__device__ __forceinline__ void run(const ConvArgs& a, const float* x, float* y,
                                    const float* state, float* state_out, uint32_t c, uint32_t t0,
                                    uint32_t t1, uint32_t count) {
  constexpr uint32_t H = W - 1;
  Channels<N> w[W], bias, row[H + STEP];
  bias = a.bias ? load<N>(a.bias + c) : Channels<N>{};
  // (the channels' weights are one run of N W floats)
#pragma unroll
  for (uint32_t m = 0; m < W; ++m) {
    const Channels<N> part = load<N>(a.weight + (size_t)c * W + m * N);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) w[(m * N + i) % W].v[(m * N + i) / W] = part.v[i];
  }
  // row j is input t0 - H + j
#pragma unroll
  for (uint32_t j = 0; j < H; ++j) {
    row[j] = Channels<N>{};
    if (t0 + j >= H)
      row[j] = load<N>(x + (size_t)(t0 + j - H) * a.x_stride + c);
    else if (state)
      row[j] = load<N>(state + (size_t)(t0 + j) * a.channels + c);
  }
  if (t0 == 0u && state_out) {
    // the last H of (state, inputs): inputs from count - H on, or what is left of the state
    Channels<N> last[H];
#pragma unroll
    for (uint32_t j = 0; j < H; ++j) {
      last[j] = Channels<N>{};
      if (count + j >= H) {
        last[j] = load<N>(x + (size_t)(count + j - H) * a.x_stride + c);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < H; ++i)
          if (i == count + j) last[j] = row[i];
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < H; ++j) store<N>(state_out + (size_t)j * a.channels + c, last[j]);
  }
  if (!y) return;
  for (uint32_t t = t0; t < t1; t += STEP) {
#pragma unroll
    for (uint32_t s = 0; s < STEP; ++s)
      if (t + s < t1) row[H + s] = load<N>(x + (size_t)(t + s) * a.x_stride + c);
#pragma unroll
    for (uint32_t s = 0; s < STEP; ++s) {
      if (t + s >= t1) break;
      Channels<N> o = bias;
#pragma unroll
      for (uint32_t j = 0; j < W; ++j)
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) o.v[i] = __builtin_fmaf(w[j].v[i], row[s + j].v[i], o.v[i]);
      if (a.silu)
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) o.v[i] = silu(o.v[i]);
      store<N>(y + (size_t)(t + s) * a.y_stride + c, o);
    }
#pragma unroll
    for (uint32_t j = 0; j < H; ++j) row[j] = row[STEP + j];
  }
}

// grid (blocks of channels, runs of tokens, sequences)
template <uint32_t W>
__global__ __launch_bounds__(kThreads) void conv_kernel(ConvArgs a, uint32_t each) {
  const uint32_t seq = blockIdx.z, count = tokens_of(a.count, seq);
  const uint32_t t0 = blockIdx.y * each;
  if (t0 >= count && t0 != 0u) return;
  const uint32_t t1 = min(count, t0 + each);
  const uint32_t c = 4u * (blockIdx.x * kThreads + threadIdx.x);
  if (c >= a.channels) return;
  const size_t rows = (size_t)seq * a.count.tokens, held = (size_t)seq * (W - 1u) * a.channels;
  const float* x = a.x + rows * a.x_stride;
  float* y = a.y ? a.y + rows * a.y_stride : nullptr;
  const float* state = a.state ? a.state + held : nullptr;
  float* state_out = a.state_out ? a.state_out + held : nullptr;
  if (c + 4u <= a.channels) {
    run<W, 4, kStep>(a, x, y, state, state_out, c, t0, t1, count);
  } else {
    for (uint32_t i = c; i < a.channels; ++i) run<W, 1, 1>(a, x, y, state, state_out, i, t0, t1, count);
  }
}

}  // namespace

hipError_t launch_conv(const ConvArgs& a, hipStream_t s) {
  const uint32_t blocks = (a.channels + 4u * kThreads - 1u) / (4u * kThreads);
  // Runs of tokens: long ones read their first inputs again the least; no longer than what leaves
  // four waves a SIMD, and within a launch's 65535 runs.
  const uint32_t tokens = a.count.tokens;
  uint32_t each = a.y ? 64u : tokens;
  if (a.y) {
    while (each > 8u && (uint64_t)blocks * a.sequences * (tokens / each) < 4096u) each /= 2u;
    while ((tokens + each - 1u) / each > 65535u) each *= 2u;
  }
  const dim3 grid(blocks, a.y ? (tokens + each - 1u) / each : 1u, a.sequences);
  auto go = [&](auto width) {
    conv_kernel<decltype(width)::value><<<grid, kThreads, 0, s>>>(a, each);
    return hipGetLastError();
  };
  using std::integral_constant;
  switch (a.width) {
    case 2: return go(integral_constant<uint32_t, 2>{});
    case 3: return go(integral_constant<uint32_t, 3>{});
    case 4: return go(integral_constant<uint32_t, 4>{});
    case 5: return go(integral_constant<uint32_t, 5>{});
    case 6: return go(integral_constant<uint32_t, 6>{});
    case 7: return go(integral_constant<uint32_t, 7>{});
    default: return go(integral_constant<uint32_t, 8>{});
  }
}

}  // namespace sihip
