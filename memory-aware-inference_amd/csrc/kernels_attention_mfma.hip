// Attention over a paged cache on the matrix cores: which calls take it, and
// the join of sequences that lie in several workgroups' shares.
#include "attention_common.h"

namespace sihip {

using namespace attn;

namespace {

constexpr uint32_t kThreads = 512;

// grid (kv_heads * rows, sequences): threads take four values of the row each,
// in groups that take every so-manieth share.
__global__ __launch_bounds__(kThreads) void attention_join(AttentionArgs a, Outputs o) {
  __shared__ float4 shared[kThreads];
  const CacheView& c = a.cache;
  const uint32_t rows = a.tokens * a.group, head = blockIdx.x, kv = head / rows;
  const uint32_t r = head - kv * rows;
  const uint32_t seq = blockIdx.y, tid = threadIdx.x, lane = tid & 63u;
  // the rounds before the sequence's, and its own
  uint32_t before = 0u, total = 0u;
  for (uint32_t i = lane; i < c.sequences; i += 64u) {
    const uint32_t n = span_of(a, i, o.round).rounds;
    total += n;
    if (i < seq) before += n;
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) {
    before += __shfl_xor(before, s, 64);
    total += __shfl_xor(total, s, 64);
  }
  const Deal deal = deal_of(total, c.sequences, o);
  const uint32_t first = before + deal.start * seq, share0 = first / deal.each;
  const uint32_t shares = (first + span_of(a, seq, o.round).rounds - 1u) / deal.each - share0 + 1u;
  if (shares == 1u) return;  // written already
  const auto at = [&](uint32_t p) { return (size_t)(share0 + p + seq) * c.kv_heads * rows + head; };
  // (the first of the thread's shares are under way while the maximum is found)
  const uint32_t dim = c.head_dim, width = dim / 4u, groups = kThreads / width;
  const uint32_t group = tid / width, d = (tid - group * width) * 4u;
  constexpr uint32_t kAhead = 8;
  float4 x[kAhead];
  float x_m[kAhead];
#pragma unroll
  for (uint32_t k = 0; k < kAhead; ++k) {
    const uint32_t p = group + k * groups;
    if (k * groups >= shares) break;
    x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    x_m[k] = -INFINITY;
    if (group < groups && p < shares) {
      x[k] = *reinterpret_cast<const float4*>(o.part_out + at(p) * dim + d);
      x_m[k] = o.part_stats[at(p)].x;
    }
  }
  float top = -INFINITY;
  for (uint32_t p = lane; p < shares; p += 64u) top = fmaxf(top, o.part_stats[at(p)].x);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  Joined sum_l;
  for (uint32_t p = lane; p < shares; p += 64u) sum_l.add(o.part_stats[at(p)], top);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) sum_l.l += __shfl_xor(sum_l.l, s, 64);
  sum_l.minus = __builtin_amdgcn_ballot_w64(sum_l.minus) != 0u;
  const float2 st = sum_l.result(top);
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (group < groups) {
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k)
      if (k * groups < shares) add_share(x_m[k], top, x[k], sum);
    for (uint32_t p = group + kAhead * groups; p < shares; p += groups) {
      add_share(o.part_stats[at(p)].x, top,
                *reinterpret_cast<const float4*>(o.part_out + at(p) * dim + d), sum);
    }
    shared[group * width + d / 4u] = sum;
  }
  __syncthreads();
  if (group != 0u) return;
  for (uint32_t g = 1; g < groups; ++g) {
    const float4 x = shared[g * width + d / 4u];
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  const uint32_t t = r / a.group, h = kv * a.group + (r - t * a.group);
  float* to = a.out + (((size_t)seq * a.tokens + t) * a.heads + h) * dim + d;
  const float4 v = finished(sum, st);
  *reinterpret_cast<Floats4*>(to) = Floats4{v.x, v.y, v.z, v.w};
  if (o.stats && tid == 0u)
    o.stats[(size_t)seq * c.kv_heads * rows + head] = row_stats(st, o.shift);
}

}  // namespace

hipError_t launch_attention_join(const AttentionArgs& a, const Outputs& o, hipStream_t s) {
  const dim3 grid(a.cache.kv_heads * a.tokens * a.group, a.cache.sequences);
  attention_join<<<grid, kThreads, 0, s>>>(a, o);
  return hipGetLastError();
}

hipError_t launch_attention_mfma(const AttentionArgs& a, const Space& sp, bool* taken,
                                 hipStream_t s) {
  const CacheView& c = a.cache;
  // rows of whole sixteen-byte pieces, whose words are words of memory.  (The general kernel
  // is for the others: 8 sequences of 4000 slots of 8 heads of 128 take it 1190 us, this one
  // 31.  Below some 15 slots it would be the faster one, 7.0 against 10.1 us for a single
  // slot, but the lengths are on the device.)
  const uint32_t row = c.head_dim * (c.type == kKvF32 ? 4u : 2u);
  *taken = row % 16u == 0u && aligned4(c.keys) && aligned4(c.values);
  // (the rounds of all sequences are counted in 31 bits)
  *taken = *taken && (uint64_t)c.sequences * (c.capacity / 32u + 3u) < 0x7fffffffu;
  if (!*taken) return hipSuccess;
  uint8_t* w = static_cast<uint8_t*>(a.workspace);
  Outputs o{};
  o.part_stats = reinterpret_cast<float2*>(w + sp.part_stats);
  o.part_out = reinterpret_cast<float*>(w + sp.part_out);
  o.stats = a.weights ? reinterpret_cast<float2*>(w + sp.stats) : nullptr;
  o.scores = a.weights ? reinterpret_cast<float*>(w + sp.scores) : nullptr;
  o.score_stride = sp.score_stride;
  o.counters = static_cast<uint32_t*>(a.report);
  o.by_group = divisor_of(a.group);
  o.by_heads = divisor_of(c.kv_heads);
  if (c.type == kKvF32) return launch_attention_f32(a, o, s);
  if (c.type == kKvF16) return launch_attention_f16(a, o, s);
  return launch_attention_bf16(a, o, s);
}

}  // namespace sihip
