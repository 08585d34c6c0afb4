// Attention over a paged BF16 cache (attention_mfma.h).
#include "attention_mfma.h"

namespace sihip {

hipError_t launch_attention_bf16(const AttentionArgs& a, const attn::Outputs& o, hipStream_t s) {
  return attn::launch_type<attn::Bf16>(a, o, s);
}

}  // namespace sihip
