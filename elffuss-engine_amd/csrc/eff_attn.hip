// Attention over the paged cache without rules on the scores (eff_attn.h).
#include "eff_attn.h"

namespace eff {

size_t kv_attn_scratch(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a) {
  return attn_scratch(attn_plan(kv, b, a), kv);
}

hipError_t launch_kv_attn(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, void *scratch, hipStream_t stream) {
  return kv.type == EFF_KV_F16 ? attn_dim<EFF_KV_F16>(kv, b, a, NoRules{}, scratch, stream) : attn_dim<EFF_KV_I8>(kv, b, a, NoRules{}, scratch, stream);
}

}  // namespace eff
