// Attention over the paged cache with rules on the scores (eff_attn.h).
#include "eff_attn.h"

namespace eff {

size_t kv_attn_rules_scratch(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, const KvRulesView &r) {
  return attn_scratch(attn_plan(kv, b, a, r), kv);
}

hipError_t launch_kv_attn_rules(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, const KvRulesView &r, void *scratch,
                                hipStream_t stream) {
  return kv.type == EFF_KV_F16 ? attn_dim<EFF_KV_F16>(kv, b, a, r, scratch, stream) : attn_dim<EFF_KV_I8>(kv, b, a, r, scratch, stream);
}

}  // namespace eff
