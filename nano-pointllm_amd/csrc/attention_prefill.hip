// Causal attention of prompts and prompt chunks (attention_prefill.h).
#include "attention_prefill.h"

namespace w8a8 {

int64_t paged_prefill_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                int64_t head_dim, int64_t max_keys) {
  return workspace_of(tokens, batch, q_heads, kv_heads, head_dim, max_keys);
}

hipError_t launch_paged_prefill(const PagedAttention& a, bool clear, int dtype, hipStream_t st) {
  PrefillParams p{};
  return launch<Seen::kCausal>(p, a, a.max_keys, clear, dtype, st);
}

}  // namespace w8a8
