// Attention of prompts and prompt chunks of which a row sees its last `window`
// keys and the sequence's first `sinks` (attention_prefill.h): the units of keys
// between the two are neither read nor computed, nor are their pages looked up.
//
// Bound as a prompt without a window: 16384 tokens of 32 heads over 8 with a window of
// 4096 take 0.99 to 1.05 ms (0.92 to 0.98 PFLOP/s of what is seen) once the clock has
// settled, up to 1.18 ms in the first dozen launches after idle time; 5 of the 131
// units of a row tile have masks.  A short prompt is one row tile's units in a row: 560
// tokens of 32 heads take 11.4 us with a window of one key, 12.4 with 32, 15.1 with 128,
// 17.9 with 256, and 19.3 with one of 559 (calls in a captured graph; back to back 0.2
// more, as a trace's durations 0.6 more); 10 of the 13 units of a window of 256 have
// masks, which cost about 0.25 us each on top of a unit's 0.55.
#include "attention_prefill.h"

namespace w8a8 {

int64_t paged_prefill_window_workspace(int64_t tokens, int64_t batch, int64_t q_heads,
                                       int64_t kv_heads, int64_t head_dim, int64_t max_keys,
                                       int64_t window, int64_t sinks) {
  return workspace_of(tokens, batch, q_heads, kv_heads, head_dim,
                      seen_keys(max_keys, q_heads / kv_heads, window, sinks));
}

hipError_t launch_paged_prefill_window(const PagedAttention& a, int window, int sinks, bool clear,
                                       int dtype, hipStream_t st) {
  PrefillParams p{};
  p.window = window;
  p.sinks = sinks;
  return launch<Seen::kWindow>(p, a, seen_keys(a.max_keys, a.q_heads / a.kv_heads, window, sinks),
                               clear, dtype, st);
}

}  // namespace w8a8
