// Attention of trees of drafted tokens: a sequence's rows see all of its cached keys
// and, by a mask, each other's.  Few rows per sequence and key head run as
// attention_drafts.hip, the others as a prompt's (attention_prefill.h): 4 trees of 33 to 45
// tokens, 32 heads over 8, behind 24000 to 32768 take 147 us and a join of 9, 0.5 PFLOP/s
// of what is seen, in row tiles of 128 of which the second holds 4 to 52 rows: blocks of
// 32 rows on the four SIMDs two, two, one and one (132 rows: two, one, one, one).  No
// unit is the bound: the matrix units are busy 24% of the time, the vector units 30%,
// and wavefronts wait 41%.
#include "attention_prefill.h"

namespace w8a8 {

int64_t paged_tree_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                             int64_t head_dim, int64_t max_keys) {
  if (small_trees(tokens, batch, q_heads, kv_heads, head_dim))
    return small_trees_workspace(tokens, batch, q_heads, kv_heads, head_dim, max_keys);
  return workspace_of(tokens, batch, q_heads, kv_heads, head_dim, max_keys);
}

hipError_t launch_paged_tree(const PagedAttention& a, const uint64_t* masks, int64_t ld_masks,
                             int words, bool clear, int dtype, hipStream_t st) {
  if (small_trees(a.tokens, a.batch, a.q_heads, a.kv_heads, a.head_dim))
    return launch_small_trees(a, masks, ld_masks, words, clear, dtype, st);
  PrefillParams p{};
  p.masks = masks;
  p.ld_masks = ld_masks;
  p.words = words;
  return launch<Seen::kTree>(p, a, a.max_keys, clear, dtype, st);
}

}  // namespace w8a8
