// Attention over a paged cache of 16 or 32 bits (paged_attn.h).
#include "paged_attn.h"

extern "C" size_t nkl_paged_attention_workspace_bytes(const nkl_paged_cache* cache, int H, int window, int sinks,
                                                      int tree) {
  return nkl::paged_bytes<false>(cache, H, window, sinks, tree, cache ? cache->dtype : NKL_BF16);
}

extern "C" int nkl_paged_attention(const nkl_paged_cache* cache, const void* q, void* o, int H, long q_row, long q_head,
                                   long o_row, long o_head, int window, int sinks, const void* tree, int tree_words,
                                   float scale, void* workspace, size_t workspace_bytes, void* stream) {
  return nkl::paged_run<false>("nkl_paged_attention", cache, nullptr, cache ? cache->dtype : NKL_BF16, q, o, H, q_row, q_head,
                               o_row, o_head, window, sinks, tree, tree_words, scale, workspace, workspace_bytes, stream);
}
