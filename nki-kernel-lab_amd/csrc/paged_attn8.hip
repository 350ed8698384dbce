// Attention over a paged cache of 8 bits (paged_attn.h).
#include "paged_attn.h"

extern "C" size_t nkl_paged_attention8_workspace_bytes(const nkl_paged_cache* cache, int H, int window, int sinks, int tree,
                                                       int dtype) {
  return nkl::paged_bytes<true>(cache, H, window, sinks, tree, dtype);
}

extern "C" int nkl_paged_attention8(const nkl_paged_cache* cache, const nkl_cache_scales* scales, int dtype, const void* q,
                                    void* o, int H, long q_row, long q_head, long o_row, long o_head, int window, int sinks,
                                    const void* tree, int tree_words, float scale, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  return nkl::paged_run<true>("nkl_paged_attention8", cache, scales, dtype, q, o, H, q_row, q_head, o_row, o_head, window,
                              sinks, tree, tree_words, scale, workspace, workspace_bytes, stream);
}
