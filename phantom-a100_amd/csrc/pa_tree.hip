// C ABI of the attention of trees of drafted tokens over the paged cache: the kernels of paged_attn with a mask of the
// new tokens instead of their order.
#include <hip/hip_runtime.h>

#include "paged_host.hpp"

extern "C" {

int pa_paged_tree_attn_fwd(const pa_paged_cache* cache, const void* q, void* o, int dtype, int64_t tokens, int64_t heads_q,
                           int64_t q_token_stride, int64_t q_head_stride, int64_t o_token_stride, int64_t o_head_stride,
                           const int32_t* cu_seqlens, int64_t max_new, const int32_t* mask, int64_t mask_words,
                           int64_t mask_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "paged_tree_attn";
  if (!mask) return pa::fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (mask_words <= 0 || mask_words > pa::kPagedMaxPos / 32 || mask_stride < 0)
    return pa::fail(PA_ERR_INVALID, "%s: the mask must have 1 to 2^25 words a row and a stride that is not negative", name);
  pa::TreeWork w{};
  w.causal = 0;
  w.mask = reinterpret_cast<const uint32_t*>(mask);
  w.mask_stride = mask_stride;
  w.words = (int)mask_words;
  return pa::attn_call<true>(name, cache, {q, o, q_token_stride, q_head_stride, o_token_stride, o_head_stride, 0, (int)heads_q},
                             dtype, tokens, heads_q, cu_seqlens, max_new, w, workspace, workspace_bytes, stream);
}

int64_t pa_paged_tree_attn_workspace(const pa_paged_cache* cache, int dtype, int64_t tokens, int64_t heads_q,
                                     const int32_t* cu_seqlens, int64_t max_new) {
  return pa::attn_workspace_of("paged_tree_attn", cache, dtype, tokens, heads_q, cu_seqlens, max_new, true);
}

}  // extern "C"
