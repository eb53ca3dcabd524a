// C ABI of the paged key/value cache: cache_write, cache_read and paged_attn. Argument checks, choice of the
// kernel and launch on the caller's stream; no allocation, no synchronisation.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "paged_host.hpp"

namespace {

using pa::aligned16;
using pa::check_cache;
using pa::check_strides;
using pa::check_tokens;
using pa::fail;
using pa::hip_status;
using pa::with_types;

}  // namespace

extern "C" {

int pa_cache_write(const pa_paged_cache* cache, const void* k, const void* v, int dtype, int64_t tokens,
                   int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                   const int32_t* cu_seqlens, void* stream) {
  const char* name = "cache_write";
  pa::PagedCache c;
  if (int rc = check_cache(name, cache, dtype, &c)) return rc;
  if (!k || !v) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (int rc = check_tokens(name, tokens, cu_seqlens, &c)) return rc;
  if (!aligned16(k) || !aligned16(v)) return fail(PA_ERR_INVALID, "%s: inputs must be 16-byte aligned", name);
  if (int rc = check_strides(name, {k_token_stride, k_head_stride, v_token_stride, v_head_stride})) return rc;
  const int64_t rows_per_block = 256 / (cache->d / 8);
  const int64_t blocks = (tokens * 2 * cache->heads + rows_per_block - 1) / rows_per_block;
  if (blocks >= (1 << 24)) return fail(PA_ERR_UNSUPPORTED, "%s: too many rows for one launch", name);
  const hipError_t e = with_types(dtype, cache->dtype, cache->d, [&](auto t, auto ct, auto dim) {
    hipLaunchKernelGGL((pa::cache_write_rows<decltype(t), decltype(ct), decltype(dim)::value>), dim3((unsigned)blocks),
                       dim3(256), 0, static_cast<hipStream_t>(stream), c, pa::RowsIn{k, k_token_stride, k_head_stride},
                       pa::RowsIn{v, v_token_stride, v_head_stride});
    return hipGetLastError();
  });
  return hip_status(e, name);
}

int pa_cache_read(const pa_paged_cache* cache, void* k, void* v, int dtype, int64_t n, void* stream) {
  const char* name = "cache_read";
  pa::PagedCache c;
  if (int rc = check_cache(name, cache, dtype, &c)) return rc;
  if (!k || !v) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (n <= 0) return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (n > pa::kPagedMaxPos) return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^30 rows", name);
  if (!aligned16(k) || !aligned16(v)) return fail(PA_ERR_INVALID, "%s: inputs must be 16-byte aligned", name);
  const int64_t x = cache->seqs * cache->heads;
  if (x >= (1 << 24)) return fail(PA_ERR_UNSUPPORTED, "%s: too many rows for one launch", name);
  const int64_t rows_per_block = 256 / (cache->d / 8);
  const int64_t y = std::min<int64_t>((n + rows_per_block - 1) / rows_per_block, 65535);
  const hipError_t e = with_types(dtype, cache->dtype, cache->d, [&](auto t, auto ct, auto dim) {
    typedef decltype(t) T;
    const bool past_caches = x * n >= pa::kStreamBytes / (2 * cache->d * (int64_t)sizeof(T));
    const auto kernel = past_caches ? pa::cache_read_rows<T, decltype(ct), decltype(dim)::value, true>
                                  : pa::cache_read_rows<T, decltype(ct), decltype(dim)::value, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)x, (unsigned)y), dim3(256), 0, static_cast<hipStream_t>(stream), c,
                       static_cast<T*>(k), static_cast<T*>(v), (int)n);
    return hipGetLastError();
  });
  return hip_status(e, name);
}

int pa_paged_attn_fwd(const pa_paged_cache* cache, const void* q, void* o, int dtype, int64_t tokens, int64_t heads_q,
                      int64_t q_token_stride, int64_t q_head_stride, int64_t o_token_stride, int64_t o_head_stride,
                      const int32_t* cu_seqlens, int64_t max_new, int causal, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  pa::AttnWork w{};
  w.causal = causal;
  return pa::attn_call<false>("paged_attn", cache, {q, o, q_token_stride, q_head_stride, o_token_stride, o_head_stride, 0, (int)heads_q},
                              dtype, tokens, heads_q, cu_seqlens, max_new, w, workspace, workspace_bytes, stream);
}

int64_t pa_paged_attn_workspace(const pa_paged_cache* cache, int dtype, int64_t tokens, int64_t heads_q,
                                const int32_t* cu_seqlens, int64_t max_new) {
  return pa::attn_workspace_of("paged_attn", cache, dtype, tokens, heads_q, cu_seqlens, max_new, false);
}

}  // extern "C"
