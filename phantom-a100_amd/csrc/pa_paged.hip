// C ABI of the paged key/value cache: cache_write, cache_read and paged_attn. Argument checks, choice of the
// kernel and launch on the caller's stream; no allocation, no synchronisation.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "phantom_attn.h"
#include "host_common.hpp"
#include "kernels/paged_attn.hpp"

namespace {

using pa::fail;
using pa::hip_status;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool is_16bit(int dtype) { return dtype == PA_DTYPE_F16 || dtype == PA_DTYPE_BF16; }
bool is_8bit(int dtype) { return dtype == PA_DTYPE_I8 || dtype == PA_DTYPE_E4M3; }

// Checks what every call needs of a cache and fills the kernels' view of it (but for the new tokens).
int check_cache(const char* name, const pa_paged_cache* c, int dtype, pa::PagedCache* out) {
  if (!c) return fail(PA_ERR_INVALID, "%s: null cache", name);
  if (!c->k || !c->v || !c->page_table || !c->lengths) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (!is_16bit(dtype)) return fail(PA_ERR_UNSUPPORTED, "%s: float16 or bfloat16 only", name);
  if (c->dtype != dtype && !is_8bit(c->dtype))
    return fail(PA_ERR_UNSUPPORTED, "%s: the cache must hold the tensors' dtype, int8 or float8_e4m3", name);
  if (is_8bit(c->dtype) && (!c->k_scale || !c->v_scale))
    return fail(PA_ERR_INVALID, "%s: an 8-bit cache needs k_scale and v_scale", name);
  if (c->d != 64 && c->d != 128)
    return fail(PA_ERR_UNSUPPORTED, "%s: only head dimensions 64 and 128 are compiled (got %lld)", name, (long long)c->d);
  if (c->pages <= 0 || c->page_size <= 0 || c->heads <= 0 || c->seqs <= 0 || c->table_cols <= 0)
    return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (c->page_size > pa::kPagedMaxPos || c->table_cols > pa::kPagedMaxPos / c->page_size)
    return fail(PA_ERR_UNSUPPORTED, "%s: the page table spans more than 2^30 positions", name);
  if (c->heads > INT_MAX / c->page_size || c->pages > INT_MAX / (c->heads * c->page_size))
    return fail(PA_ERR_UNSUPPORTED, "%s: the cache has more than 2^31-1 rows", name);
  if (c->seqs > (1 << 24) || c->table_stride < 0)
    return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^24 sequences, or a negative page table stride", name);
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(PA_ERR_INVALID, "%s: inputs must be 16-byte aligned", name);
  *out = pa::PagedCache{c->k, c->v, c->k_scale, c->v_scale, c->page_table, c->lengths, nullptr,
                        (int)c->pages, (int)c->page_size, (int)c->heads, (int)c->seqs, (int)c->table_cols, 0, 0,
                        (int)(c->table_cols * c->page_size), c->table_stride, pa::make_page_div((uint32_t)c->page_size)};
  return PA_OK;
}

int check_tokens(const char* name, int64_t tokens, const int32_t* cu_seqlens, pa::PagedCache* c) {
  if (tokens <= 0) return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (tokens > pa::kPagedMaxPos) return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^30 new tokens", name);
  if (!cu_seqlens && tokens % c->seqs != 0)
    return fail(PA_ERR_INVALID, "%s: without cu_seqlens the tokens must divide evenly over the sequences", name);
  c->cu = cu_seqlens;
  c->tokens = (int)tokens;
  c->per_seq = cu_seqlens ? 0 : (int)(tokens / c->seqs);
  return PA_OK;
}

int check_strides(const char* name, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s < 0 || s % 8 != 0) return fail(PA_ERR_INVALID, "%s: strides must be whole 16-byte steps", name);
  return PA_OK;
}

// Calls f(T{}, C{}, integral_constant<int, D>{}) for the tensors' type, the cache's and the head dim.
template <typename T, typename F>
hipError_t with_cache_type(int cache_dtype, int64_t d, F f) {
  auto with_dim = [&](auto cache) {
    return d == 64 ? f(T{}, cache, std::integral_constant<int, 64>{}) : f(T{}, cache, std::integral_constant<int, 128>{});
  };
  if (cache_dtype == PA_DTYPE_I8) return with_dim(pa::i8{});
  if (cache_dtype == PA_DTYPE_E4M3) return with_dim(pa::e4m3{});
  return with_dim(T{});
}
template <typename F>
hipError_t with_types(int dtype, int cache_dtype, int64_t d, F f) {
  return dtype == PA_DTYPE_F16 ? with_cache_type<pa::f16>(cache_dtype, d, f) : with_cache_type<pa::bf16>(cache_dtype, d, f);
}

constexpr int kCUs = 256;   // MI355X / gfx950. (A constant: a workspace's size is asked for without a GPU.)

// The launch of an attention call: rows of a tile, workgroups, and whether tiles are cut.
struct AttnPlan {
  int rows, wgs;
  bool whole;
};
// A cache of at most so many positions a sequence is read in a few steps: its tiles are not cut over workgroups,
// which saves the second launch that joins them. One to 32 tokens over 200 keys: a call takes 17 to 18 us, cut 22;
// 2 x 100 tokens over 900 take 27 us cut and 47 whole.
constexpr int kWholeCapacity = 256;
AttnPlan attn_plan(const pa::PagedCache& c, int64_t d, bool k8, int64_t heads_q, int64_t max_new) {
  const int64_t group = heads_q / c.heads;
  const int64_t new_tokens = !c.cu ? c.per_seq : max_new > 0 ? std::min<int64_t>(max_new, c.tokens) : c.tokens;
  const int64_t most = new_tokens * group;   // rows of a sequence and key/value head
  // Few rows in tiles of 16 or 32, up to two of them over the same keys, more in chunks. 64 x 16 tokens of 4 heads
  // over 8192 keys as two tiles of 32 and as a chunk: 16 bits 325 and 322 us, 8 bits 228 and 378 (64 dims, 16 bits:
  // 156 and 137); 128 x 16 of 64 dims over 1000 in 8 bits 46 and 55. 17 to 32 rows as two
  // tiles of 16: 272 for 226. Tiles of 64 were between the two (315, 314), and slower at 128 rows than chunks (434, 308).
  const int rows = most <= 16 ? 16 : most <= 64 ? 32 : pa::chunk_rows_of((int)d);
  // As many workgroups as are resident at once, or fewer where the work's bound is below their least share.
  const pa::TileShape t = pa::make_tiles((int)group, rows);
  const double tiles = (double)c.tokens / t.tokens + c.seqs;
  const double units = tiles * c.heads * t.splits * ((double)pa::kTileCost + c.capacity);
  const int resident = kCUs * (rows > 64 ? pa::chunk_wgs((int)d, k8) : pa::few_wgs((int)d, k8, rows / 16));
  const int wgs = (int)std::max(1.0, std::min<double>(resident, units / pa::kMinUnits + 1));
  return {rows, wgs, c.capacity <= kWholeCapacity};
}
// The kernels count a call's work in 63 bits: each sequence could have all tokens (offsets out of order), each token
// the longest keys.
int check_work(const char* name, const pa::PagedCache& c, const AttnPlan& plan, int64_t heads_q) {
  const pa::TileShape t = pa::make_tiles((int)(heads_q / c.heads), plan.rows);
  const double tiles = ((double)c.tokens / t.tokens + 1) * c.seqs * c.heads * t.splits;
  if (tiles * (pa::kTileCost + (double)c.capacity + 2.0 * c.tokens) < 0x1p62) return PA_OK;
  return fail(PA_ERR_UNSUPPORTED, "%s: the sequences, tokens and positions make more than 2^62 steps of work", name);
}

template <typename T, int D, int ROWS, typename Kernel>
hipError_t launch_attn(Kernel kernel, int threads, const pa::PagedCache& c, const pa::RowsQ& a, const AttnPlan& plan,
                       int causal, void* workspace, hipStream_t stream) {
  const pa::AttnWork w{pa::make_tiles(a.group, ROWS), pa::kMinUnits, plan.whole, causal, pa::kLog2e / sqrtf((float)D),
                       static_cast<pa::PartRecord*>(workspace),
                       reinterpret_cast<float*>(static_cast<char*>(workspace) + pa::attn_record_bytes(plan.wgs))};
  hipLaunchKernelGGL(kernel, dim3((unsigned)plan.wgs), dim3(threads), 0, stream, c, a, w);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || plan.whole) return e;
  hipLaunchKernelGGL((pa::paged_attn_join<T, D, ROWS>), dim3((unsigned)plan.wgs, ROWS / 16), dim3(256), 0,
                     stream, c, a, w, plan.wgs);
  return hipGetLastError();
}

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
  const char* name = "paged_attn";
  pa::PagedCache c;
  if (int rc = check_cache(name, cache, dtype, &c)) return rc;
  if (!q || !o) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (int rc = check_tokens(name, tokens, cu_seqlens, &c)) return rc;
  if (heads_q <= 0 || heads_q > (1 << 16) || heads_q % cache->heads != 0)
    return fail(PA_ERR_INVALID, "%s: the query heads must be a multiple of the cache's heads", name);
  if (!aligned16(q) || !aligned16(o)) return fail(PA_ERR_INVALID, "%s: inputs must be 16-byte aligned", name);
  if (int rc = check_strides(name, {q_token_stride, q_head_stride, o_token_stride, o_head_stride})) return rc;
  const auto apart = [&](int64_t outer, int64_t outer_n, int64_t inner, int64_t inner_n) {
    return (inner_n == 1 || inner >= cache->d) && (outer_n == 1 || outer >= (inner_n - 1) * inner + cache->d);
  };
  if (!apart(o_token_stride, tokens, o_head_stride, heads_q) && !apart(o_head_stride, heads_q, o_token_stride, tokens))
    return fail(PA_ERR_INVALID, "%s: out's rows must not overlap", name);
  if (max_new < 0) return fail(PA_ERR_INVALID, "%s: max_new must not be negative", name);
  const AttnPlan plan = attn_plan(c, cache->d, is_8bit(cache->dtype), heads_q, max_new);
  if (int rc = check_work(name, c, plan, heads_q)) return rc;
  if (workspace_bytes < pa::attn_workspace(plan.wgs, plan.rows, (int)cache->d) || !workspace || !aligned16(workspace))
    return fail(PA_ERR_INVALID, "%s: the workspace is too small, null or not 16-byte aligned", name);
  const pa::RowsQ a{q, o, q_token_stride, q_head_stride, o_token_stride, o_head_stride, (int)(heads_q / cache->heads),
                    (int)heads_q};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = with_types(dtype, cache->dtype, cache->d, [&](auto t, auto ct, auto dim) {
    typedef decltype(t) T;
    typedef decltype(ct) C;
    constexpr int D = decltype(dim)::value;
    constexpr int CR = pa::chunk_rows_of(D);
    switch (plan.rows) {
      case 16: return launch_attn<T, D, 16>(pa::paged_attn_few<T, C, D, 1>, 256, c, a, plan, causal, workspace, st);
      case 32: return launch_attn<T, D, 32>(pa::paged_attn_few<T, C, D, 2>, 256, c, a, plan, causal, workspace, st);
      default: break;
    }
    const uint64_t cache_rows = (uint64_t)c.pages * c.heads * c.page_size;
    if (cache_rows * std::max<size_t>(D * sizeof(C), 4) > pa::kPastBuffer)
      return launch_attn<T, D, CR>(pa::paged_attn_chunk<T, C, D, CR, true>, 2 * CR, c, a, plan, causal, workspace, st);
    return launch_attn<T, D, CR>(pa::paged_attn_chunk<T, C, D, CR, false>, 2 * CR, c, a, plan, causal, workspace, st);
  });
  return hip_status(e, name);
}

int64_t pa_paged_attn_workspace(const pa_paged_cache* cache, int dtype, int64_t tokens, int64_t heads_q,
                                const int32_t* cu_seqlens, int64_t max_new) {
  const char* name = "paged_attn";
  pa::PagedCache c;
  if (int rc = check_cache(name, cache, dtype, &c)) return rc;
  if (int rc = check_tokens(name, tokens, cu_seqlens, &c)) return rc;
  if (heads_q <= 0 || heads_q > (1 << 16) || heads_q % cache->heads != 0 || max_new < 0)
    return fail(PA_ERR_INVALID, "%s: the query heads must be a multiple of the cache's heads, max_new not negative", name);
  const AttnPlan plan = attn_plan(c, cache->d, is_8bit(cache->dtype), heads_q, max_new);
  if (int rc = check_work(name, c, plan, heads_q)) return rc;
  return pa::attn_workspace(plan.wgs, plan.rows, (int)cache->d);
}

}  // extern "C"
