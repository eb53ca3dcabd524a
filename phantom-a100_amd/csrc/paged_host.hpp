// What the C entries over the paged cache share: checks of a cache and of the new tokens, the choice of an attention
// call's launch, and the launch itself.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>

#include "phantom_attn.h"
#include "host_common.hpp"
#include "kernels/paged_attn.hpp"

namespace pa {

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
inline bool is_16bit(int dtype) { return dtype == PA_DTYPE_F16 || dtype == PA_DTYPE_BF16; }
inline bool is_8bit(int dtype) { return dtype == PA_DTYPE_I8 || dtype == PA_DTYPE_E4M3; }

// Checks what every call needs of a cache and fills the kernels' view of it (but for the new tokens).
inline int check_cache(const char* name, const pa_paged_cache* c, int dtype, PagedCache* out) {
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
  if (c->page_size > kPagedMaxPos || c->table_cols > kPagedMaxPos / c->page_size)
    return fail(PA_ERR_UNSUPPORTED, "%s: the page table spans more than 2^30 positions", name);
  if (c->heads > INT_MAX / c->page_size || c->pages > INT_MAX / (c->heads * c->page_size))
    return fail(PA_ERR_UNSUPPORTED, "%s: the cache has more than 2^31-1 rows", name);
  if (c->seqs > (1 << 24) || c->table_stride < 0)
    return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^24 sequences, or a negative page table stride", name);
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(PA_ERR_INVALID, "%s: inputs must be 16-byte aligned", name);
  *out = PagedCache{c->k, c->v, c->k_scale, c->v_scale, c->page_table, c->lengths, nullptr,
                        (int)c->pages, (int)c->page_size, (int)c->heads, (int)c->seqs, (int)c->table_cols, 0, 0,
                        (int)(c->table_cols * c->page_size), c->table_stride, make_page_div((uint32_t)c->page_size)};
  return PA_OK;
}

inline int check_tokens(const char* name, int64_t tokens, const int32_t* cu_seqlens, PagedCache* c) {
  if (tokens <= 0) return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (tokens > kPagedMaxPos) return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^30 new tokens", name);
  if (!cu_seqlens && tokens % c->seqs != 0)
    return fail(PA_ERR_INVALID, "%s: without cu_seqlens the tokens must divide evenly over the sequences", name);
  c->cu = cu_seqlens;
  c->tokens = (int)tokens;
  c->per_seq = cu_seqlens ? 0 : (int)(tokens / c->seqs);
  return PA_OK;
}

inline int check_strides(const char* name, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s < 0 || s % 8 != 0) return fail(PA_ERR_INVALID, "%s: strides must be whole 16-byte steps", name);
  return PA_OK;
}

// Whether two ranges of bytes share memory (a null one does not).
inline bool share_memory(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && (x < y ? y - x < (uint64_t)a_bytes : x - y < (uint64_t)b_bytes);
}
struct Bytes {
  const void* p;
  int64_t n;
};
// Whether one of `written` shares memory with one of `read`, or with another of `written`.
inline bool any_shared(std::initializer_list<Bytes> written, std::initializer_list<Bytes> read) {
  for (const Bytes& w : written) {
    for (const Bytes& r : read)
      if (share_memory(w.p, w.n, r.p, r.n)) return true;
    for (const Bytes& o : written)
      if (&o != &w && share_memory(w.p, w.n, o.p, o.n)) return true;
  }
  return false;
}
// Bytes from the first to the last of `rows` rows of `cols` elements, `stride` apart (not negative).
inline int64_t span_bytes(int64_t rows, int64_t stride, int64_t cols, int64_t size) {
  const int64_t far = rows > 1 && stride > (INT64_MAX >> 8) / rows ? INT64_MAX >> 8 : (rows - 1) * stride;
  return (far + cols) * size;
}

// Calls f(T{}, C{}, integral_constant<int, D>{}) for the tensors' type, the cache's and the head dim.
template <typename T, typename F>
hipError_t with_cache_type(int cache_dtype, int64_t d, F f) {
  auto with_dim = [&](auto cache) {
    return d == 64 ? f(T{}, cache, std::integral_constant<int, 64>{}) : f(T{}, cache, std::integral_constant<int, 128>{});
  };
  if (cache_dtype == PA_DTYPE_I8) return with_dim(i8{});
  if (cache_dtype == PA_DTYPE_E4M3) return with_dim(e4m3{});
  return with_dim(T{});
}
template <typename F>
hipError_t with_types(int dtype, int cache_dtype, int64_t d, F f) {
  return dtype == PA_DTYPE_F16 ? with_cache_type<f16>(cache_dtype, d, f) : with_cache_type<bf16>(cache_dtype, d, f);
}

constexpr int kCUs = 256;   // MI355X / gfx950. (A constant: a workspace's size is asked for without a GPU.)

// Whether a cache, or its scales, reach past the 32-bit offsets of a buffer.
inline bool past_buffer(const PagedCache& c, int64_t d, bool k8) {
  return (uint64_t)c.pages * c.heads * c.page_size * std::max<uint64_t>(d * (k8 ? 1 : 2), 4) > kPastBuffer;
}

// Rows of a tile for trees of more than 32 rows a key/value head: the tile whose time is the least by a start and a rate,
// a us and f times the time that reading the keys and values once takes, for each tile that goes over them. (The table's
// capacity stands for the lengths, which the host does not know.) Measured, us:
//                                                                 32     128     256 rows
//   D = 128, 32 heads over 8, bf16   32 x 12 over 8192 (1 GB)    371     205     205
//                                    32 x 28                     730     214     215
//                                    32 x 48                    1089     406     272
//                                    24 x 48 over 4096           373     181     130
//                                    16 x 48 over 1000 (66 MB)    82      38      59
//                                    16 x 12                      33      34      45
//                                     4 x 48 over 500             22      35      30
//                            e4m3    32 x 12 over 8192           284     209     231
//                                    32 x 48                     825     388     316
//                                    16 x 48 over 4000           207     120     105
//                                    16 x 16 over 1000            44      43      59
//                                     4 x 24                      34      37      53
//                 fp16 over e4m3     32 x 12 over 8192           293     238     272
//                                    16 x 16 over 1000            46      53      65
//   D = 64, 16 heads over 4, f16     24 x 16 over 4096            48      44
//                                    16 x 32 over 1000            28      31
//                            int8    24 x 24 over 4096            67      57
//                                    16 x 24 over 1000            28      34
// (Tiles of 64 rows were nowhere more than 2 % faster than the better of these.)
struct TileTime {
  int rows;
  double a, f;
};
inline int tree_rows(const PagedCache& c, int64_t d, bool k8, int64_t most) {
  static const TileTime kTimes[4][3] = {{{32, 14, 0.9}, {128, 25, 1.02}, {256, 34, 1.45}},   // D = 128
                                        {{32, 17, 2.1}, {128, 31, 1.9}, {256, 50, 2.8}},     // in 8 bits
                                        {{32, 12, 1.0}, {128, 27, 0.75}, {0, 0, 0}},         // D = 64
                                        {{32, 18, 1.3}, {128, 26, 2.6}, {0, 0, 0}}};
  const double once = 2.0 * c.seqs * c.heads * (double)c.capacity * d * (k8 ? 1 : 2) / 5e6;   // us at 5 TB/s
  int rows = 0;
  double least = 0;
  for (const TileTime& t : kTimes[(d == 64 ? 2 : 0) + (k8 ? 1 : 0)]) {
    if (t.rows == 0) break;
    const double us = t.a + t.f * once * (double)((most + t.rows - 1) / t.rows);
    if (rows == 0 || us < least) rows = t.rows, least = us;
  }
  return rows;
}
// Trees of few rows are not cut up to here: one of 4 tokens over 500 keys 15.2 us, cut 17.5, over 1000 19 and 18; of 16
// tokens 16.8 and 17.5, 24 and 18.
constexpr int kTreeWholeCapacity = 512;
// Least units of a workgroup with larger tiles, whose parts cost as much to write and join as that many keys: 4 x 64
// tokens over 4000, 256 rows, at least 128 units 65 us, 1024 55; 24 x 24 over 2048, 64 dims, 128 rows, 37 and (512) 34. It
// limits how tiles are cut, not how many workgroups take whole ones: tiles of fewer units have one each (share_count). Under a
// table of 8192 positions, 32 heads over 8, bf16, 32 x 48 tokens over 200 take 28 us so and 58 with the limit alone, over 50
// to 350 45 and 59, over 500 34 and 57; fp16 over e4m3 37, 61, 47 and 78, 80, 76.
inline int tree_units(int rows) { return 4 * rows; }

// The launch of an attention call: rows of a tile, workgroups, and whether tiles are cut.
struct AttnPlan {
  int rows, wgs, min_units;
  bool whole;
};
// A cache of at most so many positions a sequence is read in a few steps: its tiles are not cut over workgroups,
// which saves the second launch that joins them. One to 32 tokens over 200 keys: a call takes 17 to 18 us, cut 22;
// 2 x 100 tokens over 900 take 27 us cut and 47 whole.
constexpr int kWholeCapacity = 256;
inline AttnPlan attn_plan(const PagedCache& c, int64_t d, bool k8, int64_t heads_q, int64_t max_new, bool tree) {
  const int64_t group = heads_q / c.heads;
  const int64_t new_tokens = !c.cu ? c.per_seq : max_new > 0 ? std::min<int64_t>(max_new, c.tokens) : c.tokens;
  const int64_t most = new_tokens * group;   // rows of a sequence and key/value head
  // Few rows in tiles of 16 or 32, up to two of them over the same keys, more in chunks. 64 x 16 tokens of 4 heads
  // over 8192 keys as two tiles of 32 and as a chunk: 16 bits 325 and 322 us, 8 bits 228 and 378 (64 dims, 16 bits:
  // 156 and 137); 128 x 16 of 64 dims over 1000 in 8 bits 46 and 55. 17 to 32 rows as two
  // tiles of 16: 272 for 226. Tiles of 64 were between the two (315, 314), and slower at 128 rows than chunks (434, 308).
  const int rows = tree && most > 32 && !past_buffer(c, d, k8) ? tree_rows(c, d, k8, most)
                   : most <= 16 ? 16 : most <= 64 ? 32 : chunk_rows_of((int)d);
  // As many workgroups as are resident at once, or fewer where the work's bound is below their least share.
  const TileShape t = make_tiles((int)group, rows);
  const double tiles = (double)c.tokens / t.tokens + c.seqs;
  const double units = tiles * c.heads * t.splits * ((double)kTileCost + c.capacity);
  const int resident = kCUs * (rows > 32 ? chunk_wgs((int)d, k8, rows, tree) : few_wgs((int)d, k8, rows / 16));
  const int least = tree && rows > 32 ? tree_units(rows) : kMinUnits;
  const double shares = std::max(units / least, least > kMinUnits ? tiles * c.heads * t.splits : 0);
  const int wgs = (int)std::max(1.0, std::min<double>(resident, shares + 1));
  return {rows, wgs, least, c.capacity <= (tree && rows <= 32 ? kTreeWholeCapacity : kWholeCapacity)};
}
// The kernels count a call's work in 63 bits: each sequence could have all tokens (offsets out of order), each token
// the longest keys.
inline int check_work(const char* name, const PagedCache& c, const AttnPlan& plan, int64_t heads_q) {
  const TileShape t = make_tiles((int)(heads_q / c.heads), plan.rows);
  const double tiles = ((double)c.tokens / t.tokens + 1) * c.seqs * c.heads * t.splits;
  if (tiles * (kTileCost + (double)c.capacity + 2.0 * c.tokens) < 0x1p62) return PA_OK;
  return fail(PA_ERR_UNSUPPORTED, "%s: the sequences, tokens and positions make more than 2^62 steps of work", name);
}

// w comes with what is the kernel's own (causal, a tree's mask).
template <typename T, int D, int ROWS, typename Kernel, typename Work>
hipError_t launch_attn(Kernel kernel, int threads, const PagedCache& c, const RowsQ& a, const AttnPlan& plan, Work w,
                       void* workspace, hipStream_t stream) {
  w.tiles = make_tiles(a.group, ROWS);
  w.min_units = plan.min_units;
  w.whole = plan.whole;
  w.scale_log2 = kLog2e / sqrtf((float)D);
  w.records = static_cast<PartRecord*>(workspace);
  w.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + attn_record_bytes(plan.wgs));
  hipLaunchKernelGGL(kernel, dim3((unsigned)plan.wgs), dim3(threads), 0, stream, c, a, w);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || plan.whole) return e;
  hipLaunchKernelGGL((paged_attn_join<T, D, ROWS>), dim3((unsigned)plan.wgs, ROWS / 16), dim3(256), 0,
                     stream, c, a, (AttnWork)w, plan.wgs);
  return hipGetLastError();
}

// An attention call: its checks, its plan and its launch. a: q, o and their strides.
template <bool TREE>
int attn_call(const char* name, const pa_paged_cache* cache, RowsQ a, int dtype, int64_t tokens, int64_t heads_q,
              const int32_t* cu_seqlens, int64_t max_new, const WorkOf<TREE>& w, void* workspace, int64_t workspace_bytes,
              void* stream) {
  PagedCache c;
  if (int rc = check_cache(name, cache, dtype, &c)) return rc;
  if (!a.q || !a.o) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (int rc = check_tokens(name, tokens, cu_seqlens, &c)) return rc;
  if (heads_q <= 0 || heads_q > (1 << 16) || heads_q % cache->heads != 0)
    return fail(PA_ERR_INVALID, "%s: the query heads must be a multiple of the cache's heads", name);
  if (!aligned16(a.q) || !aligned16(a.o)) return fail(PA_ERR_INVALID, "%s: inputs must be 16-byte aligned", name);
  if (int rc = check_strides(name, {a.q_token, a.q_head, a.o_token, a.o_head})) return rc;
  const auto apart = [&](int64_t outer, int64_t outer_n, int64_t inner, int64_t inner_n) {
    return (inner_n == 1 || inner >= cache->d) && (outer_n == 1 || outer >= (inner_n - 1) * inner + cache->d);
  };
  if (!apart(a.o_token, tokens, a.o_head, heads_q) && !apart(a.o_head, heads_q, a.o_token, tokens))
    return fail(PA_ERR_INVALID, "%s: out's rows must not overlap", name);
  if (max_new < 0) return fail(PA_ERR_INVALID, "%s: max_new must not be negative", name);
  const AttnPlan plan = attn_plan(c, cache->d, is_8bit(cache->dtype), heads_q, max_new, TREE);
  if (int rc = check_work(name, c, plan, heads_q)) return rc;
  if (workspace_bytes < attn_workspace(plan.wgs, plan.rows, (int)cache->d) || !workspace || !aligned16(workspace))
    return fail(PA_ERR_INVALID, "%s: the workspace is too small, null or not 16-byte aligned", name);
  a.group = (int)(heads_q / cache->heads);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = with_types(dtype, cache->dtype, cache->d, [&](auto t, auto ct, auto dim) {
    typedef decltype(t) T;
    typedef decltype(ct) C;
    constexpr int D = decltype(dim)::value;
    constexpr int CR = chunk_rows_of(D);
    switch (plan.rows) {
      case 16: return launch_attn<T, D, 16>(paged_attn_few<T, C, D, 1, TREE>, 256, c, a, plan, w, workspace, st);
      case 32: return launch_attn<T, D, 32>(paged_attn_few<T, C, D, 2, TREE>, 256, c, a, plan, w, workspace, st);
      default: break;
    }
    if (past_buffer(c, D, cache_type<C>::k8bit))
      return launch_attn<T, D, CR>(paged_attn_chunk<T, C, D, CR, true, TREE>, 2 * CR, c, a, plan, w, workspace, st);
    if constexpr (TREE && CR != 128)
      if (plan.rows == 128) return launch_attn<T, D, 128>(paged_attn_chunk<T, C, D, 128, false, TREE>, 256, c, a, plan, w, workspace, st);
    return launch_attn<T, D, CR>(paged_attn_chunk<T, C, D, CR, false, TREE>, 2 * CR, c, a, plan, w, workspace, st);
  });
  return hip_status(e, name);
}

// Bytes of workspace of an attention call.
inline int64_t attn_workspace_of(const char* name, const pa_paged_cache* cache, int dtype, int64_t tokens, int64_t heads_q,
                                 const int32_t* cu_seqlens, int64_t max_new, bool tree) {
  PagedCache c;
  if (int rc = check_cache(name, cache, dtype, &c)) return rc;
  if (int rc = check_tokens(name, tokens, cu_seqlens, &c)) return rc;
  if (heads_q <= 0 || heads_q > (1 << 16) || heads_q % cache->heads != 0 || max_new < 0)
    return fail(PA_ERR_INVALID, "%s: the query heads must be a multiple of the cache's heads, max_new not negative", name);
  const AttnPlan plan = attn_plan(c, cache->d, is_8bit(cache->dtype), heads_q, max_new, tree);
  if (int rc = check_work(name, c, plan, heads_q)) return rc;
  return attn_workspace(plan.wgs, plan.rows, (int)cache->d);
}

}  // namespace pa
