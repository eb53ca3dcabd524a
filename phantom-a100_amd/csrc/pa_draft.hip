// C ABI of the operators around drafted tokens: rotary positions, trees of drafts, their verification, and the cache rows
// of the accepted ones. Argument checks and launches on the caller's stream; no allocation, no synchronisation.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "paged_host.hpp"
#include "kernels/draft.hpp"
#include "kernels/rope.hpp"

namespace {

using pa::aligned16;
using pa::fail;
using pa::hip_status;

// Where a head's tokens follow each other, (B, heads, N, d), groups of several tokens read longer runs of memory, and 4096
// workgroups are enough. us with groups of 1, 2, 4 and 8: 4 x 4096 tokens, 64 heads of 128, half turned 116, 106, 104, 108 (of 4
// on 2048 workgroups 105; all turned 109, 108, 102, on 2048 112); 4 x 8192, 32 heads of 64 71, 57, 54, 51; 8 x 8192, 32 of 128, half
// turned 248, 241, 222, 209; 16 x 4096, 16 of 64, half turned 89, 64, 54, 49 (of 16, as the rule has it, 51); 2 x 4096, 32 of 128
// 29, 29, 27. Packed tokens of 40 heads, 32768 of them, one each 120 us, four 129.
constexpr int64_t kRopeBlocks = 4096;
template <typename T, int W>
hipError_t launch_rope(const pa::RopeArgs& a, bool interleaved, hipStream_t stream) {
  const unsigned blocks = (unsigned)std::min<int64_t>((a.tokens + a.group - 1) / a.group, 1 << 22);
  if (interleaved) hipLaunchKernelGGL((pa::rope_rows<T, W, true>), dim3(blocks), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((pa::rope_rows<T, W, false>), dim3(blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_rope(pa::RopeArgs a, int width, bool interleaved, hipStream_t stream) {
  const int wide = interleaved ? std::max(width, 2) : 2 * width;
  a.units = interleaved ? (a.d + wide - 1) / wide : a.pairs / width + (a.d - 2 * a.pairs + wide - 1) / wide;
  a.heads = a.x[0].heads + a.x[1].heads;
  // Tokens of a workgroup at a time: as many as give each thread a unit; where a head's tokens follow each other in memory,
  // as many as there are threads for their angles, but at least kRopeBlocks workgroups.
  a.heads_outer = a.x[0].in_h > a.x[0].in_n;
  const int64_t token_units = (int64_t)a.heads * a.units;
  const int64_t fill = std::min<int64_t>(256 / token_units, pa::kRopeTurns / a.pairs);
  const int64_t run = a.heads_outer ? std::min<int64_t>({256 / a.pairs, a.tokens / kRopeBlocks, (1 << 30) / token_units}) : 1;
  a.group = (int)std::max<int64_t>({fill, run, 1});
  a.by_n = pa::make_page_div((uint32_t)a.n), a.by_pairs = pa::make_page_div((uint32_t)a.pairs);
  a.by_units = pa::make_page_div((uint32_t)a.units);
  a.by_inner = pa::make_page_div((uint32_t)((a.heads_outer ? a.group : a.heads) * a.units));
  switch (width) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_rope<T, 8>(a, interleaved, stream);
    case 4: return launch_rope<T, 4>(a, interleaved, stream);
    case 2: return launch_rope<T, 2>(a, interleaved, stream);
    default: return launch_rope<T, 1>(a, interleaved, stream);
  }
}

int64_t verify_runs(int64_t vocab) { return (vocab + pa::kRun - 1) / pa::kRun; }
// Rows of so many elements go in one workgroup and one launch: up to 32 runs, 64 where drafts were drawn (a third launch
// saved, of a call that has three). 48 chains of 8 over 32000 and 65537 tokens, in a graph: 9.5 and 13.3 us, in three
// launches 10.3 and 11.6, and from Python, where a launch costs 2.3 us more, 16 for 21; one chain without, 9.6 and
// 13.0 for 9.0 and 9.1, from Python 15.5 for 17.8.
bool verify_in_one(int64_t vocab, bool drawn) { return verify_runs(vocab) <= (drawn ? 64 : 32); }
int64_t verify_state_bytes(int64_t seqs) { return seqs * (int64_t)sizeof(pa::VerifyState); }
int check_verify_sizes(const char* name, int64_t seqs, int64_t vocab) {
  if (seqs <= 0 || vocab <= 0) return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (seqs > 65535) return fail(PA_ERR_UNSUPPORTED, "%s: more than 65535 sequences", name);
  if (vocab > (1 << 24)) return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^24 tokens in the vocabulary", name);
  return PA_OK;
}

}  // namespace

extern "C" {

int pa_rope(const pa_rope_rows* q, const pa_rope_rows* k, int dtype, int64_t b, int64_t n, int64_t d, const void* positions,
            int positions64, int64_t position_b, int64_t position_n, const double* freqs, int64_t pairs, int interleaved,
            int inverse, float scale, void* stream) {
  const char* name = "rope";
  if (!q || !positions || !freqs) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (dtype != PA_DTYPE_F32 && dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_BF16)
    return fail(PA_ERR_UNSUPPORTED, "%s: float32, float16 or bfloat16 only", name);
  if (b <= 0 || n <= 0 || d <= 0 || pairs <= 0) return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (d > pa::kRopeMaxDim) return fail(PA_ERR_UNSUPPORTED, "%s: head dims up to %d", name, pa::kRopeMaxDim);
  if (pairs > d / 2) return fail(PA_ERR_INVALID, "%s: more pairs than a head has", name);
  if (n > pa::kPagedMaxPos || b > pa::kPagedMaxPos / n) return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^30 tokens", name);
  const int64_t size = dtype == PA_DTYPE_F32 ? 4 : 2;
  pa::RopeArgs a{};
  a.positions = positions, a.freqs = freqs, a.pos_b = position_b, a.pos_n = position_n;
  a.tokens = b * n, a.n = (int)n, a.d = (int)d, a.pairs = (int)pairs;
  a.pos64 = positions64, a.inverse = inverse, a.scale = scale;
  // The widest unit that everything is a multiple of: 16 bytes where a quarter of a row's bytes and all strides are.
  int64_t width = 16 / size;
  auto fits = [&](int64_t x, int64_t unit) {
    while (x % (width * unit) != 0) width /= 2;
  };
  fits(interleaved ? 2 * pairs : pairs, 1), fits(d, 1);

  for (int i = 0; i < 2; ++i) {
    const pa_rope_rows* x = i ? k : q;
    if (!x) continue;
    if (!x->in || !x->out) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
    if (x->heads <= 0 || x->heads > (1 << 16)) return fail(PA_ERR_INVALID, "%s: 1 to 65536 heads", name);
    for (int64_t s : {x->in_b, x->in_n, x->in_h, x->out_b, x->out_n, x->out_h})
      if (s < 0) return fail(PA_ERR_INVALID, "%s: strides must not be negative", name);
    const uintptr_t in = reinterpret_cast<uintptr_t>(x->in), out = reinterpret_cast<uintptr_t>(x->out);
    if (in % size || out % size) return fail(PA_ERR_INVALID, "%s: inputs must be aligned to their elements", name);
    fits((int64_t)((in | out) % 16), size);
    if (b > 1) fits(x->in_b, 1), fits(x->out_b, 1);
    if (n > 1) fits(x->in_n, 1), fits(x->out_n, 1);
    if (x->heads > 1) fits(x->in_h, 1), fits(x->out_h, 1);
    a.x[i] = pa::RopeRows{x->in, x->out, x->in_b, x->in_n, x->in_h, x->out_b, x->out_n, x->out_h, (int)x->heads};

  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = dtype == PA_DTYPE_F32   ? launch_rope<float>(a, (int)width, interleaved != 0, st)
                       : dtype == PA_DTYPE_F16 ? launch_rope<pa::f16>(a, (int)width, interleaved != 0, st)
                                               : launch_rope<pa::bf16>(a, (int)width, interleaved != 0, st);
  return hip_status(e, name);
}

int pa_draft_tree(const int32_t* parents, const int32_t* lengths, const int32_t* cu_seqlens, int64_t tokens, int64_t seqs,
                  int64_t max_new, int32_t* mask, int32_t* positions, void* stream) {
  const char* name = "draft_tree";
  if (!parents || !lengths || !mask || !positions) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (tokens <= 0 || seqs <= 0) return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (tokens > pa::kPagedMaxPos || seqs > (1 << 22)) return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^30 tokens or 2^22 sequences", name);
  if (max_new <= 0 || max_new > pa::kTreeMax)
    return fail(PA_ERR_INVALID, "%s: max_new must be a number of tokens from 1 to %d", name, pa::kTreeMax);
  if (!cu_seqlens && tokens % seqs != 0)
    return fail(PA_ERR_INVALID, "%s: without cu_seqlens the tokens must divide evenly over the sequences", name);
  const int words = (int)((max_new + 31) / 32);
  // (a sequence's workgroups write rows while others still read its parents)
  if (pa::any_shared({{mask, tokens * words * 4}, {positions, tokens * 4}},
                     {{parents, tokens * 4}, {lengths, seqs * 4}, {cu_seqlens, (seqs + 1) * 4}}))
    return fail(PA_ERR_INVALID, "%s: results must share no memory with each other or with what the call reads", name);
  const pa::TreeArgs a{parents, lengths, cu_seqlens, (int)tokens, cu_seqlens ? 0 : (int)(tokens / seqs), (int)max_new, words,
                       mask, positions};
  const int64_t y = std::min<int64_t>((max_new * words + 255) / 256, 64);
  hipLaunchKernelGGL(pa::draft_tree_rows, dim3((unsigned)seqs, (unsigned)y), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return hip_status(hipGetLastError(), name);
}

int64_t pa_verify_draft_workspace(int64_t seqs, int64_t vocab, int drawn) {
  if (int rc = check_verify_sizes("verify_draft", seqs, vocab)) return rc;
  if (verify_in_one(vocab, drawn != 0)) return 0;
  return verify_state_bytes(seqs) + seqs * verify_runs(vocab) * (int64_t)sizeof(double);
}

int pa_verify_draft(const int64_t* tokens, const int32_t* parents, const float* target_probs, int64_t target_stride,
                    const float* draft_probs, int64_t draft_stride, const float* uniform, const int32_t* cu_seqlens,
                    int64_t n_tokens, int64_t seqs, int64_t vocab, int64_t max_new, int32_t* path, int32_t* accepted,
                    int64_t* next_tokens, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "verify_draft";
  if (!tokens || !parents || !target_probs || !uniform || !cu_seqlens || !path || !accepted || !next_tokens)
    return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (int rc = check_verify_sizes(name, seqs, vocab)) return rc;
  if (n_tokens <= 0) return fail(PA_ERR_INVALID, "%s: inputs must be non-empty", name);
  if (n_tokens > pa::kPagedMaxPos) return fail(PA_ERR_UNSUPPORTED, "%s: more than 2^30 tokens", name);
  if (max_new <= 0 || max_new > pa::kTreeMax)
    return fail(PA_ERR_INVALID, "%s: max_new must be a number of tokens from 1 to %d", name, pa::kTreeMax);
  if (target_stride < 0 || draft_stride < 0) return fail(PA_ERR_INVALID, "%s: strides must not be negative", name);
  const bool in_one = verify_in_one(vocab, draft_probs != nullptr);
  const int64_t need = pa_verify_draft_workspace(seqs, vocab, draft_probs != nullptr);
  if (!in_one && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(PA_ERR_INVALID, "%s: the workspace is too small, null or not 16-byte aligned", name);
  // (one workgroup of a sequence writes its path while others still walk)
  if (pa::any_shared({{path, seqs * max_new * 4}, {accepted, seqs * 4}, {next_tokens, seqs * 8}, {need ? workspace : nullptr, need}},
                     {{tokens, n_tokens * 8}, {parents, n_tokens * 4}, {uniform, n_tokens * 4}, {cu_seqlens, (seqs + 1) * 4},
                      {target_probs, pa::span_bytes(n_tokens, target_stride, vocab, 4)},
                      {draft_probs, pa::span_bytes(n_tokens, draft_stride, vocab, 4)}}))
    return fail(PA_ERR_INVALID, "%s: results and workspace must share no memory with each other or with what the call reads", name);
  const int runs = (int)verify_runs(vocab);
  pa::VerifyState* states = static_cast<pa::VerifyState*>(workspace);
  const pa::VerifyArgs a{tokens, parents, target_probs, draft_probs, uniform, cu_seqlens, target_stride, draft_stride,
                         (int)n_tokens, (int)vocab, (int)max_new, runs, path, accepted, next_tokens, states,
                         reinterpret_cast<double*>(static_cast<char*>(workspace) + verify_state_bytes(seqs))};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 four((unsigned)((runs + 3) / 4), (unsigned)seqs), each((unsigned)seqs);
  if (in_one) {
    const unsigned lds = (unsigned)(runs * sizeof(double));
    if (draft_probs) hipLaunchKernelGGL((pa::verify_whole<true>), each, dim3(1024), lds, st, a);
    else hipLaunchKernelGGL((pa::verify_whole<false>), each, dim3(1024), lds, st, a);
    return hip_status(hipGetLastError(), name);
  }
  if (draft_probs) {
    hipLaunchKernelGGL(pa::verify_drawn, each, dim3(1024), 0, st, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return hip_status(e, name);
    hipLaunchKernelGGL((pa::verify_sums<true>), four, dim3(256), 0, st, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return hip_status(e, name);
    hipLaunchKernelGGL((pa::verify_pick<true>), each, dim3(pa::kWave), 0, st, a);
  } else {
    hipLaunchKernelGGL((pa::verify_sums<false>), four, dim3(256), 0, st, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return hip_status(e, name);
    hipLaunchKernelGGL((pa::verify_pick<false>), each, dim3(pa::kWave), 0, st, a);
  }
  return hip_status(hipGetLastError(), name);
}

int pa_cache_keep(const pa_paged_cache* cache, const int32_t* path, int64_t path_width, int64_t path_stride,
                  const int32_t* accepted, const int32_t* cu_seqlens, int32_t* new_lengths, void* stream) {
  const char* name = "cache_keep";
  pa::PagedCache c;
  if (!cache) return fail(PA_ERR_INVALID, "%s: null cache", name);
  // (rows move as they are: an 8-bit cache is checked as one of fp16 tensors)
  if (int rc = pa::check_cache(name, cache, pa::is_8bit(cache->dtype) ? PA_DTYPE_F16 : cache->dtype, &c)) return rc;
  if (!path || !accepted || !cu_seqlens || !new_lengths) return fail(PA_ERR_INVALID, "%s: null tensor pointer", name);
  if (path_width <= 0 || path_width > pa::kPagedMaxPos || path_stride < 0)
    return fail(PA_ERR_INVALID, "%s: path must have 1 to 2^30 columns and a stride that is not negative", name);
  c.cu = cu_seqlens;
  c.tokens = (int)pa::kPagedMaxPos;
  if (!pa::is_8bit(cache->dtype)) c.k_scale = c.v_scale = nullptr;
  const int64_t bytes = cache->d * (pa::is_8bit(cache->dtype) ? 1 : 2), columns = 2 * cache->heads * (bytes / 16);
  const int64_t y = (columns + 255) / 256;
  if (y > 65535) return fail(PA_ERR_UNSUPPORTED, "%s: too many heads for one launch", name);
  // (the first workgroup of a sequence writes its length while others still read what the call is given)
  const int64_t seqs = cache->seqs, rows = cache->pages * cache->heads * cache->page_size, scales = c.k_scale ? rows * 4 : 0;
  if (pa::any_shared({{new_lengths, seqs * 4}},
                     {{cache->lengths, seqs * 4}, {accepted, seqs * 4}, {cu_seqlens, (seqs + 1) * 4},
                      {path, pa::span_bytes(seqs, path_stride, path_width, 4)},
                      {cache->page_table, pa::span_bytes(seqs, cache->table_stride, cache->table_cols, 4)}, {cache->k, rows * bytes},
                      {cache->v, rows * bytes}, {c.k_scale, scales}, {c.v_scale, scales}}))
    return fail(PA_ERR_INVALID, "%s: new_lengths must share no memory with what the call reads", name);
  const pa::KeepArgs a{path, accepted, new_lengths, path_stride, (int)path_width};
  const dim3 grid((unsigned)cache->seqs, (unsigned)y);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (bytes) {
    case 64: hipLaunchKernelGGL((pa::cache_keep_rows<64>), grid, dim3(256), 0, st, c, a); break;
    case 128: hipLaunchKernelGGL((pa::cache_keep_rows<128>), grid, dim3(256), 0, st, c, a); break;
    default: hipLaunchKernelGGL((pa::cache_keep_rows<256>), grid, dim3(256), 0, st, c, a); break;
  }
  return hip_status(hipGetLastError(), name);
}

}  // extern "C"
