/*
 * phantom_attn.h - C ABI of the MI355X (gfx950) attention-forward library libphantom_attn.so.
 *
 * This is the drop-in boundary for the reference's attention forward path. Each entry point
 * replaces one reference launcher (L1, csrc/kernels/<name>.cuh) together with the torch glue
 * around it (L2, csrc/attn_<name>.cu); the Python package cuda_attn binds these through ctypes
 * in place of the reference's pybind11 module cuda_attn._C (csrc/bindings.cpp:40-54).
 *
 * Conventions shared by every entry point
 *   - q, k, v, o are device pointers to contiguous [BH][N][d] arrays (the reference's
 *     (B, H, N, d) tensors viewed as [B*H][N][d], csrc/bindings.cpp:12-22). Inputs are only
 *     read; o is only written. The library never allocates or frees device memory: outputs and
 *     the score workspace of the unfused paths are allocated by the caller (pa_tiled_fwd_noalloc
 *     instead uses a fixed array compiled into the library).
 *   - dtype / out_dtype take the PA_DTYPE_* codes below. out_dtype lets a caller ask for fp32
 *     output from fp16/bf16 inputs (the reference always writes o in the input dtype).
 *   - stream is a hipStream_t passed as void* (NULL = the null stream). Launches are
 *     asynchronous; nothing synchronises.
 *   - Return value: 0 on success; a positive hipError_t from the HIP runtime; or a negative
 *     PA_ERR_* code for a rejected argument. pa_last_error() then returns a message for the
 *     calling thread (the reference turned cudaError_t into RuntimeError through ATTN_CHECK,
 *     csrc/common.cuh:21-25).
 *   - Every entry point is re-entrant; the only state is a thread-local error string and a
 *     per-device attribute cache.
 */
#ifndef PHANTOM_ATTN_H_
#define PHANTOM_ATTN_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum pa_dtype {
  PA_DTYPE_F32 = 0,
  PA_DTYPE_F16 = 1,
  PA_DTYPE_BF16 = 2,
  PA_DTYPE_I8 = 3,   /* these two: paged caches only */
  PA_DTYPE_E4M3 = 4  /* the OCP format: 4 exponent bits, 3 mantissa bits, largest value 448 */
};

enum pa_status {
  PA_OK = 0,
  PA_ERR_INVALID = -1,     /* bad pointer, size, dtype or flag */
  PA_ERR_UNSUPPORTED = -2  /* shape/dtype/tile combination that is not compiled */
};

/* v1 naive: three kernels, fp32 N x N scores in the caller's workspace s (BH*N*N floats).
 * dtype: F32 or F16 (out in the same dtype); any d >= 1.
 * Replaces attn::launch_naive (csrc/kernels/naive.cuh:55-64) and naive_forward
 * (csrc/attn_naive.cu:5-14). */
int pa_naive_fwd(const void* q, const void* k, const void* v, void* o, float* s,
                 int dtype, int64_t bh, int64_t n, int64_t d, int causal, void* stream);

/* v2 tiled: two kernels (scores; softmax and P.V) with the fp32 scores in workspace s between them,
 * or, for head dims that are not whole 16-byte rows up to 128, three. What s holds afterwards is not
 * specified.
 * dtype: F32 or F16; any d >= 1.
 * Replaces attn::launch_tiled (csrc/kernels/tiled.cuh:108-117) and tiled_forward
 * (csrc/attn_tiled.cu:5-14). */
int pa_tiled_fwd(const void* q, const void* k, const void* v, void* o, float* s,
                 int dtype, int64_t bh, int64_t n, int64_t d, int causal, void* stream);

/* tiled_forward without allocation: pa_tiled_fwd with the score workspace taken from a static
 * device array of the library instead of the caller. For callers that cannot allocate device
 * memory (code under stream/graph capture, serving loops, harnesses that forbid hipMalloc).
 * Limit: B*H*N*N <= 16777216 scores (64 MiB, held by every GPU the library runs on until the
 * process ends); larger calls return PA_ERR_UNSUPPORTED and should use pa_tiled_fwd. Calls no
 * allocating routine. Every call on one GPU shares that GPU's array: calls that overlap on one
 * GPU (two streams, two host threads) race and must be serialised by the caller.
 * No counterpart in the reference (its glue always allocates the workspace with torch,
 * csrc/attn_tiled.cu:5-14). */
int pa_tiled_fwd_noalloc(const void* q, const void* k, const void* v, void* o,
                         int dtype, int64_t bh, int64_t n, int64_t d, int causal, void* stream);

/* v3 fused: online softmax with fp32 arithmetic, errors against float64 no larger than the fp32 matrix
 * core's.
 * fp32 inputs: the fp32 matrix core, or, on larger grids, the bf16 one with Q, K, V and P in three bf16
 * terms each (24 significant bits from 2^-112 up, an absolute 2^-134 below) and the six largest term
 * products (what is left out of a product is below 2^-25 of it).
 * fp16 inputs: the fp16 matrix core, whose products are exact, with P in two fp16 terms (22
 * significant bits of a weight down to 2^-21 of its row's largest, an absolute 2^-43 of that below, which
 * fp16 output does not show). These calls take fused_tc's launch forms, and pa_set_persistent() applies to them.
 * dtype: F32 or F16; out_dtype: dtype or F32; d == 64.
 * Replaces attn::launch_fused<T> (csrc/kernels/fused.cuh:106-112) and fused_forward
 * (csrc/attn_fused.cu:5-14). */
int pa_fused_fwd(const void* q, const void* k, const void* v, void* o,
                 int dtype, int out_dtype, int64_t bh, int64_t n, int64_t d, int causal, void* stream);

/* v3.1/v3.2 fused_tuned: the fp16 MFMA kernel at query tile br and key tile bc, with
 * (double_buffer=1) or without (0) the two-stage LDS pipeline.
 * dtype: F16; out_dtype: F16 or F32; d == 64; (br, bc) in {(64,32),(64,64),(128,32),(128,64)}.
 * Replaces attn::launch_fused_tuned (csrc/kernels/fused_tuned.cuh:212-228) and
 * fused_tuned_forward (csrc/attn_fused_tuned.cu:5-21). */
int pa_fused_tuned_fwd(const void* q, const void* k, const void* v, void* o,
                       int dtype, int out_dtype, int64_t bh, int64_t n, int64_t d, int causal,
                       int double_buffer, int br, int bc, void* stream);

/* v4 fused_tc: QK^T and PV on MFMA (fp16/bf16 in, fp32 accumulate), online softmax between.
 * dtype: F16 or BF16; out_dtype: dtype or F32; d in {64, 128}.
 * The launch is persistent (as many workgroups as fit on the device at once, walking the query
 * blocks) for causal == 0 with an even number of 64-key tiles (or an odd number, above one, of
 * full ones), and for every causal != 0 call (its walk over the query blocks chosen from the
 * shape); unless pa_set_persistent(0) switched that off (see below). Otherwise one workgroup per
 * query block. pa_fused_tc_kernel names the choice.
 * Both launches give the same bits.
 * Replaces attn::launch_fused_tc (csrc/kernels/fused_tc.cuh:187-196) and fused_tc_forward
 * (csrc/attn_fused_tc.cu:5-19). */
int pa_fused_tc_fwd(const void* q, const void* k, const void* v, void* o,
                    int dtype, int out_dtype, int64_t bh, int64_t n, int64_t d, int causal,
                    void* stream);

/* The kernel instantiation and launch shape pa_fused_tc_fwd would use for these arguments, as
 * text ("" if the combination is not compiled). For reports and profiles; no GPU needed (without
 * a device the persistent launch is not chosen, as in pa_fused_tc_fwd).
 * No reference counterpart: the reference launches one fixed kernel (csrc/kernels/fused_tc.cuh:187-196). */
const char* pa_fused_tc_kernel(int dtype, int out_dtype, int64_t bh, int64_t n, int64_t d, int causal);

/* Process-wide switch of the persistent launch (fused_tc, and fused with fp16 inputs): enable = 0 selects one workgroup
 * per query block, nonzero the persistent launch. Returns the previous setting. The initial
 * setting is read once, when the library is loaded, from the environment variable
 * PA_PERSISTENT ("0" = off; unset or anything else = on). For A/B measurements and tests; calls
 * already launched are not affected.
 * No reference counterpart (the reference has one launch form). */
int pa_set_persistent(int enable);

/* LDS bytes one workgroup of fused_tuned needs, or -1 if (br, bc, d, dtype) is not compiled.
 * Replaces fused_tuned_smem_bytes (csrc/kernels/fused_tuned.cuh:188-190). No GPU needed. */
int64_t pa_fused_tuned_lds_bytes(int br, int bc, int double_buffer, int64_t d, int dtype);

/* LDS bytes one workgroup of fused_tc needs, or -1 if (d, dtype) is not compiled: the largest of
 * its launch forms (the persistent forms add rows that stage O before its stores).
 * Replaces fused_tc_smem_bytes (csrc/kernels/fused_tc.cuh:184). No GPU needed. */
int64_t pa_fused_tc_lds_bytes(int64_t d, int dtype);

/* LDS bytes one workgroup may use on `device`, written to *bytes.
 * Replaces smem_optin_bytes (csrc/common.cuh:35-40). */
int pa_device_lds_limit(int device, int64_t* bytes);

/* ---- Paged key/value cache: rows of earlier tokens kept in pages, and attention over them ----
 *
 * A cache is two arrays [pages][heads][page_size][d], one for keys and one for values. Position p of
 * sequence s is row p % page_size of page page_table[s * table_stride + p / page_size]; a table entry
 * outside [0, pages) is an absent page (not written, read as zeros, its keys not attended).
 * lengths[s] is the number of tokens sequence s holds once the call's new tokens are in the cache: its
 * new token i (of `count`) is at position lengths[s] - count + i. The new tokens of all sequences are
 * packed one after another, [tokens][heads][d] with the strides given (in elements, multiples of 8, the
 * d elements of a row contiguous); those of sequence s are the rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1,
 * or, with cu_seqlens NULL, tokens / seqs rows each. page_table, lengths and cu_seqlens are int32 on the
 * device and read by the kernels. Whatever they hold, no access leaves the tensors: rows without a
 * position in the table are not written and see no key; offsets are clamped to [0, tokens], and a row that
 * offsets out of order give to two sequences is written for the first of them and may hold either's result.
 *
 * dtype is the tensors' (F16 or BF16); the cache's own is the same, or I8 or E4M3 with an fp32 scale for
 * each row in k_scale / v_scale [pages][heads][page_size]: a row stands for code * scale.
 * d in {64, 128}. All pointers to rows 16-byte aligned. */
typedef struct pa_paged_cache {
  void* k;
  void* v;
  float* k_scale; /* 8-bit caches only */
  float* v_scale;
  const int32_t* page_table;
  const int32_t* lengths;
  int64_t pages, page_size, heads, d;
  int64_t seqs, table_cols, table_stride;
  int dtype;
} pa_paged_cache;

/* Writes the new tokens' keys and values to their positions. 8-bit caches: scale = amax / L and
 * code = round(x * (L / amax)) to nearest even in fp32, L = 127 (int8) or 448 (e4m3), amax the row's
 * largest magnitude; a row below 2^-100 is held as zeros, one with an element that is not finite gets a
 * NaN scale. The positions written in one call must be distinct: of two rows for one position either, or
 * parts of both, may remain. k and v may be rows of the cache itself, but none that the call writes. */
int pa_cache_write(const pa_paged_cache* cache, const void* k, const void* v, int dtype, int64_t tokens,
                   int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                   const int32_t* cu_seqlens, void* stream);

/* Lays the first n positions of every sequence out as [seqs][heads][n][d] (the other entry points'
 * layout) in dtype, code * scale rounded once; zeros from lengths[s] on. */
int pa_cache_read(const pa_paged_cache* cache, void* k, void* v, int dtype, int64_t n, void* stream);

/* Attention of the new tokens over the cache (which holds them already): new token i of sequence s sees
 * the positions up to its own (causal != 0) or all lengths[s] of them, scores scaled by 1/sqrt(d); a
 * token that sees nothing gets zeros, one whose visible scores are all -inf a NaN. q and o are [tokens][heads_q][d] with the strides given, heads_q a
 * multiple of the cache's heads (query head h reads head h / (heads_q / heads)); o must share no memory
 * with q or anything else that the call reads (its rows may lie between q's). Rows behind the last
 * sequence's are left as they are. max_new: an upper bound of the new tokens of a sequence, 0 if unknown;
 * only the choice of the kernel depends on it. workspace: pa_paged_attn_workspace() bytes of device memory,
 * 16-byte aligned, used until the call's kernels end; calls that may overlap need one each. */
int pa_paged_attn_fwd(const pa_paged_cache* cache, const void* q, void* o, int dtype, int64_t tokens, int64_t heads_q,
                      int64_t q_token_stride, int64_t q_head_stride, int64_t o_token_stride, int64_t o_head_stride,
                      const int32_t* cu_seqlens, int64_t max_new, int causal, void* workspace, int64_t workspace_bytes,
                      void* stream);

/* Bytes of workspace that pa_paged_attn_fwd needs for a call with these arguments; a negative PA_ERR_* code if it
 * refuses them (PA_ERR_UNSUPPORTED also where sequences, tokens and positions could make 2^62 steps of work). It
 * depends on sizes alone, not on what the tensors hold. No GPU needed. */
int64_t pa_paged_attn_workspace(const pa_paged_cache* cache, int dtype, int64_t tokens, int64_t heads_q,
                                const int32_t* cu_seqlens, int64_t max_new);

/* ---- Drafted tokens: a step that verifies several tokens of a sequence at once ----
 *
 * A sequence's new tokens of such a step are a tree: its token 0, the root, is certain; parents[i] (an index among the
 * sequence's new tokens, before i; anything else: none) is the token that token i was drafted behind. The new tokens of all
 * sequences are packed as above, tokens of sequence s being the rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1. The first
 * max_new (at most 1024) of a sequence are its tree. All of this is read by the kernels, and whatever it holds, no access
 * leaves the tensors. Results and workspaces share no memory with each other or with anything that a call reads, where nothing
 * else is said. */

/* mask[i], ceil(max_new / 32) words a token: bit j % 32 of word j / 32 is set for j the token itself or one of its
 * ancestors (tokens behind the tree: none). positions[i]: that of the sequence's first new token, lengths[s] - count, plus
 * the token's depth. Rows behind the last sequence's are left as they are. cu_seqlens NULL: tokens / seqs each. */
int pa_draft_tree(const int32_t* parents, const int32_t* lengths, const int32_t* cu_seqlens, int64_t tokens, int64_t seqs,
                  int64_t max_new, int32_t* mask, int32_t* positions, void* stream);

/* pa_paged_attn_fwd with a mask in the place of `causal`: a new token sees the positions before its sequence's new tokens,
 * and the new token j whose bit j % 32 of word j / 32 is set in its row mask + i * mask_stride (mask_words words, those past
 * them 0; any bits, not only a tree's). Workspace: pa_paged_tree_attn_workspace() bytes, otherwise as there. */
int pa_paged_tree_attn_fwd(const pa_paged_cache* cache, const void* q, void* o, int dtype, int64_t tokens, int64_t heads_q,
                           int64_t q_token_stride, int64_t q_head_stride, int64_t o_token_stride, int64_t o_head_stride,
                           const int32_t* cu_seqlens, int64_t max_new, const int32_t* mask, int64_t mask_words,
                           int64_t mask_stride, void* workspace, int64_t workspace_bytes, void* stream);
int64_t pa_paged_tree_attn_workspace(const pa_paged_cache* cache, int dtype, int64_t tokens, int64_t heads_q,
                                     const int32_t* cu_seqlens, int64_t max_new);

/* Rows to turn: [b][n][heads][d] with the strides given, in elements; the d elements of a row contiguous. out may be in,
 * with its strides; otherwise they share no memory. */
typedef struct pa_rope_rows {
  const void* in;
  void* out;
  int64_t in_b, in_n, in_h, out_b, out_n, out_h;
  int64_t heads;
} pa_rope_rows;

/* Rotary positions of queries and (k not NULL) keys. dtype: F32, F16 or BF16; d up to 1024. The first 2 * pairs elements of
 * a row are turned, pair p by positions[..] * freqs[p] (inverse != 0: by its negative): (x, y) becomes
 * scale * (x cos - y sin, x sin + y cos). Pairs are elements p and p + pairs, or (interleaved != 0) 2 p and 2 p + 1. The
 * others are copied. positions: int32, or int64 (positions64 != 0), of token (b, n) at b * position_b + n * position_n.
 * Angles are in 64 bits, right at any 32-bit position. */
int pa_rope(const pa_rope_rows* q, const pa_rope_rows* k, int dtype, int64_t b, int64_t n, int64_t d, const void* positions,
            int positions64, int64_t position_b, int64_t position_n, const double* freqs, int64_t pairs, int interleaved,
            int inverse, float scale, void* stream);

/* Verification of drafted tokens. From each sequence's root on, the drafts behind the current token are tried in order,
 * and the first one accepted becomes the current token. With p, q the current token's rows of target_probs and draft_probs
 * [n_tokens][vocab], t the draft's token and u its number in uniform [n_tokens]:
 *   draft_probs given (each draft a sample of its parent's row): accepted iff u q(t) S(c) < max(p(t) - c q(t), 0), where
 *     c = 0 and S(0) = 1 at first; after each rejection c grows by S(c), the sum of max(p - c q, 0);
 *   draft_probs NULL (drafts chosen without chance): accepted iff u m < p(t), m = 1 at first; after each rejection m falls by
 *     p(t), and t counts as 0.
 * Then the next token: the first whose sum of weights up to it exceeds u S, u the root's number, S the sum of the weights
 * max(p - c q, 0) (or of p but for the rejected tokens); p where those are all 0; -1 where p is too. An element of p or q
 * that is not a positive finite number is 0; a draft whose token is not in [0, vocab) is none. Sums, products and comparisons
 * are in 64 bits. path [seqs][max_new]: the accepted tokens, root first, as indices among the sequence's new tokens, then
 * -1; accepted [seqs]: their number, the root's among them; next_tokens [seqs]. A sequence without tokens: -1, 0, -1.
 * Strides in elements. vocab up to 2^24, seqs up to 65535. workspace: pa_verify_draft_workspace() bytes (drawn: whether
 * draft_probs are given), 16-byte aligned; calls that may overlap need one each. 0 bytes: it may be NULL. */
int pa_verify_draft(const int64_t* tokens, const int32_t* parents, const float* target_probs, int64_t target_stride,
                    const float* draft_probs, int64_t draft_stride, const float* uniform, const int32_t* cu_seqlens,
                    int64_t n_tokens, int64_t seqs, int64_t vocab, int64_t max_new, int32_t* path, int32_t* accepted,
                    int64_t* next_tokens, void* workspace, int64_t workspace_bytes, void* stream);
int64_t pa_verify_draft_workspace(int64_t seqs, int64_t vocab, int drawn);

/* Leaves of a step's new tokens the accepted ones: row path[s * path_stride + j] of sequence s's new tokens becomes row j,
 * j = 0 .. accepted[s] - 1, keys, values and scales, in place. Paths must ascend (as pa_verify_draft's do); an entry that is
 * no new token leaves its row as it is. new_lengths[s] = lengths[s] - count + accepted[s], at least 0; it shares no memory with
 * lengths or anything else that the call reads (every layer's call takes the same lengths). */
int pa_cache_keep(const pa_paged_cache* cache, const int32_t* path, int64_t path_width, int64_t path_stride,
                  const int32_t* accepted, const int32_t* cu_seqlens, int32_t* new_lengths, void* stream);

/* Message for the last nonzero status returned on this thread ("" if none). */
const char* pa_last_error(void);

/* Library version and the offload architecture it was compiled for. */
const char* pa_version(void);

#ifdef __cplusplus
}
#endif

#endif /* PHANTOM_ATTN_H_ */
