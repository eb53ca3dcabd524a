"""The paged key/value cache: rows of earlier tokens kept in pages, and attention of new tokens over them.

    cuda_attn.cache_write(k, v, k_cache, v_cache, page_table, lengths, cu_seqlens)   # the new tokens' rows
    o = cuda_attn.paged_attn(q, k_cache, v_cache, page_table, lengths, cu_seqlens)   # their attention
    kd, vd = cuda_attn.cache_read(k_cache, v_cache, page_table, lengths)             # dense (B, H, N, d) again

Tensors, all on one GPU:

    k_cache, v_cache   (pages, heads, page_size, d), contiguous, d = 64 or 128. float16 or bfloat16 like q, k
                       and v, or int8 / float8_e4m3fn with k_scale, v_scale (pages, heads, page_size) float32:
                       a row stands for code * scale.
    page_table         (B, columns) int32. Position p of sequence s is row p % page_size of page
                       page_table[s, p // page_size]. An entry that is no page (-1, say) is absent: nothing
                       is written there, it reads as zeros and its keys are not attended.
    lengths            (B,) int32: the tokens each sequence holds once the new ones are in.
    q, k, v            (tokens, heads, d): the new tokens of all sequences, one sequence after another; views
                       with any token and head strides of whole 16-byte steps (slices of one projection, say).
    cu_seqlens         (B + 1,) int32: sequence s has rows cu_seqlens[s] to cu_seqlens[s + 1] - 1, at positions
                       lengths[s] - count to lengths[s] - 1. None: tokens / B rows each (B rows: one token each).

page_table, lengths and cu_seqlens are read on the GPU, so a captured call follows what they hold when it is
replayed. Whatever they hold, no access leaves the tensors. Rows behind the last sequence's are ignored.
"""
from __future__ import annotations

import struct

import torch

from . import _checks, _native

_DTYPE_CODE = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16,
               torch.int8: _native.DTYPE_I8, torch.float8_e4m3fn: _native.DTYPE_E4M3}


_pack = struct.Struct("PPPPPPqqqqqqqi4x").pack   # pa_paged_cache, several times faster than its fields one by one


def _cache_args(k_cache, v_cache, page_table, lengths, k_scale, v_scale):
    pages, heads, page_size, d = k_cache.shape
    seqs, cols = page_table.shape
    return _native.PagedCacheArgs.from_buffer_copy(_pack(
        k_cache.data_ptr(), v_cache.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
        0 if v_scale is None else v_scale.data_ptr(), page_table.data_ptr(), lengths.data_ptr(),
        pages, page_size, heads, d, seqs, cols, page_table.stride(0), _DTYPE_CODE[k_cache.dtype]))


def _check(name, rows, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale):
    if not _checks.paged_ok(rows, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale):
        _checks.check_paged(name, rows, k_cache, v_cache, page_table, lengths, k_scale, v_scale)
        if rows is not None:
            _checks.check_rows(name, rows, k_cache, lengths, cu_seqlens)


def cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                page_table: torch.Tensor, lengths: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """Write the new tokens' keys and values, (tokens, heads, d), to their positions in the cache.

    An 8-bit cache gets codes and scales: scale = amax / L, code = round(x * (L / amax)) to nearest even in
    fp32, with amax the row's largest magnitude and L = 127 (int8) or 448 (float8_e4m3fn). A row below 2**-100
    is held as zeros; one with an element that is not finite gets a NaN scale. The positions written in one
    call must be distinct (no page shared by two sequences where both write). k and v may be rows of the cache
    itself (a page copied to another), but none that the call writes."""
    from . import _call, _stream_ptr

    _check("cache_write", k, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale)
    _checks.check_same_rows("cache_write", k, v, k_cache)
    ks, vs = k.stride(), v.stride()
    cache = _cache_args(k_cache, v_cache, page_table, lengths, k_scale, v_scale)
    _call("pa_cache_write", "cache_write", k.device, cache, k.data_ptr(), v.data_ptr(), _DTYPE_CODE[k.dtype], k.shape[0],
          ks[0], ks[1], vs[0], vs[1], None if cu_seqlens is None else cu_seqlens.data_ptr(),
          _stream_ptr(k.device))


def cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
               max_len: int | None = None, dtype: torch.dtype | None = None, k_scale: torch.Tensor | None = None,
               v_scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The cache's rows as two (B, heads, N, d) tensors, the layout of the other entry points.

    N is max_len (default: all columns of the page table). Rows from a sequence's length on are zeros. dtype:
    the cache's own, or, for an 8-bit cache, float16 or bfloat16 (required): code * scale rounded once."""
    from . import _call, _stream_ptr

    dtype = _checks.read_dtype("cache_read", k_cache, dtype)
    _check("cache_read", None, k_cache, v_cache, page_table, lengths, None, k_scale, v_scale)
    b, (_, heads, page_size, d) = page_table.shape[0], k_cache.shape
    n = page_table.shape[1] * page_size if max_len is None else max_len
    _checks.check_max_len("cache_read", n)
    k = torch.empty((b, heads, n, d), dtype=dtype, device=k_cache.device)
    v = torch.empty_like(k)
    cache = _cache_args(k_cache, v_cache, page_table, lengths, k_scale, v_scale)
    _call("pa_cache_read", "cache_read", k.device, cache, k.data_ptr(), v.data_ptr(), _DTYPE_CODE[dtype], n,
          _stream_ptr(k.device))
    return k, v


def paged_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
               lengths: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *, causal: bool = True,
               max_new: int | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the new tokens, q (tokens, heads_q, d), over the cache, which holds their keys already.

    A token sees the positions up to its own (causal) or all of its sequence's; scores are scaled by
    1/sqrt(d); query head h reads the cache's head h // (heads_q / heads). A token that sees nothing gets
    zeros, one whose visible scores are all -inf a NaN. max_new, an upper bound of the new tokens of a sequence, picks the kernel where cu_seqlens hides
    it (a wrong one costs time, not correctness). out: where to write (q's shape and dtype, strides of whole
    16-byte steps, no memory shared with q or the other tensors; with q's own strides its rows may lie between
    q's, as slices of one buffer do); its rows behind the last sequence's stay as they are, those of a new
    tensor are not set."""
    from . import _call, _stream_ptr

    _check("paged_attn", q, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale)
    _checks.check_query_heads("paged_attn", q, k_cache)
    if out is None:
        out = torch.empty_like(q)
    else:
        _checks.check_out("paged_attn", q, out, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale)
    bound = 0 if max_new is None else _checks.check_max_new("paged_attn", max_new)
    cache = _cache_args(k_cache, v_cache, page_table, lengths, k_scale, v_scale)
    tokens, heads_q, _ = q.shape
    code = _DTYPE_CODE[q.dtype]
    cu = None if cu_seqlens is None else cu_seqlens.data_ptr()
    need = _native.lib().pa_paged_attn_workspace(cache, code, tokens, heads_q, cu, bound)
    if need < 0:
        _native.check(need, "paged_attn")
    workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    qs, outs = q.stride(), out.stride()
    _call("pa_paged_attn_fwd", "paged_attn", q.device, cache, q.data_ptr(), out.data_ptr(), code, tokens, heads_q,
          qs[0], qs[1], outs[0], outs[1], cu, bound, 1 if causal else 0, workspace.data_ptr(),
          need, _stream_ptr(q.device))
    return out
