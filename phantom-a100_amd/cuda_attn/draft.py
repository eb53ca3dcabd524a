"""Steps that verify several drafted tokens of a sequence at once, over the paged cache (paged.py).

    mask, positions = cuda_attn.draft_tree(parents, lengths, cu_seqlens, max_new=n)
    # each layer: rope to `positions`, cache_write, then
    o = cuda_attn.paged_tree_attn(q, k_cache, v_cache, page_table, lengths, mask, cu_seqlens, max_new=n)
    # the target's and the draft's probabilities behind each token
    path, accepted, token = cuda_attn.verify_draft(tokens, parents, target_probs, uniform, cu_seqlens,
                                                   draft_probs=draft_probs, max_new=n)
    for k_cache, v_cache in caches:   # each layer's, all from the lengths with the new tokens
        after = cuda_attn.cache_keep(k_cache, v_cache, page_table, lengths, path, accepted, cu_seqlens)
    lengths = after

A sequence's new tokens are a tree. Its token 0, the root, is certain: the one that the last step drew. parents (tokens,)
int32 holds for each other token the one that it was drafted behind, as an index among the sequence's new tokens and
before its own; for a chain of drafts, 0, 1, 2, ... behind the root's -1. An entry that is no earlier token is none. The
first max_new tokens of a sequence, at most 1024, are its tree. The new tokens of all sequences are packed as in
paged.py, cu_seqlens (B + 1,) int32 their offsets. Everything that is on the GPU is read there, so that a captured call
follows it; whatever it holds, no access leaves the tensors.
"""
from __future__ import annotations

import torch

from . import _call, _checks, _native, _stream_ptr
from .paged import _DTYPE_CODE, _cache_args, _check

TREE_MAX = 1024


def draft_tree(parents: torch.Tensor, lengths: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
               max_new: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Masks and positions of trees of drafted tokens: (mask, positions), both int32.

    mask is (tokens, ceil(max_new / 32)): bit j % 32 of word j / 32 of a token's row is set for itself and its ancestors,
    j being indices among the sequence's new tokens. positions is (tokens,): lengths - count, where the sequence's
    first new token is, plus the token's depth. lengths (B,) int32 counts the new tokens. max_new: the most new tokens of
    a sequence (default: tokens / B without cu_seqlens, else all tokens, up to 1024). Rows behind the last sequence's
    are not set."""
    seqs = lengths.shape
    if cu_seqlens is not None and len(seqs) == 1 and _checks.trees_ok(
            parents, ((lengths, torch.int32, seqs), (cu_seqlens, torch.int32, (seqs[0] + 1,))), max_new):
        most = max_new
    else:
        _checks.check_vector("draft_tree", "lengths", lengths, torch.int32, None, parents.device)
        most = _checks.check_tree("draft_tree", parents, seqs[0], cu_seqlens, max_new)
    tokens = parents.shape[0]
    mask = torch.empty((tokens, (most + 31) // 32), dtype=torch.int32, device=parents.device)
    positions = torch.empty_like(parents)
    _call("pa_draft_tree", "draft_tree", parents.device, parents.data_ptr(), lengths.data_ptr(),
          None if cu_seqlens is None else cu_seqlens.data_ptr(), tokens, seqs[0], most, mask.data_ptr(),
          positions.data_ptr(), _stream_ptr(parents.device))
    return mask, positions


def paged_tree_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, mask: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                    max_new: int | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """paged_attn with a mask over the new tokens: attention of trees of drafted tokens over the cache.

    A token sees the positions before its sequence's new tokens, and the new token j (the one at lengths - count + j) where
    bit j % 32 of word j / 32 of its row of mask, (tokens, words) int32 with contiguous rows, is set; words past the row are
    0. Masks need not be a tree's: what a row sees is what its bits say, itself included. All else is paged_attn's:
    scores scaled by 1/sqrt(d), zeros for a token that sees nothing, query heads in groups, the cache in 16 or 8 bits,
    max_new a hint, out."""
    name = "paged_tree_attn"
    _check(name, q, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale)
    _checks.check_query_heads(name, q, k_cache)
    _checks.check_mask(name, mask, q)
    if out is None:
        out = torch.empty_like(q)
    else:
        _checks.check_out(name, q, out, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale)
        _checks.check_no_overlap(name, out, mask, "the mask")
    bound = 0 if max_new is None else _checks.check_max_new(name, max_new)
    cache = _cache_args(k_cache, v_cache, page_table, lengths, k_scale, v_scale)
    tokens, heads_q, _ = q.shape
    code = _DTYPE_CODE[q.dtype]
    cu = None if cu_seqlens is None else cu_seqlens.data_ptr()
    need = _native.lib().pa_paged_tree_attn_workspace(cache, code, tokens, heads_q, cu, bound)
    if need < 0:
        _native.check(need, name)
    workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    qs, outs = q.stride(), out.stride()
    _call("pa_paged_tree_attn_fwd", name, q.device, cache, q.data_ptr(), out.data_ptr(), code, tokens, heads_q,
          qs[0], qs[1], outs[0], outs[1], cu, bound, mask.data_ptr(), mask.shape[1], mask.stride(0),
          workspace.data_ptr(), need, _stream_ptr(q.device))
    return out


def verify_draft(tokens: torch.Tensor, parents: torch.Tensor, target_probs: torch.Tensor, uniform: torch.Tensor,
                 cu_seqlens: torch.Tensor, *, draft_probs: torch.Tensor | None = None,
                 max_new: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Verify drafted tokens so that what is kept is distributed as the target's own samples: (path, accepted, next).

    tokens (tokens,) int64: the vocabulary's numbers of the new tokens (the roots' are not looked at). target_probs
    (tokens, vocab) float32: the target's probabilities behind each token. uniform (tokens,) float32 in [0, 1): a random
    number for each token's acceptance, the root's for the draw of the next token. draft_probs: like target_probs, the
    distribution that the drafts behind each token were drawn from, each by itself; None for drafts that are no samples
    (the most likely ones, a lookup's).

    path (B, max_new) int32: the accepted tokens of each sequence, root first, as indices among its new tokens, then -1;
    accepted (B,) int32: how many, the root among them; next (B,) int64: the token behind the last one accepted. From
    the root on, the drafts behind the current token are tried in order. p, q: the current token's rows, t the
    draft's token, u its number. With draft_probs it is accepted iff u q(t) S(c) < max(p(t) - c q(t), 0): c = 0 and
    S(0) = 1 at first, and each rejection adds S(c) = sum(max(p - c q, 0)) to c. Without, iff u m < p(t): m = 1 at first, and
    each rejection takes p(t) from m, t counting as 0 from then on. next is the first token whose sum of weights up to
    it exceeds u S, with u the root's number, S the sum of the weights: max(p - c q, 0), or p without the rejected
    tokens; p if they are all 0; -1 if p is too, or for a sequence without tokens (accepted 0). Elements that are not
    positive finite numbers are 0, a draft whose token is not in the vocabulary is none. Sums and comparisons are in 64 bits.
    max_new: the most new tokens of a sequence (default: all tokens, up to 1024)."""
    name = "verify_draft"
    shape, device, offsets = parents.shape, parents.device, cu_seqlens.shape
    if (len(offsets) == 1 and offsets[0] > 1 and len(target_probs.shape) == 2
            and _checks.trees_ok(parents, ((tokens, torch.int64, shape), (uniform, torch.float32, shape), (cu_seqlens, torch.int32, offsets)), max_new)
            and all(x is None or _checks.probs_ok(x, shape[0], device, target_probs.shape[1]) for x in (target_probs, draft_probs))):
        most = max_new
    else:
        _checks.check_vector(name, "cu_seqlens", cu_seqlens, torch.int32, None, device)
        most = _checks.check_tree(name, parents, offsets[0] - 1, cu_seqlens, max_new)
        _checks.check_vector(name, "tokens", tokens, torch.int64, shape[0], device)
        _checks.check_vector(name, "uniform", uniform, torch.float32, shape[0], device)
        _checks.check_probs(name, "target_probs", target_probs, shape[0], device)
        if draft_probs is not None:
            _checks.check_probs(name, "draft_probs", draft_probs, shape[0], device, target_probs.shape[1])
    n, seqs, vocab = shape[0], offsets[0] - 1, target_probs.shape[1]
    path = torch.empty((seqs, most), dtype=torch.int32, device=device)
    accepted = torch.empty(seqs, dtype=torch.int32, device=device)
    drawn = torch.empty(seqs, dtype=torch.int64, device=device)
    need = _native.lib().pa_verify_draft_workspace(seqs, vocab, 0 if draft_probs is None else 1)
    if need < 0:
        _native.check(need, name)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _call("pa_verify_draft", name, device, tokens.data_ptr(), parents.data_ptr(), target_probs.data_ptr(),
          target_probs.stride(0), None if draft_probs is None else draft_probs.data_ptr(),
          0 if draft_probs is None else draft_probs.stride(0), uniform.data_ptr(), cu_seqlens.data_ptr(), n, seqs, vocab,
          most, path.data_ptr(), accepted.data_ptr(), drawn.data_ptr(), None if workspace is None else workspace.data_ptr(),
          need, _stream_ptr(device))
    return path, accepted, drawn


def cache_keep(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
               path: torch.Tensor, accepted: torch.Tensor, cu_seqlens: torch.Tensor, *,
               k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Leave of a step's new tokens the accepted ones in the cache, in place; returns the lengths after that, (B,) int32.

    The row of sequence s's new token path[s, j] becomes that of its new token j, for j below accepted[s] (verify_draft's
    results: paths ascend); keys, values and, in 8 bits, their codes and scales as they are. An entry that is no new
    token of the sequence leaves its row as it is. The new length is lengths - count + accepted. lengths itself stays as it is:
    every layer's call takes the same, and the result is the next step's."""
    name = "cache_keep"
    _check(name, None, k_cache, v_cache, page_table, lengths, None, k_scale, v_scale)
    seqs, device = lengths.shape[0], k_cache.device
    _checks.check_vector(name, "cu_seqlens", cu_seqlens, torch.int32, seqs + 1, device)
    _checks.check_vector(name, "accepted", accepted, torch.int32, seqs, device)
    _checks.check_path(name, path, seqs, device)
    after = torch.empty_like(lengths)
    cache = _cache_args(k_cache, v_cache, page_table, lengths, k_scale, v_scale)
    _call("pa_cache_keep", name, device, cache, path.data_ptr(), path.shape[1], path.stride(0), accepted.data_ptr(),
          cu_seqlens.data_ptr(), after.data_ptr(), _stream_ptr(device))
    return after
