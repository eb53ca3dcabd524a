"""Argument checks of the attention entry points, run in Python before the native call.

Same checks, order and message substrings as the reference's C++ glue, so callers (and the
reference's tests, which match on "contiguous", "dtype", "head dimension", "float16",
"not compiled" and "shared memory") see the same errors:
  check_inputs        /root/reference/csrc/bindings.cpp:12-22
  float/half dispatch /root/reference/csrc/common.cuh:14-19
  fp16 / d=64 / align /root/reference/csrc/common.cuh:27-33
  tile set and LDS    /root/reference/csrc/attn_fused_tuned.cu:8-14, attn_fused_tc.cu:11-13
Deliberate extensions: fused_tc also takes bfloat16 and d = 128; every fused entry takes an
optional fp32 output dtype.
"""
from __future__ import annotations

import torch

TUNED_CONFIGS = ((64, 32), (64, 64), (128, 32), (128, 64))  # /root/reference/csrc/kernels/fused_tuned.cuh:207
TC_HEAD_DIMS = (64, 128)
TC_DTYPES = (torch.float16, torch.bfloat16)


def _fail(msg: str):
    raise RuntimeError(msg)


def check_inputs(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, require_cuda: bool = True) -> None:
    """Checks shared by every entry point (csrc/bindings.cpp:12-22)."""
    # Valid inputs pass on each property read once; anything else goes through the checks one by one for
    # its message. A small call is bound by this host path: with properties read once here and in the
    # entry points, fused_tc fp16 42x128 d=64 9.6 -> 7.7 us a call, fused fp32 8.2 -> 7.4.
    shape, dtype, device = q.shape, q.dtype, q.device
    if (len(shape) == 4 and (q.is_cuda or not require_cuda) and q.is_contiguous() and k.is_contiguous()
            and v.is_contiguous() and k.dtype is dtype and v.dtype is dtype and k.shape == shape and v.shape == shape
            and k.device == device and v.device == device and 0 not in shape):
        return
    for t in (q, k, v):
        if require_cuda and not t.is_cuda:
            _fail("inputs must be CUDA tensors")
        if not t.is_contiguous():
            _fail("inputs must be contiguous")
        if t.dim() != 4:
            _fail("inputs must be shaped (B, H, N, d)")
        if t.dtype != q.dtype:
            _fail("q, k, v must share a dtype")
    if q.shape != k.shape or q.shape != v.shape:
        _fail("q, k, v must have the same shape")
    if q.device != k.device or q.device != v.device:
        _fail("q, k, v must be on the same device")
    if q.numel() == 0:
        _fail("inputs must be non-empty")


def check_float_half(name: str, q: torch.Tensor) -> None:
    if q.dtype not in (torch.float32, torch.float16):
        _fail(f"{name}: only float32 and float16 are supported")


def check_head_dim(name: str, q: torch.Tensor, allowed=(64,)) -> None:
    d = q.shape[3]
    if d not in allowed:
        if len(allowed) == 1:
            _fail(f"{name}: only head dimension {allowed[0]} is compiled (got {d})")
        dims = " and ".join(str(a) for a in allowed)
        _fail(f"{name}: only head dimensions {dims} are compiled (got {d})")


def check_aligned(name: str, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.data_ptr() % 16 != 0:
            _fail(f"{name}: inputs must be 16-byte aligned")


def check_fp16_d64_aligned(name: str, q, k, v) -> None:
    """The reference's fp16-only / d=64 / 16-byte check (csrc/common.cuh:27-33)."""
    if q.dtype != torch.float16:
        _fail(f"{name}: float16 only")
    check_head_dim(name, q, (64,))
    check_aligned(name, q, k, v)


def check_tc(q, k, v) -> None:
    """fused_tc: fp16 or bf16, d in {64, 128}, 16-byte aligned (extends csrc/common.cuh:27-33)."""
    if q.dtype not in TC_DTYPES:
        _fail("fused_tc: float16 or bfloat16 only")
    check_head_dim("fused_tc", q, TC_HEAD_DIMS)
    check_aligned("fused_tc", q, k, v)


def check_tuned_config(br: int, bc: int) -> None:
    if (int(br), int(bc)) not in TUNED_CONFIGS:
        _fail(f"fused_tuned: (br, bc) = ({br}, {bc}) not compiled; available: (64,32) (64,64) (128,32) (128,64)")


def resolve_out_dtype(name: str, q: torch.Tensor, out_dtype) -> torch.dtype:
    """Output dtype: the input dtype by default (as in the reference) or float32 on request."""
    if out_dtype is None or out_dtype == q.dtype:
        return q.dtype
    if out_dtype == torch.float32:
        return torch.float32
    _fail(f"{name}: out_dtype must be the input dtype or torch.float32 (got {out_dtype})")


def check_lds(name: str, need: int, limit: int, detail: str = "") -> None:
    """Per-workgroup LDS against the device limit (reference wording: 'shared memory')."""
    if need < 0:
        _fail(f"{name}: configuration not compiled")
    if need > limit:
        if detail:
            _fail(f"{name}: {detail} needs {need} bytes of shared memory; this GPU allows {limit}")
        _fail(f"{name}: needs {need} bytes of shared memory, GPU allows {limit}")


# ---------------------------------------------------------------- the paged cache (paged.py)
EIGHT_BIT = (torch.int8, torch.float8_e4m3fn)


def check_paged(name: str, rows, k_cache, v_cache, page_table, lengths, k_scale, v_scale, *,
                require_cuda: bool = True) -> None:
    """The cache's own tensors; `rows` is a tensor of the call's new tokens (None for cache_read)."""
    device, dtype = k_cache.device, k_cache.dtype
    tensors = [k_cache, v_cache, page_table, lengths] + [t for t in (rows, k_scale, v_scale) if t is not None]
    for t in tensors:
        if require_cuda and not t.is_cuda:
            _fail(f"{name}: inputs must be CUDA tensors")
        if t.device != device:
            _fail(f"{name}: inputs must be on the same device")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        _fail(f"{name}: k_cache and v_cache must be shaped (pages, heads, page_size, d), both alike")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous():
        _fail(f"{name}: k_cache and v_cache must be contiguous")
    if dtype != v_cache.dtype:
        _fail(f"{name}: k_cache and v_cache must share a dtype")
    if dtype not in TC_DTYPES and dtype not in EIGHT_BIT:
        _fail(f"{name}: the cache's dtype must be float16, bfloat16, int8 or float8_e4m3fn")
    if rows is not None:
        if rows.dtype not in TC_DTYPES:
            _fail(f"{name}: float16 or bfloat16 only")
        if dtype != rows.dtype and dtype not in EIGHT_BIT:
            _fail(f"{name}: the cache's dtype must be the inputs' or an 8-bit one")
    check_head_dim(name, k_cache, TC_HEAD_DIMS)
    if k_cache.numel() == 0 or page_table.numel() == 0:
        _fail(f"{name}: inputs must be non-empty")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.stride(1) != 1 and page_table.shape[1] > 1:
        _fail(f"{name}: page_table must be a (B, columns) int32 tensor with contiguous rows")
    if lengths.shape != page_table.shape[:1] or lengths.dtype != torch.int32 or not lengths.is_contiguous():
        _fail(f"{name}: lengths must be a contiguous (B,) int32 tensor")
    check_aligned(name, k_cache, v_cache)
    if dtype in EIGHT_BIT:
        for s in (k_scale, v_scale):
            if s is None or s.shape != k_cache.shape[:3] or s.dtype != torch.float32 or not s.is_contiguous():
                _fail(f"{name}: an 8-bit cache needs k_scale and v_scale, contiguous (pages, heads, page_size) float32")
    elif k_scale is not None or v_scale is not None:
        _fail(f"{name}: k_scale and v_scale are for 8-bit caches")


def paged_ok(rows, k_cache, v_cache, page_table, lengths, cu_seqlens, k_scale, v_scale) -> bool:
    """Whether a call passes check_paged and check_rows, each property read once: a small call is bound by this
    host path. Anything that this does not accept goes through those checks for its message."""
    shape, dtype, device = k_cache.shape, k_cache.dtype, k_cache.device
    table = page_table.shape
    if not (len(shape) == 4 and shape[3] in TC_HEAD_DIMS and k_cache.is_cuda and k_cache.is_contiguous()
            and v_cache.shape == shape and v_cache.dtype is dtype and v_cache.device == device and v_cache.is_contiguous()
            and 0 not in shape and len(table) == 2 and 0 not in table and page_table.dtype is torch.int32
            and page_table.stride(1) == 1 and page_table.device == device and lengths.dtype is torch.int32
            and lengths.shape == table[:1] and lengths.device == device and lengths.is_contiguous()
            and (k_cache.data_ptr() | v_cache.data_ptr()) % 16 == 0):
        return False
    if dtype in EIGHT_BIT:
        for s in (k_scale, v_scale):
            if not (s is not None and s.shape == shape[:3] and s.dtype is torch.float32 and s.device == device and s.is_contiguous()):
                return False
    elif k_scale is not None or v_scale is not None:
        return False
    if rows is None:
        return dtype in TC_DTYPES or dtype in EIGHT_BIT
    x, strides = rows.shape, rows.stride()
    if not (len(x) == 3 and x[2] == shape[3] and 0 not in x and strides[2] == 1 and (strides[0] | strides[1]) % 8 == 0
            and rows.device == device and rows.data_ptr() % 16 == 0 and rows.dtype in TC_DTYPES
            and (dtype is rows.dtype or dtype in EIGHT_BIT)):
        return False
    if cu_seqlens is None:
        return x[0] % table[0] == 0
    return (cu_seqlens.dtype is torch.int32 and cu_seqlens.shape == (table[0] + 1,) and cu_seqlens.device == device
            and cu_seqlens.is_contiguous())


def check_rows(name: str, x, k_cache, lengths, cu_seqlens) -> None:
    """A tensor of new tokens, (tokens, heads, d)."""
    if x.dim() != 3 or x.shape[2] != k_cache.shape[3]:
        _fail(f"{name}: the new tokens' tensors must be shaped (tokens, heads, d) with the cache's d")
    if x.numel() == 0:
        _fail(f"{name}: inputs must be non-empty")
    if x.stride(2) != 1 or x.stride(0) % 8 or x.stride(1) % 8:
        _fail(f"{name}: rows must be contiguous, at strides of whole 16-byte steps")
    check_aligned(name, x)
    if cu_seqlens is None:
        if x.shape[0] % lengths.shape[0]:
            _fail(f"{name}: without cu_seqlens the tokens must divide evenly over the sequences")
    elif (cu_seqlens.shape != (lengths.shape[0] + 1,) or cu_seqlens.dtype != torch.int32
          or not cu_seqlens.is_contiguous() or cu_seqlens.device != k_cache.device):
        _fail(f"{name}: cu_seqlens must be a contiguous (B + 1,) int32 tensor on the inputs' device")


def check_same_rows(name: str, k, v, k_cache) -> None:
    """v against k, which has been checked."""
    if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.shape[1] != k_cache.shape[1]:
        _fail(f"{name}: k and v must share shape, dtype and device and have the cache's heads")
    strides = v.stride()
    if strides[2] != 1 or strides[0] % 8 or strides[1] % 8:
        _fail(f"{name}: rows must be contiguous, at strides of whole 16-byte steps")
    check_aligned(name, v)


def check_query_heads(name: str, q, k_cache) -> None:
    if q.shape[1] % k_cache.shape[1]:
        _fail(f"{name}: the query heads must be a multiple of the cache's heads")


def _span(t) -> tuple[int, int]:
    """The bytes from a tensor's first element to past its last one."""
    size = t.element_size()
    return t.data_ptr(), t.data_ptr() + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _apart(a, b) -> bool:
    """Whether no row of a, (tokens, heads, d), shares memory with one of b, of a's shape. Rows of one may lie between
    those of the other where both have the same strides (slices of one buffer); of unlike strides, a and b must lie
    apart altogether."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    axes = sorted((n, s, t) for n, s, t in zip(a.shape[:2], a.stride(), b.stride()) if n > 1)
    if any(s != t for _, s, t in axes):
        return False
    # Rows differ by delta + i s0 + j s1 elements, |i| < n0, |j| < n1: for each i the j nearest to none, on either side.
    delta, d = (b0 - a0) // a.element_size(), a.shape[2]
    (n0, s0), (n1, s1) = ([(1, 0), (1, 0)] + [(n, s) for n, s, _ in axes])[-2:]
    for i in range(1 - n0, n0):
        at = delta + i * s0
        j = max(1 - n1, min(n1 - 1, -at // s1)) if s1 else 0
        if abs(at + j * s1) < d or j < n1 - 1 and abs(at + (j + 1) * s1) < d:
            return False
    return True


def check_out(name: str, q, out, *others) -> None:
    """out, where a call with queries q writes; `others` are the tensors that it reads beside q (None: none)."""
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        _fail(f"{name}: out must have q's shape, dtype and device")
    if out.stride(2) != 1 or out.stride(0) % 8 or out.stride(1) % 8:
        _fail(f"{name}: rows must be contiguous, at strides of whole 16-byte steps")
    check_aligned(name, out)
    (tokens, heads, d), (ts, hs, _) = out.shape, out.stride()
    by_token = (heads == 1 or hs >= d) and (tokens == 1 or ts >= (heads - 1) * hs + d)
    by_head = (tokens == 1 or ts >= d) and (heads == 1 or hs >= (tokens - 1) * ts + d)
    if not by_token and not by_head:
        _fail(f"{name}: out's rows must not overlap")
    if not _apart(q, out):
        _fail(f"{name}: out must not share memory with q")
    o0, o1 = _span(out)
    for t in others:
        if t is not None and t.data_ptr() < o1 and _span(t)[1] > o0:
            _fail(f"{name}: out must not share memory with the cache, its scales, the page table, the lengths or the offsets")


def check_max_new(name: str, max_new) -> int:
    if isinstance(max_new, bool) or not isinstance(max_new, int) or max_new < 1:
        _fail(f"{name}: max_new must be a positive number of tokens")
    return min(max_new, 2 ** 30)


def check_max_len(name: str, n) -> None:
    if isinstance(n, bool) or not isinstance(n, int) or n < 1 or n > 2 ** 30:
        _fail(f"{name}: max_len must be a number of tokens from 1 to 2^30")


def read_dtype(name: str, k_cache, dtype) -> torch.dtype:
    """The dtype of the rows read back: the cache's own 16-bit one, or the caller's choice for an 8-bit cache."""
    if k_cache.dtype in EIGHT_BIT:
        if dtype not in TC_DTYPES:
            _fail(f"{name}: dtype must be float16 or bfloat16 for an 8-bit cache")
        return dtype
    if dtype is not None and dtype != k_cache.dtype:
        _fail(f"{name}: dtype must be the cache's own ({k_cache.dtype})")
    return k_cache.dtype


# ---------------------------------------------------------------- drafted tokens (draft.py) and rotary positions (rope.py)
TREE_MAX = 1024


def check_vector(name: str, what: str, x, dtype, size, device, *, require_cuda: bool = True) -> None:
    """A contiguous vector of `size` elements (None: any number of at least one) beside the others of a call."""
    if (x.dtype is dtype and x.dim() == 1 and (x.shape[0] == size or size is None and x.shape[0] > 0)
            and x.is_contiguous() and x.device == device and (x.is_cuda or not require_cuda)):
        return
    if require_cuda and not x.is_cuda:
        _fail(f"{name}: inputs must be CUDA tensors")
    if x.device != device:
        _fail(f"{name}: inputs must be on the same device")
    if x.numel() == 0:
        _fail(f"{name}: inputs must be non-empty")
    shape = "" if size is None else f" of {size} elements"
    _fail(f"{name}: {what} must be a contiguous {str(dtype).replace('torch.', '')} vector{shape}")


def check_tree(name: str, parents, seqs: int, cu_seqlens, max_new, *, require_cuda: bool = True) -> int:
    """The new tokens of a call and their trees; the most tokens of a tree."""
    check_vector(name, "parents", parents, torch.int32, None, parents.device, require_cuda=require_cuda)
    tokens = parents.shape[0]
    if seqs < 1:
        _fail(f"{name}: inputs must be non-empty")
    if cu_seqlens is None:
        if tokens % seqs:
            _fail(f"{name}: without cu_seqlens the tokens must divide evenly over the sequences")
    else:
        check_vector(name, "cu_seqlens", cu_seqlens, torch.int32, seqs + 1, parents.device, require_cuda=require_cuda)
    if max_new is None:
        most = tokens // seqs if cu_seqlens is None else tokens
        if cu_seqlens is None and most > TREE_MAX:
            _fail(f"{name}: a tree has at most {TREE_MAX} tokens")
        return min(most, TREE_MAX)
    if isinstance(max_new, bool) or not isinstance(max_new, int) or not 1 <= max_new <= TREE_MAX:
        _fail(f"{name}: max_new must be a number of tokens from 1 to {TREE_MAX}")
    return max_new


def trees_ok(parents, vectors, max_new) -> bool:
    """Whether new tokens and (tensor, dtype, size) vectors beside them pass check_tree and check_vector, each property read
    once: a small call is bound by this host path. Anything that this does not accept goes through those checks for its message."""
    shape, device = parents.shape, parents.device
    if not (len(shape) == 1 and shape[0] > 0 and parents.dtype is torch.int32 and parents.is_cuda and parents.is_contiguous()
            and type(max_new) is int and 1 <= max_new <= TREE_MAX):
        return False
    for x, dtype, size in vectors:
        if not (x.dtype is dtype and x.shape == size and 0 not in size and x.device == device and x.is_contiguous()):
            return False
    return True


def probs_ok(x, tokens, device, vocab) -> bool:
    """As above, for check_probs."""
    return (len(x.shape) == 2 and x.shape == (tokens, vocab) and vocab > 0 and x.dtype is torch.float32
            and (x.stride(1) == 1 or vocab == 1) and x.device == device)


def check_mask(name: str, mask, q) -> None:
    """A mask of the new tokens of q."""
    if mask.device != q.device:
        _fail(f"{name}: inputs must be on the same device")
    if (mask.dim() != 2 or mask.dtype is not torch.int32 or mask.shape[0] != q.shape[0] or mask.shape[1] < 1
            or mask.stride(1) != 1 and mask.shape[1] > 1):
        _fail(f"{name}: mask must be a (tokens, words) int32 tensor with contiguous rows")


def check_no_overlap(name: str, out, x, what: str) -> None:
    (o0, o1), (x0, x1) = _span(out), _span(x)
    if x0 < o1 and o0 < x1:
        _fail(f"{name}: out must not share memory with {what}")


def check_probs(name: str, what: str, x, tokens: int, device, vocab=None, *, require_cuda: bool = True) -> None:
    if require_cuda and not x.is_cuda:
        _fail(f"{name}: inputs must be CUDA tensors")
    if x.device != device:
        _fail(f"{name}: inputs must be on the same device")
    if x.dim() != 2 or x.shape[0] != tokens or x.dtype is not torch.float32 or x.stride(1) != 1 and x.shape[1] > 1:
        _fail(f"{name}: {what} must be a (tokens, vocab) float32 tensor with contiguous rows")
    if x.shape[1] < 1:
        _fail(f"{name}: inputs must be non-empty")
    if vocab is not None and x.shape[1] != vocab:
        _fail(f"{name}: target_probs and draft_probs must be of one vocabulary")


def check_path(name: str, path, seqs: int, device) -> None:
    if path.device != device:
        _fail(f"{name}: inputs must be on the same device")
    if (path.dim() != 2 or path.shape[0] != seqs or path.shape[1] < 1 or path.dtype is not torch.int32
            or path.stride(1) != 1 and path.shape[1] > 1):
        _fail(f"{name}: path must be a (B, columns) int32 tensor with contiguous rows")


ROPE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
ROPE_MAX_DIM = 1024


def _rows_overlap(x) -> bool:
    """Whether elements of a tensor may share memory: its axes, by their strides, must each step past all inner ones."""
    end = 1
    for stride, size in sorted((s, n) for n, s in zip(x.shape, x.stride()) if n > 1):
        if stride < end:
            return True
        end = stride * (size - 1) + end
    return False


def _tokens_apart(q, k, token: int) -> bool:
    """Whether q and k, of the same tokens, share no memory: they lie apart, or each token's rows of the one beside those of
    the other within one stride of the tokens (slices of one projection)."""
    (q0, q1), (k0, k1) = _span(q), _span(k)
    if q1 <= k0 or k1 <= q0:
        return True
    step = q.stride(token)
    others = [s for x in (q, k) for i, (n, s) in enumerate(zip(x.shape, x.stride())) if i not in (1, token, x.dim() - 1) and n > 1]
    if k.stride(token) != step or step < 1 or any(s % step for s in others):
        return False
    size = q.element_size()
    if (k0 - q0) % size:
        return False
    wide = [(x.shape[1] - 1) * x.stride(1) + x.shape[-1] for x in (q, k)]
    at = (k0 - q0) // size % step
    return at >= wide[0] and at + wide[1] <= step


def rope_ok(q, k, positions, freqs) -> bool:
    """Whether a call into new tensors passes check_rope, each property read once: a small call is bound by this host path.
    Anything that this does not accept goes through that check for its message."""
    shape, dtype, device, at = q.shape, q.dtype, q.device, positions.shape
    axes = len(shape)
    if not ((axes == 3 and at == shape[:1] or axes == 4 and at in ((shape[2],), (shape[0], shape[2]))) and q.is_cuda
            and dtype in ROPE_DTYPES and 0 not in shape and shape[-1] <= ROPE_MAX_DIM and q.stride(-1) == 1
            and positions.dtype in (torch.int32, torch.int64) and positions.device == device and freqs.device == device
            and freqs.dtype is torch.float64 and freqs.dim() == 1 and freqs.is_contiguous() and 1 <= freqs.shape[0] <= shape[-1] // 2):
        return False
    if k is None:
        return True
    other = k.shape
    return (k.dtype is dtype and k.device == device and len(other) == axes and 0 not in other and other[0] == shape[0]
            and other[2:] == shape[2:] and k.stride(-1) == 1)


def check_rope(name: str, q, k, positions, freqs, inplace: bool, *, require_cuda: bool = True) -> None:
    device, dtype, shape = q.device, q.dtype, q.shape
    for t in (q, k, positions, freqs):
        if t is None:
            continue
        if require_cuda and not t.is_cuda:
            _fail(f"{name}: inputs must be CUDA tensors")
        if t.device != device:
            _fail(f"{name}: inputs must be on the same device")
    if len(shape) not in (3, 4):
        _fail(f"{name}: q and k must be shaped (tokens, heads, d) or (B, heads, N, d)")
    if dtype not in ROPE_DTYPES:
        _fail(f"{name}: float32, float16 or bfloat16 only")
    if 0 in shape or k is not None and 0 in k.shape:
        _fail(f"{name}: inputs must be non-empty")
    if k is not None:
        if k.dtype is not dtype:
            _fail(f"{name}: q and k must share a dtype")
        if k.dim() != len(shape) or k.shape[0] != shape[0] or k.shape[2:] != shape[2:]:
            _fail(f"{name}: q and k must have the same tokens and head dimension")
    if shape[-1] > ROPE_MAX_DIM:
        _fail(f"{name}: head dimensions up to {ROPE_MAX_DIM}")
    for x in (q, k):
        if x is not None and x.stride(-1) != 1 and shape[-1] > 1:
            _fail(f"{name}: rows must be contiguous")
    if positions.dtype not in (torch.int32, torch.int64):
        _fail(f"{name}: positions must be int32 or int64")
    if len(shape) == 3:
        fits = positions.shape == shape[:1]
    else:
        fits = positions.shape == (shape[2],) or positions.shape == (shape[0], shape[2])
    if not fits:
        _fail(f"{name}: positions must be (tokens,), or (N,) or (B, N) for (B, heads, N, d)")
    if freqs.dim() != 1 or freqs.dtype is not torch.float64 or not freqs.is_contiguous() or not 1 <= freqs.shape[0] <= shape[-1] // 2:
        _fail(f"{name}: freqs must be a contiguous float64 vector of 1 to d / 2 elements")
    if inplace:
        if torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad):
            _fail(f"{name}: tensors that require a gradient are not turned in place")
        for x in (q, k):
            if x is not None and _rows_overlap(x):
                _fail(f"{name}: rows that are written must not overlap")
        if k is not None and not _tokens_apart(q, k, 0 if len(shape) == 3 else 2):
            _fail(f"{name}: q and k must not share memory")
