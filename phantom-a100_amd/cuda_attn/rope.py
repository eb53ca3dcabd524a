"""Rotary positions of queries and keys.

    freqs, scale = cuda_attn.rope_frequencies(128, 500000.0, device="cuda")
    q, k = cuda_attn.rope(q, k, positions, freqs, scale=scale)
"""
from __future__ import annotations

import math
import struct

import torch
from torch.autograd.graph import increment_version

from . import _call, _checks, _native, _stream_ptr

_DTYPE_CODE = {torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}


def rope_frequencies(dim: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                     original: int = 4096, low: float = 1.0, high: float = 32.0,
                     device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """(freqs, scale) for rope: the angle per position of each of dim / 2 pairs, float64, and the factor of the result.

    base ** (-2 p / dim) for pair p; for contexts `factor` times as long as the `original` ones that a model was trained
    on, by `scaling`:
      None       as they are
      "linear"   divided by factor: positions interpolated (published as position interpolation)
      "ntk"      base times factor ** (dim / (dim - 2)): the slowest pair interpolated, the fastest as it is (NTK-aware)
      "smooth"   by the turns r = original f / (2 pi) that a pair makes in an original context: divided by factor below
                 `low` turns, as they are above `high`, between them f ((1 - w) / factor + w), w = (r - low) / (high - low)
      "parts"    interpolated linearly in the pair's number instead, between the numbers (rounded outwards) of the pairs that
                 make `high` and `low` turns, and the result times 0.1 ln(factor) + 1 (YaRN)"""
    if isinstance(dim, bool) or not isinstance(dim, int) or dim < 2 or dim % 2:
        raise RuntimeError("rope_frequencies: dim must be a positive even number")
    if scaling not in (None, "linear", "ntk", "smooth", "parts"):
        raise RuntimeError("rope_frequencies: scaling must be None, 'linear', 'ntk', 'smooth' or 'parts'")
    if not base > 0 or not factor >= 1.0 or not original >= 1 or scaling in ("smooth", "parts") and not 0 < low < high:
        raise RuntimeError("rope_frequencies: base, factor (from 1 on), original and 0 < low < high must be numbers")
    if scaling == "parts" and not (base > 1 and all(math.isfinite(x) for x in (base, factor, original, high))):
        raise RuntimeError("rope_frequencies: 'parts' takes a base above 1 (pairs that turn ever slower) and finite numbers")
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    pair = torch.arange(dim // 2, dtype=torch.float64)
    freqs = torch.as_tensor(base, dtype=torch.float64) ** (-2.0 * pair / dim)
    scale = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "smooth":
        w = ((original * freqs / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        freqs = freqs * ((1 - w) / factor + w)
    elif scaling == "parts":
        number = lambda turns: dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(number(high)), 0), min(math.ceil(number(low)), dim - 1)
        w = 1 - ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
        freqs = freqs * ((1 - w) / factor + w)
        scale = 0.1 * math.log(factor) + 1.0
    return freqs.to(device), scale


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, *,
         interleaved: bool = False, scale: float = 1.0, inverse: bool = False,
         inplace: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Queries and keys turned to their positions: (q, k) in new tensors, or themselves (inplace).

    q and k (None: none) are (tokens, heads, d) with positions (tokens,), or (B, heads, N, d) with positions (N,) or (B, N),
    int32 or int64; views with any strides, each row's d elements contiguous; float32, float16 or bfloat16, d up to 1024.
    freqs (r / 2,) float64, r <= d: pair p of a row's first r elements is turned by the angle position * freqs[p],
    (x, y) -> scale * (x cos - y sin, x sin + y cos); the d - r others pass as they are. Pairs are the elements p and
    p + r / 2, or 2 p and 2 p + 1 (interleaved). inverse: by the negative angle: applied to the gradients of the results,
    with the same scale, it gives those of q and k. There is no autograd function: results are cut from its graph, and tensors
    that require a gradient are refused in place while it records. Angles are computed in 64 bits (right at any 32-bit
    position), the turn in 32."""
    if inplace or not _checks.rope_ok(q, k, positions, freqs):
        _checks.check_rope("rope", q, k, positions, freqs, inplace)
    shape, device = q.shape, q.device
    dense = len(shape) == 4
    q_out, rows = _rows(q, dense, inplace)
    k_out, k_rows = (None, None) if k is None else _rows(k, dense, inplace)
    ps = positions.stride()
    pb, pn = ps if len(ps) == 2 else (0, ps[0])
    b, n = (shape[0], shape[2]) if dense else (1, shape[0])
    _call("pa_rope", "rope", device, rows, k_rows, _DTYPE_CODE[q.dtype], b, n, shape[-1], positions.data_ptr(),
          1 if positions.dtype is torch.int64 else 0, pb, pn, freqs.data_ptr(), freqs.shape[0], 1 if interleaved else 0,
          1 if inverse else 0, scale, _stream_ptr(device))
    if inplace:   # what autograd has saved of them is no longer what it was
        increment_version(q if k is None else (q, k))
    return q_out, k_out


_pack = struct.Struct("PP7q").pack   # pa_rope_rows


def _rows(x, dense, inplace):
    """Where x's rows go, and the rows as the library takes them."""
    shape = x.shape
    y = x if inplace else torch.empty(shape, dtype=x.dtype, device=x.device)
    if dense:
        xb, xh, xn, _ = x.stride()
        yb, yh, yn, _ = y.stride()
        return y, _pack(x.data_ptr(), y.data_ptr(), xb, xn, xh, yb, yn, yh, shape[1])
    xn, xh, _ = x.stride()
    yn, yh, _ = y.stride()
    return y, _pack(x.data_ptr(), y.data_ptr(), 0, xn, xh, 0, yn, yh, shape[1])
