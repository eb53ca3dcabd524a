"""paged_attn: an infinite value that a row sees is infinite in the row, however small the key's weight is."""
import math
import os
import sys

import pytest
import torch

import cuda_attn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731
SEQS = {"few": [(3, 200)], "few long": [(4, 3000)], "chunk": [(100, 400)], "chunk2": [(70, 200), (90, 500)], "long chunk": [(300, 2500)],
        "prompt": [(200, 200)]}


def low_key(p, s, pos, score):
    """Position pos gives every row of sequence s that score; its value is finite as it was."""
    pg, rw = po.slot(p, s, pos)
    p.k_cache[pg, :, rw] = 0
    p.k_cache[pg, :, rw, 0] = score * math.sqrt(p.q.shape[2]) / 8.0
    return pg, rw


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_infinite_values_of_small_weight(kind, dtype, d, causal):
    """A weight of e^-40 or so of two keys, early and late, in dims of their own and in one that they share."""
    p = po.make(SEQS[kind], d=d, hq=4, hkv=2, dtype=dtype)
    p.q[..., 0] = 8.0
    first = 0
    expect = {}
    for s, (count, length) in enumerate(SEQS[kind]):
        for pos in (5, length - count // 2 - 1):
            pg, rw = low_key(p, s, pos, -40.0)
            p.v_cache[pg, :, rw, 3 if pos == 5 else 9] = math.inf
            p.v_cache[pg, :, rw, 20] = math.inf if pos == 5 else -math.inf
            p.v_cache[pg, 0, rw, 21] = -math.inf
        expect[s] = first, count, length
        first += count
    ref, bound, _ = po.attn(p, causal)
    g = p.to("cuda")
    got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu, causal=causal).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), (int(torch.isnan(got).sum()), int(torch.isnan(ref).sum()))
    inf = torch.isinf(ref)
    assert bool(inf.any()) and torch.equal(got[inf], ref[inf]) and not bool(torch.isinf(got[~inf]).any())
    fine = torch.isfinite(ref)
    assert bool(((got - ref).abs() <= bound)[fine].all())
    for s, (first, count, length) in expect.items():   # by the definition, apart from the oracle's arithmetic
        sees = torch.arange(length - count, length) >= 5 if causal else torch.ones(count, dtype=torch.bool)
        assert bool((got[first:first + count, :, 3][sees] == math.inf).all())
        assert bool(torch.isnan(got[first + count - 1, :, 20]).all())


@pytest.mark.parametrize("kind", ["chunk", "long chunk"])
def test_a_nan_value_of_small_weight(kind):
    """A NaN value stays one, beside an infinite one in another dim."""
    p = po.make(SEQS[kind], d=64, hq=2, hkv=1, dtype=F16)
    p.q[..., 0] = 8.0
    pg, rw = low_key(p, 0, 70, -40.0)
    p.v_cache[pg, :, rw, 11], p.v_cache[pg, :, rw, 12] = math.nan, -math.inf
    g = p.to("cuda")
    got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu).cpu()
    assert bool(torch.isnan(got[..., 11]).all()) and bool((got[..., 12] == -math.inf).all())
    got[..., 11:13] = 0
    assert bool(torch.isfinite(got).all())
