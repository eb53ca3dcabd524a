"""Offsets of new tokens that are out of order or out of range: which rows cache_write and paged_attn take for whose."""
import os
import sys

import pytest
import torch

import cuda_attn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu

F16, BF16, I8 = torch.float16, torch.bfloat16, torch.int8
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def written_once(p):
    """The caches after cache_write where a row of two sequences is written for the first of them."""
    seen, q = set(), po.Problem(**vars(p))
    kc, vc, scales = p.k_cache.clone(), p.v_cache.clone(), {n: t.clone() for n, t in p.scales.items()}
    for s, (first, count, length) in enumerate(po.layout(p, p.k.shape[0])):
        for i in range(count):
            at = po.slot(p, s, length - count + i)
            if first + i in seen or at is None:
                seen.add(first + i)
                continue
            seen.add(first + i)
            for x, c, name in ((q.k, kc, "k_scale"), (q.v, vc, "v_scale")):
                row = x[first + i]
                if scales:
                    row, scale = po.quantise(row, c.dtype)
                    scales[name][at[0], :, at[1]] = scale
                c[at[0], :, at[1]] = row
    return kc, vc, scales


@pytest.mark.parametrize("cu", [[0, 5, 3], [0, 9, 4, 4], [4, 9, 2, 9], [-3, 4, 1, 99], [3, 0, 6], [9, 9, 0], [0, 2, 9, 5, 5], [2, 2, 2, 7],
                                [0] + [9] * 70 + [3] * 70, [5] * 66 + [0] * 66 + [9] * 3])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, I8)], ids=IDS)
def test_rows_of_offsets_in_any_order(cu, dtype, cache):
    seqs = len(cu) - 1
    p = po.make([(0, 20)] * seqs, hq=2, hkv=1, d=64, page=16, dtype=dtype, cache=cache, stale=0.0)
    g = torch.Generator().manual_seed(1)
    p.q, p.k, p.v = (torch.randn(9, h, 64, generator=g).to(dtype) for h in (2, 1, 1))
    p.cu = torch.tensor(cu, dtype=torch.int32)
    kc, vc, scales = written_once(p)
    x = p.to("cuda")
    cuda_attn.cache_write(x.k, x.v, *x.cache(), x.cu, **x.scales)
    assert torch.equal(x.k_cache.cpu(), kc) and torch.equal(x.v_cache.cpu(), vc)
    for n in scales:
        assert torch.equal(x.scales[n].cpu(), scales[n])
    p.k_cache, p.v_cache, p.scales = kc, vc, scales
    ref, bound, mine = po.attn(p)
    claimed = torch.zeros(9, dtype=torch.bool)
    for first, count, _ in po.layout(p, 9):
        claimed[first:first + count] = True
    out = torch.full_like(x.q, 7.0)
    cuda_attn.paged_attn(x.q, *x.cache(), x.cu, out=out, **x.scales)
    got = out.double().cpu()
    assert bool(((got - ref).abs() <= bound)[mine].all())
    assert bool((got[~claimed] == 7).all())
