"""Keys that are not finite under a mask, and masks over 8-bit caches past 4 GiB, on the GPU against the plain float64 form
(tests/draft_oracle.py)."""
import math
import os
import random
import sys

import pytest
import torch

import cuda_attn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import draft_oracle as do  # noqa: E402
import paged_oracle as po  # noqa: E402
from test_gpu_draft import BF16, E4M3, F16, F32, I8, IDS, MANY, TYPES, tree_masks  # noqa: E402

pytestmark = pytest.mark.gpu

BEFORE, BAD = 70, 4   # keys before the first sequence's new tokens, and the new token whose key is not finite


def trees(n):
    """Trees of n and 3 tokens: (sequences, sets of seen tokens, mask, rows that see BAD of the first)."""
    rng = random.Random(7)
    seqs = [(n, n + BEFORE), (3, 50)]
    sets = [set(do.ancestors(t, i)) for c, _ in seqs for t in [do.random_tree(c, 3, rng)] for i in range(c)]
    sees = torch.tensor([i < n and BAD in s for i, s in enumerate(sets)])
    assert sees.any() and not sees.all()
    return seqs, sets, do.words(sets, -(-n // 32)), sees


def run(p, mask):
    g = p.to("cuda")
    return cuda_attn.paged_tree_attn(g.q, *g.cache(), mask.cuda(), g.cu, **g.scales).double().cpu()


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("n,d", [(6, 64), (20, 64), (20, 128), (120, 64), (120, 128)])
@pytest.mark.parametrize("columns", [None, MANY])
def test_a_nan_key_reaches_every_row_that_sees_it(dtype, cache, n, d, columns):
    """A key of a drafted token (8 bits: its scale), then one before the tree, which the whole sequence sees."""
    seqs, _, mask, sees = trees(n)
    for pos, rows in ((BEFORE + BAD, sees), (30, torch.arange(n + 3) < n)):
        p = po.make(seqs, d=d, hq=4, hkv=2, dtype=dtype, cache=cache, columns=columns)
        ref, bound, _ = do.attn(p, mask)
        pg, rw = po.slot(p, 0, pos)
        if p.scales:
            p.scales["k_scale"][pg, :, rw] = math.nan
        else:
            p.k_cache[pg, :, rw, 9] = math.nan
        got = run(p, mask)
        assert bool(torch.isnan(got[rows]).all())
        assert bool(((got - ref).abs() <= bound)[~rows].all())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("n,d", [(6, 64), (20, 64), (20, 128), (120, 64), (120, 128)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("columns", [None, MANY])
def test_an_infinite_key(dtype, n, d, sign, columns):
    """A row that sees it has a score of infinity by the sign of its query: NaN, or no weight, as if it did not see the key."""
    seqs, sets, mask, sees = trees(n)
    p = po.make(seqs, d=d, hq=4, hkv=2, dtype=dtype, columns=columns)
    hidden = do.words([s - {BAD} if i < n else s for i, s in enumerate(sets)], mask.shape[1])
    ref, bound, _ = do.attn(p, hidden)
    pg, rw = po.slot(p, 0, BEFORE + BAD)
    p.k_cache[pg, :, rw, 9] = sign * math.inf
    up = sees[:, None] & (sign * p.q[..., 9] > 0)
    assert up.any() and (sees[:, None] & ~up).any()
    got = run(p, mask)
    assert torch.equal(torch.isnan(got), up[..., None].expand_as(got))
    assert bool(((got - ref).abs() <= bound)[~up].all())


@pytest.mark.parametrize("dtype,cache", [(F16, I8), (F16, E4M3), (BF16, E4M3)], ids=IDS)
@pytest.mark.parametrize("d,n", [(64, 60), (128, 70), (128, 30), (128, 6)])
def test_8_bits_past_32_bit_offsets(dtype, cache, d, n):
    """A cache of a little over 4 GiB, pages in use at both ends, values' scales over 20 powers of 2; then an infinite one."""
    page = 128
    pages = 2 ** 32 // (page * d) + 64
    kc, vc = (torch.zeros((pages, 1, page, d), dtype=cache, device="cuda") for _ in range(2))
    seqs = [(n, 300), (3, 200)]
    mask = tree_masks(seqs)
    p = po.make(seqs, d=d, hq=4, hkv=1, page=page, dtype=dtype, cache=cache, stale=0.0)
    g = torch.Generator().manual_seed(n)
    # (results within fp16: the largest scale is as it was)
    p.scales["v_scale"] *= 2.0 ** -torch.randint(0, 21, p.scales["v_scale"].shape, generator=g)
    where = torch.tensor([pages - 1, 1, pages - 2, pages // 2, 0, pages - 3, pages - 4, 2], device="cuda")[:p.k_cache.shape[0]]
    kc[where], vc[where] = p.k_cache.cuda(), p.v_cache.cuda()
    table = torch.where(p.table >= 0, where.cpu()[p.table.clamp(min=0).long()].to(torch.int32), p.table).cuda()

    def call():
        scales = {}
        for name, s in p.scales.items():
            scales[name] = torch.zeros((pages, 1, page), device="cuda", dtype=F32)
            scales[name][where] = s.cuda()
        got = cuda_attn.paged_tree_attn(p.q.cuda(), kc, vc, table, p.lengths.cuda(), mask.cuda(), p.cu.cuda(), **scales).double().cpu()
        small = p.to("cuda")
        same = cuda_attn.paged_tree_attn(small.q, *small.cache(), mask.cuda(), small.cu, **small.scales).double().cpu()
        return got, same
    ref, bound, _ = do.attn(p, mask)
    got, same = call()
    assert bool(((got - ref).abs() <= bound).all()) and bool(((same - ref).abs() <= bound).all())
    at = po.slot(p, 0, 300 - n + 2)
    p.scales["v_scale"][at[0], :, at[1]] = math.inf
    later, _, _ = do.attn(p, mask)
    got, same = call()
    for x in (got, same):
        assert torch.equal(torch.isnan(x), torch.isnan(later)) and torch.equal(torch.isinf(x), torch.isinf(later))
        rest = torch.isfinite(later)
        assert bool(((x - ref).abs() <= bound)[rest].all())
