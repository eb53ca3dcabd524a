"""paged_attn where scores are infinite: a row whose visible scores are all -inf is NaN, as its softmax is; zeros are for
a row that sees no key. Against the plain float64 form (tests/paged_oracle.py)."""
import math
import os
import sys

import pytest
import torch

import cuda_attn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu

F16, BF16, I8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
TYPES = [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3)]
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def check(p, causal=True):
    """NaN where the formula has NaN and nowhere else; the rest within the bound."""
    ref, bound, _ = po.attn(p, causal)
    g = p.to("cuda")
    got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu, causal=causal, **g.scales).double().cpu()
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), bad), (int(torch.isnan(got).sum()), int(bad.sum()))
    assert bool((((got - ref).abs() <= bound) | bad).all())
    return bad


def first_dim(p, value):
    """Every key's first element: `value`, in 8 bits by a scale of 1."""
    if p.scales:
        p.k_cache.view(torch.int8)[..., 0] = torch.tensor(value).to(p.k_cache.dtype).view(torch.int8)
        p.scales["k_scale"][torch.isfinite(p.scales["k_scale"])] = 1.0 / 64
    else:
        p.k_cache[..., 0] = value


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 2, 70])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_the_first_token_of_a_prompt(dtype, cache, d, new, sign):
    """One visible key and an infinite element of q: NaN whatever the key's sign."""
    p = po.make([(new, new), (1, 1)], d=d, hq=4, hkv=2, dtype=dtype, cache=cache)
    first_dim(p, sign)
    p.q[0, 1, 0], p.q[0, 2, 0] = math.inf, -math.inf
    bad = check(p)
    assert bool(bad[0, 1:3].all()) and not bool(bad[0, 0].any()) and not bool(bad[1:].any())


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 200), (2, 90)], [(3, 4000), (1, 33)], [(90, 130), (1, 64)], [(150, 2500), (40, 700)]])
@pytest.mark.parametrize("causal", [True, False])
def test_every_visible_score_is_minus_infinity(dtype, cache, d, seqs, causal):
    """In tiles that are whole and in ones that are cut over workgroups; a token that sees nothing stays zeros."""
    p = po.make(seqs + [(2, 1), (3, 0)], d=d, hq=4, hkv=2, dtype=dtype, cache=cache)
    first_dim(p, 1.0)
    rows = [0, seqs[0][0] - 1, seqs[0][0]]
    for r in rows:
        p.q[r, 0, 0] = -math.inf
    bad = check(p, causal)
    assert all(bool(bad[r, 0].all()) for r in rows) and int(bad.any(-1).sum()) == len(set(rows))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("seqs", [[(2, 200)], [(3, 4000)], [(90, 190)], [(150, 2500)]])
@pytest.mark.parametrize("one", [0, 63, 100])
def test_one_key_among_minus_infinities(dtype, seqs, one):
    """All keys but one give -inf: that one has all the weight, where a row sees it, so the row is its value."""
    p = po.make(seqs, d=64, hq=2, hkv=1, dtype=dtype)
    p.q[..., 0] = p.q[..., 0].abs() + 0.25
    pg, rw = po.slot(p, 0, one)
    kept = p.k_cache[pg, :, rw].clone()
    p.k_cache[..., 0] = -math.inf
    p.k_cache[pg, :, rw] = kept
    assert not bool(check(p, False).any())
    bad = check(p)
    sees = torch.arange(seqs[0][1] - seqs[0][0], seqs[0][1]) >= one
    assert torch.equal(~bad.all(-1).all(-1), sees)
    g = p.to("cuda")
    got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu).cpu()
    assert bool((got[sees] == p.v_cache[pg, :, rw]).all())


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
def test_absent_pages_beside_minus_infinities(dtype, cache):
    """Whether a row sees a key is a matter of pages, not of scores."""
    p = po.make([(1, 100), (1, 100), (70, 100)], d=64, hq=4, hkv=2, page=16, dtype=dtype, cache=cache)
    first_dim(p, 1.0)
    p.q[:2, :, 0] = -math.inf
    p.q[40, 3, 0] = -math.inf
    p.table[0, :] = -1     # sees nothing: zeros
    p.table[1, 1:] = -1    # sees 16 keys, all of them -inf
    bad = check(p)
    assert not bool(bad[0].any()) and bool(bad[1].all()) and bool(bad[40, 3].all())
