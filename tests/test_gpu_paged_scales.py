"""paged_attn over 8-bit caches whose value scales lie far apart: a scale matters to a row as far as the row gives its
key weight, and not at all where the row does not see the key. Against a plain float64 form (tests/paged_oracle.py)."""
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
TYPES = [(F16, I8), (F16, E4M3), (BF16, I8)]
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731
# [(new tokens, length)]: tiles of 16 and 32 rows and chunks (4 query heads over 2), whole and cut over workgroups
SEQS = {"few": [(4, 90), (3, 200)], "few2": [(12, 700), (9, 64)], "chunk": [(100, 164), (60, 300)],
        "long": [(4, 3000), (2, 1500)], "long chunk": [(300, 1500), (90, 90)]}


def attend(p, **kw):
    g = p.to("cuda")
    return cuda_attn.paged_attn(g.q, *g.cache(), g.cu, **kw, **g.scales)


def by_weight(p):
    """(output, bound) in float64, causal. As paged_oracle.attn's bound, but for what P times a value's scale loses
    below fp16's normal range: that is held in units of at most 2^-8 of the row's largest weight p_j |scale_j| so far,
    so a key loses at most 2^-25 of a unit, twice where it is scaled again: 2^-32 n max_j(p_j max|v_j|) / l."""
    tokens, hq, d = p.q.shape
    group = hq // p.k_cache.shape[1]
    out, bound = torch.zeros(p.q.shape, dtype=torch.float64), torch.zeros(p.q.shape, dtype=torch.float64)
    u = po.HALF_STEP[p.q.dtype]
    for s, (first, count, length) in enumerate(po.layout(p, tokens)):
        k, v, here = po.rows(p, s, length)
        assert bool(here.all())
        seen = torch.arange(length)[None, :] <= (length - count + torch.arange(count))[:, None]
        for h in range(hq):
            kh, vh, q = k[h // group], v[h // group], p.q[first:first + count, h].double()
            vh = torch.where(torch.isfinite(vh), vh, torch.zeros((), dtype=torch.float64))
            sc = ((q @ kh.t()) / math.sqrt(d)).masked_fill(~seen, -math.inf)
            w = torch.exp(sc - sc.amax(-1, keepdim=True))
            l = w.sum(-1, keepdim=True)
            o, a = (w @ vh) / l, (w @ vh.abs()) / l
            size = ((q.abs() @ kh.abs().t()) / math.sqrt(d)).masked_fill(~seen, 0).amax(-1, keepdim=True)
            es = 2 * ((d + 8) * 2.0 ** -24 * size + 2.0 ** -20)
            low = 2.0 ** -32 * seen.sum(-1, keepdim=True) * (w * vh.abs().amax(-1)).amax(-1, keepdim=True) / l
            out[first:first + count, h] = o
            bound[first:first + count, h] = (2 * u + es) * a + low + u * o.abs() + 2.0 ** -25
    return out, bound


def check(p, rows=slice(None), **kw):
    ref, bound = by_weight(p)
    got = attend(p, **kw)
    err = (got.double().cpu() - ref).abs()[rows]
    fine = err <= bound[rows]
    assert bool(fine.all()), (int((~fine).sum()), float((err / bound[rows]).max()))
    return got


def firsts(p):
    """First row and count of each sequence."""
    return [(first, count, length) for first, count, length in po.layout(p, p.q.shape[0])]


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ratio", [1e5, 1e8])
def test_a_later_tokens_scale_reaches_no_earlier_row(kind, dtype, cache, d, ratio):
    """The last new token's value is far larger than the others': the rows before it keep their bits."""
    p = po.make(SEQS[kind], d=d, hq=4, hkv=2, dtype=dtype, cache=cache)
    plain = check(p)
    earlier = torch.ones(p.q.shape[0], dtype=torch.bool)
    for s, (first, count, length) in enumerate(firsts(p)):
        pg, rw = po.slot(p, s, length - 1)
        p.scales["v_scale"][pg, :, rw] *= ratio
        earlier[first + count - 1] = False
    got = check(p, earlier)
    assert torch.equal(got[earlier.cuda()], plain[earlier.cuda()])


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_large_value_of_no_weight(kind, dtype, cache, d, where):
    """A seen key that no row gives weight (e^-31 and less) has a value 1e8 times the others'."""
    p = po.make(SEQS[kind], d=d, hq=4, hkv=2, dtype=dtype, cache=cache)
    p.q[..., 0] = 8.0
    largest = po.LARGEST[cache]
    for s, (first, count, length) in enumerate(firsts(p)):
        if length == count:
            continue   # (no key that every row sees but the first)
        pos = {"first": 0, "middle": (length - count) // 2, "last": length - count - 1}[where]
        pg, rw = po.slot(p, s, pos)
        p.k_cache.view(torch.int8)[pg, :, rw] = 0
        p.k_cache[pg, :, rw, 0] = torch.tensor(-largest).to(cache)
        p.scales["k_scale"][pg, :, rw] = 45.0 / largest
        p.scales["v_scale"][pg, :, rw] *= 1e8
    check(p)


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
def test_a_value_of_zero_that_has_the_weight(kind, dtype, cache):
    """The first key takes most of every row's weight and its value is held as zeros, as a row below 2^-100 is."""
    p = po.make(SEQS[kind], d=64, hq=4, hkv=2, dtype=dtype, cache=cache)
    p.q[..., 0] = 8.0
    for s in range(len(SEQS[kind])):
        pg, rw = po.slot(p, s, 0)
        p.k_cache.view(torch.int8)[pg, :, rw] = 0
        p.k_cache[pg, :, rw, 0] = torch.tensor(po.LARGEST[cache]).to(cache)
        p.scales["k_scale"][pg, :, rw] = 9.0 / po.LARGEST[cache]
        p.v_cache.view(torch.int8)[pg, :, rw] = 0
        p.scales["v_scale"][pg, :, rw] = 0.0
    check(p)


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("decades", [-6, 6])
def test_scales_that_grow_or_fall_along_a_sequence(kind, dtype, cache, decades):
    """Over six decades from a thousand times down, of either sign, with scores that let every part of the sequence have its rows."""
    p = po.make(SEQS[kind], d=64, hq=4, hkv=2, dtype=dtype, cache=cache, qk_scale=2.0)
    for s, (first, count, length) in enumerate(firsts(p)):
        for pos in range(length):
            pg, rw = po.slot(p, s, pos)
            p.scales["v_scale"][pg, :, rw] *= (-1.0) ** (pos % 3) * 10.0 ** (3 + decades * (pos / length - (decades > 0)))
    check(p)


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
def test_beside_a_value_that_is_not_finite(dtype, cache, d):
    """Tiles that are taken one by one, after an infinite value that only the last rows see."""
    p = po.make([(150, 400)], d=d, hq=4, hkv=2, dtype=dtype, cache=cache)
    for pos, scale in ((310, math.inf), (399, 2e6), (320, 1e6)):
        pg, rw = po.slot(p, 0, pos)
        p.scales["v_scale"][pg, :, rw] = scale
    check(p, slice(0, 60))   # (rows at positions 250 to 309)


@pytest.mark.parametrize("d", [64, 128])
def test_past_32_bit_offsets(d):
    """A cache of a little over 4 GiB: its chunks' tiles all go one by one."""
    page, dtype, cache = 128, F16, I8
    pages = 2 ** 32 // (page * d) + 64
    p = po.make([(100, 300), (3, 200)], d=d, hq=2, hkv=1, page=page, dtype=dtype, cache=cache, stale=0.0)
    n = p.k_cache.shape[0]
    pg, rw = po.slot(p, 0, 299)
    p.scales["v_scale"][pg, :, rw] *= 1e8
    ref, bound = by_weight(p)
    kc = torch.zeros((pages, 1, page, d), dtype=torch.int8, device="cuda")
    vc = torch.zeros_like(kc)
    scales = {name: torch.zeros((pages, 1, page), device="cuda") for name in ("k_scale", "v_scale")}
    kc[-n:], vc[-n:] = p.k_cache.cuda(), p.v_cache.cuda()
    for name in scales:
        scales[name][-n:] = p.scales[name].cuda()
    table = torch.where(p.table >= 0, p.table + (pages - n), p.table).cuda()
    got = cuda_attn.paged_attn(p.q.cuda(), kc, vc, table, p.lengths.cuda(), p.cu.cuda(), **scales).double().cpu()
    rows = [i for i in range(p.q.shape[0]) if i != 99]
    assert bool(((got - ref).abs() <= bound)[rows].all())


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [60.0, 84.0])
def test_weights_next_to_nothing(kind, dtype, cache, d, gap):
    """The first key has all the weight and a value of zero; the others' weights times their scales are e^-60 to e^-90,
    down to fp32's smallest normal numbers. Their sum is zero in 16 bits, and no more than that."""
    p = po.make(SEQS[kind], d=d, hq=4, hkv=2, dtype=dtype, cache=cache)
    p.q[..., 0] = 16.0
    largest = po.LARGEST[cache]
    for s, (first, count, length) in enumerate(firsts(p)):
        for pos in range(length):
            pg, rw = po.slot(p, s, pos)
            p.k_cache.view(torch.int8)[pg, :, rw] = 0
            p.k_cache[pg, :, rw, 0] = torch.tensor(largest if pos == 0 else -largest).to(cache)
            p.scales["k_scale"][pg, :, rw] = gap / 2 * math.sqrt(d) / 16.0 / largest
            if pos == 0:
                p.v_cache.view(torch.int8)[pg, :, rw] = 0
                p.scales["v_scale"][pg, :, rw] = 0.0
    got = check(p)
    assert bool((got == 0).all() if dtype == F16 else (got.abs() < 1e-20).all())


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES + [(BF16, E4M3)], ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [0, 40, -1])
def test_an_infinite_scale(kind, dtype, cache, d, at):
    """The rows that see it are infinite by the signs of its codes, NaN where a code is zero; the others are as they were."""
    p = po.make(SEQS[kind], d=d, hq=4, hkv=2, dtype=dtype, cache=cache)
    sees = torch.zeros(p.q.shape[0], dtype=torch.bool)
    for s, (first, count, length) in enumerate(firsts(p)):
        pos = at % length
        pg, rw = po.slot(p, s, pos)
        p.scales["v_scale"][pg, :, rw] = math.inf
        p.v_cache.view(torch.int8)[pg, :, rw, ::5] = 0
        sees[first:first + count] = torch.arange(length - count, length) >= pos
    ref, bound, _ = po.attn(p)
    got = attend(p).double().cpu()
    assert bool(torch.isnan(ref[sees][..., ::5]).all()) and bool(torch.isinf(ref[sees]).any())
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), (int(torch.isnan(got).sum()), int(torch.isnan(ref).sum()))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]) and bool(((got - ref).abs() <= bound)[~sees].all())
