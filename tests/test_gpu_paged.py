"""The paged cache operators on the GPU against their plain float64 forms (tests/paged_oracle.py)."""
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
TYPES = [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8), (F16, E4M3), (BF16, E4M3)]
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def bits(t):
    return t.view(torch.int8) if t.dtype == E4M3 else t.view(torch.int16) if t.dtype in (F16, BF16) else t


def same(a, b):
    """Equal bit for bit, any NaN equal to any NaN."""
    a, b = a.cpu(), b.cpu()
    if a.is_floating_point() and a.dtype != E4M3:
        nan = torch.isnan(a) & torch.isnan(b)
        return a.shape == b.shape and bool((nan | (a == b)).all())
    return a.shape == b.shape and torch.equal(bits(a), bits(b))


def check_attn(p, causal=True, **kw):
    ref, bound, mine = po.attn(p, causal)
    g = p.to("cuda")
    got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu, causal=causal, **kw, **g.scales).double().cpu()
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(got[mine]), bad[mine])
    err = (got - ref).abs()
    fine = ((err <= bound) | bad)[mine]
    assert bool(fine.all()), (int((~fine).sum()), float(err[mine][~fine].max()), float(bound[mine][~fine].max()))


SEQS = {
    "single": [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 200)],
    "few": [(5, 5), (3, 130), (7, 64), (2, 33)],
    "chunk": [(130, 130), (1, 77), (70, 301), (64, 64)],
    "holes": [(0, 40), (2, 2), (0, 0), (3, 1), (4, 0), (17, 90)],   # none new, none held, more new than held
    "long": [(3, 1500), (1, 1031), (33, 700)],
}


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,hq,hkv,page", [(64, 4, 2, 16), (128, 8, 1, 24), (128, 3, 3, 64)])
def test_attention(kind, dtype, cache, d, hq, hkv, page):
    check_attn(po.make(SEQS[kind], hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, cache=cache))


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, E4M3)], ids=IDS)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (7, 1), (12, 4), (16, 1), (40, 2), (64, 1), (96, 1)])
def test_head_groups(dtype, cache, hq, hkv):
    check_attn(po.make([(1, 70), (4, 100), (19, 40)], hq=hq, hkv=hkv, d=128, dtype=dtype, cache=cache))


@pytest.mark.parametrize("page", [1, 2, 7, 16, 48, 100, 256])
def test_page_sizes(page):
    check_attn(po.make([(1, 70), (4, 513), (90, 300)], d=64, page=page, dtype=BF16))


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
def test_every_key_visible(dtype, cache):
    check_attn(po.make([(1, 70), (4, 130), (90, 300), (3, 0), (3, 2)], d=128, dtype=dtype, cache=cache), causal=False)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("uniform", [1, 2, 40])
def test_without_offsets(dtype, uniform):
    check_attn(po.make([(uniform, 300), (uniform, 64), (uniform, uniform)], d=128, dtype=dtype, uniform=True))


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("max_new", [1, 8, 100000])
def test_max_new_is_a_hint(dtype, cache, max_new):
    """Any max_new gives right results, also one that is too small."""
    check_attn(po.make([(1, 70), (40, 513), (200, 300)], d=64, hq=8, dtype=dtype, cache=cache), max_new=max_new)


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
def test_peaked_scores(dtype, cache):
    check_attn(po.make([(1, 900), (80, 400)], d=128, dtype=dtype, cache=cache, qk_scale=3.0))


@pytest.mark.parametrize("cache", [F16, I8, E4M3], ids=IDS)
def test_values_of_unlike_size(cache):
    """Values whose scales lie far apart, in either order, and all of them small."""
    p = po.make([(1, 700), (60, 300), (2, 900)], d=64, dtype=F16, cache=cache)
    for t in (p.scales.values() if p.scales else [p.v_cache]):
        grow = torch.logspace(-4, 2, t.shape[0]).flip(0) if t.shape[0] % 2 else torch.logspace(-4, 2, t.shape[0])
        grow = grow.view(-1, *[1] * (t.dim() - 1))
        t.copy_((t.float() * (grow if t is not p.scales.get("k_scale") else 1)).to(t.dtype))
    check_attn(p)
    for t in ([p.scales["v_scale"]] if p.scales else [p.v_cache]):
        t.copy_((t.float() * 2.0 ** -10).to(t.dtype))
    check_attn(p)


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (BF16, I8)], ids=IDS)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_later_tokens_reach_no_earlier_row(dtype, cache, bad):
    """A value (or key) that is not finite changes the rows that see it and no others."""
    seqs = [(100, 150), (1, 90), (4, 64)]
    for which in ("v", "k"):
        p = po.make(seqs, d=64, dtype=dtype, cache=cache)
        for s, pos in ((0, 120), (2, 62)):
            pg, rw = po.slot(p, s, pos)
            if p.scales:
                p.scales[which + "_scale"][pg, :, rw] = bad
            else:
                getattr(p, which + "_cache")[pg, :, rw, 3] = bad
        ref, bound, mine = po.attn(p)
        g = p.to("cuda")
        got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu, **g.scales).double().cpu()
        clean = torch.ones(p.q.shape[0], dtype=torch.bool)
        clean[70:100] = False
        clean[103:105] = False
        assert torch.isfinite(got[clean]).all()
        assert bool(((got - ref).abs() <= bound)[clean].all())
        if which == "v" and not p.scales:   # the seen value: its own dim only, as the formula has it
            assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))


def test_pages_out_of_range_are_absent():
    p = po.make([(1, 100), (20, 120), (1, 64)], d=64, page=16, dtype=F16)
    p.table[0, 2], p.table[1, 3], p.table[1, 0] = -1, p.k_cache.shape[0], 2 ** 31 - 1
    p.table[2, :] = -5   # nothing to see
    check_attn(p)
    check_attn(p, causal=False)


def test_lengths_and_offsets_out_of_range():
    """No access leaves the tensors; rows without keys are zeros, rows of no sequence are left alone."""
    p = po.make([(2, 40), (30, 64), (2, 50)], d=64, page=16, dtype=F16)
    p.lengths[:] = torch.tensor([-7, 2 ** 31 - 1, 90], dtype=torch.int32)   # 90: past the table's columns
    check_attn(p)
    p.cu[:] = torch.tensor([-3, 2, 1, 99], dtype=torch.int32)
    check_attn(p)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, I8)], ids=IDS)
@pytest.mark.parametrize("new", [1, 70])
def test_out_and_strides(dtype, cache, new):
    """q and out as slices of wider tensors; what lies between and behind stays as it was."""
    p = po.make([(new, 90), (new, 300)], d=64, hq=4, dtype=dtype, cache=cache)
    ref, bound, mine = po.attn(p)
    g = p.to("cuda")
    tokens = 2 * new
    wide = torch.randn(tokens + 3, 9, 64, device="cuda").to(dtype)
    q = wide[:, 2:6]
    q[:tokens] = g.q
    room = torch.full((tokens + 3, 6, 64), 7.0, device="cuda", dtype=dtype)
    out = room[:, 1:5]
    back = cuda_attn.paged_attn(q, *g.cache(), g.cu, out=out, **g.scales)
    assert back is out
    assert bool(((out[:tokens].double().cpu() - ref).abs() <= bound).all())
    assert bool((room[tokens:] == 7).all()) and bool((room[:, 0] == 7).all()) and bool((room[:, 5] == 7).all())
    heads_first = torch.full((4, tokens, 64), 7.0, device="cuda", dtype=dtype)
    got = cuda_attn.paged_attn(q[:tokens], *g.cache(), g.cu, out=heads_first.transpose(0, 1), **g.scales)
    assert torch.equal(got, out[:tokens])


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,hkv", [(64, 3), (128, 1), (128, 8)])
def test_write(dtype, cache, d, hkv):
    p = po.make([(1, 40), (0, 9), (33, 33), (5, 3), (7, 64), (2, 500)], hkv=hkv, hq=hkv, d=d, page=24, dtype=dtype,
                cache=cache, columns=12)   # (500 > 12 x 24: the last ones have no position)
    p.table[4, 2] = -1
    big = torch.randn(p.k.shape[0], 2 * hkv + 1, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    big[1, :, 5], big[2, 0, 0], big[3], big[4, :, 1:] = 3e-5, math.inf, 0, 0
    big[5, :, 7] = math.nan
    p.k, p.v = big[:, :hkv], big[:, hkv:2 * hkv]
    kc, vc, scales = po.written(p)
    g = p.to("cuda")
    wide = big.cuda()
    cuda_attn.cache_write(wide[:, :hkv], wide[:, hkv:2 * hkv], *g.cache(), g.cu, **g.scales)
    assert same(g.k_cache, kc) and same(g.v_cache, vc)
    for n in scales:
        assert same(g.scales[n], scales[n])


def test_write_tiny_rows():
    """bf16 rows around 2^-100, where the largest code over amax would leave fp32."""
    p = po.make([(6, 6)], hkv=1, hq=1, d=64, dtype=BF16, cache=I8)
    for i, e in enumerate((-126, -101, -100, -99, -60, 127)):
        p.k[i] = (torch.randn(64, generator=torch.Generator().manual_seed(i)).clamp(-1, 1) * 2.0 ** e).to(BF16)
        p.k[i, 0, 3] = 2.0 ** e
    kc, _, scales = po.written(p)
    g = p.to("cuda")
    cuda_attn.cache_write(g.k, g.v, *g.cache(), g.cu, **g.scales)
    assert same(g.k_cache, kc) and same(g.scales["k_scale"], scales["k_scale"])


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 10)])
def test_read(dtype, cache, d, page):
    p = po.make([(0, 40), (0, 1), (0, 0), (0, 133), (0, -4)], hkv=3, hq=3, d=d, page=page, dtype=dtype, cache=cache)
    p.table[3, 1] = -1
    g = p.to("cuda")
    for n in (None, 1, 77, 200):
        k, v = cuda_attn.cache_read(*g.cache(), max_len=n, dtype=None if cache == dtype else dtype, **g.scales)
        rows = p.table.shape[1] * page if n is None else n
        rk, rv = po.read(p, rows)
        for got, ref, name in ((k, rk, "k_scale"), (v, rv, "v_scale")):
            assert got.shape == ref.shape and got.dtype == dtype
            # code * scale is rounded to fp32 and then to the type (fp16: or half a subnormal step)
            half = po.HALF_STEP[dtype] * (1 + 2.0 ** -10) if p.scales else 0.0
            assert bool(((got.double().cpu() - ref).abs() <= half * ref.abs() + (2.0 ** -25 if half else 0.0)).all())


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
def test_a_generation_runs_through_all_three(dtype, cache):
    """Two sequences: a prompt each, then steps of one token, then everything read back and attended densely."""
    h, hkv, d, page = 4, 2, 64, 16
    g = torch.Generator().manual_seed(7)
    total = [40, 29]
    q, k, v = [[torch.randn(n, hh, d, generator=g).to(dtype).cuda() for n in total] for hh in (h, hkv, hkv)]
    pages = 9
    table = torch.tensor([[3, 1, 7], [0, 8, 5]], dtype=torch.int32).cuda()
    kc, vc = (torch.zeros(pages, hkv, page, d, device="cuda").to(cache) for _ in range(2))
    scales = {n: torch.zeros(pages, hkv, page, device="cuda") for n in ("k_scale", "v_scale")} if cache in po.LARGEST else {}
    lengths = torch.tensor([37, 26], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 37, 63], dtype=torch.int32).cuda()
    part = lambda x, a, b: torch.cat([x[0][a[0]:b[0]], x[1][a[1]:b[1]]])  # noqa: E731
    outs = [[], []]
    cuda_attn.cache_write(part(k, (0, 0), (37, 26)), part(v, (0, 0), (37, 26)), kc, vc, table, lengths, cu, **scales)
    o = cuda_attn.paged_attn(part(q, (0, 0), (37, 26)), kc, vc, table, lengths, cu, **scales)
    outs[0].append(o[:37]), outs[1].append(o[37:])
    for step in range(3):
        lengths += 1
        a, b = (37 + step, 26 + step), (38 + step, 27 + step)
        cuda_attn.cache_write(part(k, a, b), part(v, a, b), kc, vc, table, lengths, **scales)
        o = cuda_attn.paged_attn(part(q, a, b), kc, vc, table, lengths, **scales)
        outs[0].append(o[:1]), outs[1].append(o[1:])
    kd, vd = cuda_attn.cache_read(kc, vc, table, lengths, dtype=dtype, **scales)
    p = po.Problem(torch.cat([q[0], q[1]]).cpu(), None, None, kc.cpu(), vc.cpu(), table.cpu(), lengths.cpu(),
                   torch.tensor([0, 40, 69], dtype=torch.int32), {n: t.cpu() for n, t in scales.items()})
    ref, bound, _ = po.attn(p)
    got = torch.cat(outs[0] + outs[1]).double().cpu()
    assert bool(((got - ref).abs() <= bound).all())
    for s in range(2):   # the rows read back through the dense entry point
        n = total[s]
        qd = q[s].transpose(0, 1).unsqueeze(0).contiguous()
        dense = [x[s:s + 1, :, :n].repeat_interleave(h // hkv, 1).contiguous() for x in (kd, vd)]
        od = cuda_attn.fused_tc(qd, *dense, True)[0].transpose(0, 1).double().cpu()
        r, b = (ref[:40], bound[:40]) if s == 0 else (ref[40:], bound[40:])
        # the dense kernel's own bound, and k and v rounded once more: each p moves by 2 u sum |q k| / sqrt(d)
        u = po.HALF_STEP[dtype]
        size = (qd[0].abs().float() @ dense[0][0].abs().float().transpose(1, 2).contiguous()).amax(-1).max().item() / math.sqrt(d)
        slack = (2 * u * size + u) * dense[1].abs().max().item() if scales else 0.0
        assert bool(((od - r).abs() <= b + slack).all())


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, E4M3)], ids=IDS)
def test_streams_and_graphs(new, dtype, cache):
    """A captured write and attention follow the lengths, pages and inputs of each replay; two graphs and eager
    calls between them on other streams do not disturb each other."""
    p = po.make([(new, 400), (new, 500), (new, 260)], d=128, hq=8, hkv=2, dtype=dtype, cache=cache, stale=0.0, columns=40)
    g = [p.to("cuda"), po.make([(new, 300)] * 3, d=128, hq=8, hkv=2, dtype=dtype, cache=cache, seed=5, stale=0.0, columns=40).to("cuda")]
    step = lambda x: (cuda_attn.cache_write(x.k, x.v, *x.cache(), x.cu, **x.scales),  # noqa: E731
                      cuda_attn.paged_attn(x.q, *x.cache(), x.cu, max_new=new, **x.scales))[1]
    eager = lambda x: cuda_attn.paged_attn(x.q, *x.cache(), x.cu, max_new=new, **x.scales)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for x in g:
            step(x)
        for x in g:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step(x))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for replay in range(4):
        for x in g:
            x.lengths -= 17 * replay
            x.q.copy_(torch.randn_like(x.q.float()).to(dtype))
            x.k.copy_(torch.randn_like(x.k.float()).to(dtype))
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
        other = eager(g[1])   # beside it, on another stream
        torch.cuda.current_stream().wait_stream(side)
        graphs[1].replay()
        torch.cuda.synchronize()
        assert other.shape == outs[1].shape
        for x, out in zip(g, outs):
            assert torch.equal(eager(x), out)
            ref, bound, _ = po.attn(x.to("cpu"))
            assert bool(((out.double().cpu() - ref).abs() <= bound).all())


def test_same_call_gives_the_same_bits():
    p = po.make([(1, 3000), (1, 200), (1, 1)], d=128, hq=8, hkv=2, dtype=BF16).to("cuda")
    first = cuda_attn.paged_attn(p.q, *p.cache())
    for _ in range(5):
        assert torch.equal(cuda_attn.paged_attn(p.q, *p.cache()), first)


def test_offsets_past_32_bits():
    """A cache of 6 GiB whose pages in use lie at its end."""
    pages, hkv, page, d = 98304, 2, 128, 128
    kc = torch.zeros((pages, hkv, page, d), dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[pages - 1, pages - 3, 5], [pages - 2, 70000, -1]], dtype=torch.int32)
    small = po.make([(1, 300), (60, 200)], d=d, hq=4, hkv=hkv, page=page, dtype=BF16, stale=0.0)
    small.table = torch.tensor([[0, 1, 2], [3, 4, -1]], dtype=torch.int32)
    where = torch.tensor([pages - 1, pages - 3, 5, pages - 2, 70000], device="cuda")
    small.k_cache, small.v_cache = (torch.randn(5, hkv, page, d, generator=g).to(BF16) for _ in range(2))
    k_new, v_new = (torch.randn(61, hkv, d, generator=g).to(BF16) for _ in range(2))
    small.k, small.v = k_new, v_new
    kc[where], vc[where] = small.k_cache.cuda(), small.v_cache.cuda()
    cu, lengths = small.cu.cuda(), small.lengths.cuda()
    cuda_attn.cache_write(k_new.cuda(), v_new.cuda(), kc, vc, table.cuda(), lengths, cu)
    small.k_cache, small.v_cache, _ = po.written(small)
    assert same(kc[where], small.k_cache) and same(vc[where], small.v_cache)
    ref, bound, _ = po.attn(small)
    got = cuda_attn.paged_attn(small.q.cuda(), kc, vc, table.cuda(), lengths, cu).double().cpu()
    assert bool(((got - ref).abs() <= bound).all())
    k, _ = cuda_attn.cache_read(kc, vc, table.cuda(), lengths, max_len=300)
    assert torch.equal(k.double().cpu(), po.read(small, 300)[0])


@pytest.mark.parametrize("dtype,cache", [(F16, E4M3), (BF16, I8)], ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
def test_8bit_offsets_past_32_bits(dtype, cache, d):
    """8-bit caches of a little over 4 GiB (chunks of them are read from 64-bit addresses), pages in use at both ends."""
    page, hkv = 128, 1
    pages = 2 ** 32 // (page * hkv * d) + 64
    kc = torch.zeros((pages, hkv, page, d), dtype=torch.int8, device="cuda")
    vc = torch.zeros_like(kc)
    scales = {n: torch.zeros((pages, hkv, page), device="cuda") for n in ("k_scale", "v_scale")}
    p = po.make([(100, 300), (3, 200), (1, 90)], d=d, hq=2, hkv=hkv, page=page, dtype=dtype, cache=cache, stale=0.0)
    where = torch.tensor([pages - 1, 1, pages - 2, pages // 2, 0, pages - 3, pages - 4, 2], device="cuda")[:p.k_cache.shape[0]]
    kc[where], vc[where] = p.k_cache.view(torch.int8).cuda(), p.v_cache.view(torch.int8).cuda()
    kc, vc = kc.view(cache), vc.view(cache)
    for n in scales:
        scales[n][where] = p.scales[n].cuda()
    table = torch.where(p.table >= 0, where.cpu()[p.table.clamp(min=0).long()].to(torch.int32), p.table)
    cuda_attn.cache_write(p.k.cuda(), p.v.cuda(), kc, vc, table.cuda(), p.lengths.cuda(), p.cu.cuda(), **scales)
    p.k_cache, p.v_cache, p.scales = po.written(p)
    assert same(kc.view(torch.int8)[where].view(cache), p.k_cache) and same(scales["v_scale"][where], p.scales["v_scale"])
    for bad in (False, True):
        if bad:   # a value that the first of the chunk's rows do not see
            pg, rw = po.slot(p, 0, 250)
            p.scales["v_scale"][pg, :, rw] = math.inf
            scales["v_scale"][where[pg], :, rw] = math.inf
        ref, bound, mine = po.attn(p)
        got = cuda_attn.paged_attn(p.q.cuda(), kc, vc, table.cuda(), p.lengths.cuda(), p.cu.cuda(), **scales).double().cpu()
        sees = torch.zeros(p.q.shape[0], dtype=torch.bool)
        sees[50:100] = bad
        assert bool(((got - ref).abs() <= bound)[~sees].all())
        assert not torch.isfinite(got[sees]).any()
        many = cuda_attn.paged_attn(p.q[:100].cuda(), kc, vc, table[:1].cuda(), p.lengths[:1].cuda(), causal=False, **scales)
        assert bool(torch.isfinite(many).all()) != bad


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, I8)], ids=IDS)
@pytest.mark.parametrize("seqs", [257, 700])
def test_many_sequences(dtype, cache, seqs):
    """More sequences than a workgroup has threads, some without new tokens; single tokens and chunks among them."""
    g = torch.Generator().manual_seed(seqs)
    r = lambda n: int(torch.randint(n, (1,), generator=g))  # noqa: E731
    sizes = [(0, r(50)) if i % 7 == 3 else (1, 1 + r(300)) if i % 50 else (40 + r(60), 100 + r(400)) for i in range(seqs)]
    p = po.make(sizes, d=64, hq=2, hkv=1, dtype=dtype, cache=cache)
    check_attn(p)
    check_attn(po.make([(1, 1 + r(90)) for _ in range(seqs)], d=128, hq=2, hkv=1, dtype=dtype, cache=cache, uniform=True))


@pytest.mark.parametrize("dtype,cache,what", [(*t, w) for t in TYPES for w in ("inf", "nan")]
                         + [(F16, E4M3, "code"), (BF16, E4M3, "code")], ids=IDS)
def test_values_that_are_not_finite_in_chunks(dtype, cache, what):
    """D = 128, tiles of 256 rows: a value (or its scale, or an e4m3 NaN code) that some rows of a tile see."""
    seqs = [(150, 400), (90, 513)]
    p = po.make(seqs, d=128, hq=4, hkv=2, dtype=dtype, cache=cache)
    seen_from = {0: 330, 1: 460}   # in the middle of a tile of keys, with tiles before and after it
    for s, pos in seen_from.items():
        pg, rw = po.slot(p, s, pos)
        if what == "code":
            p.v_cache.view(torch.int8)[pg, :, rw, 77] = 0x7f
        elif p.scales:
            p.scales["v_scale"][pg, :, rw] = math.inf if what == "inf" else math.nan
        else:
            p.v_cache[pg, :, rw, 77] = math.inf if what == "inf" else math.nan
    ref, bound, _ = po.attn(p)
    g = p.to("cuda")
    got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu, **g.scales).double().cpu()
    sees = torch.cat([torch.arange(n - c, n) >= seen_from[s] for s, (c, n) in enumerate(seqs)])
    assert bool(((got - ref).abs() <= bound)[~sees].all())
    if p.scales and what != "code":
        assert not torch.isfinite(got[sees]).any()
    else:   # one dim of the rows that see it, as the formula has it
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
        fine = torch.isfinite(ref)
        assert bool(((got - ref).abs() <= bound)[fine].all())


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("new,length", [(3, 90), (12, 700), (150, 700)])
def test_queries_that_are_not_finite(dtype, cache, new, length):
    """They change their own rows only; in rows that no sequence has they change nothing."""
    p = po.make([(new, length), (2, 70)], d=128, hq=4, hkv=2, dtype=dtype, cache=cache)
    p.q[1, 2, 5], p.q[2, 0, 7], p.q[new, 3, 1] = math.nan, math.inf, -math.inf
    p.q = torch.cat([p.q, torch.full((5, 4, 128), math.nan, dtype=dtype)])
    ref, bound, mine = po.attn(p)
    g = p.to("cuda")
    out = torch.full_like(g.q, 7.0)
    cuda_attn.paged_attn(g.q, *g.cache(), g.cu, out=out, **g.scales)
    got = out.double().cpu()
    assert bool((got[new + 2:] == 7).all())
    bad = torch.zeros(new + 2, 4, dtype=torch.bool)
    bad[1, 2] = bad[2, 0] = bad[new, 3] = True
    assert bool(torch.isnan(got[:new + 2][bad]).all())
    assert bool(((got - ref).abs() <= bound)[:new + 2][~bad].all())


@pytest.mark.parametrize("new", [1, 6, 90])
def test_shared_pages_and_a_table_with_strides(new):
    """Two sequences that share a prefix's pages, one that has a page twice; the table is a slice of a wider one."""
    p = po.make([(new, 200), (new, 230), (new, 190)], d=64, page=16, dtype=BF16)
    p.table[1, :6] = p.table[0, :6]
    p.table[2, 3] = p.table[2, 5]
    check_attn(p)
    g = p.to("cuda")
    wide = torch.full((4, 2 * p.table.shape[1] + 3), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    wide[:3, 2:2 + p.table.shape[1]] = g.table
    view = wide[:3, 2:2 + p.table.shape[1]]
    want = cuda_attn.paged_attn(g.q, *g.cache(), g.cu)
    assert torch.equal(cuda_attn.paged_attn(g.q, g.k_cache, g.v_cache, view, g.lengths, g.cu), want)
    for a, b in zip(cuda_attn.cache_read(g.k_cache, g.v_cache, view, g.lengths), cuda_attn.cache_read(*g.cache())):
        assert torch.equal(a, b)
    one = g.table[:1].expand(3, -1)   # every sequence the same pages
    p.table = p.table[:1].expand(3, -1).contiguous()
    p.lengths[:] = 190
    ref, bound, _ = po.attn(p)
    got = cuda_attn.paged_attn(g.q, g.k_cache, g.v_cache, one, p.lengths.cuda(), g.cu).double().cpu()
    assert bool(((got - ref).abs() <= bound).all())


@pytest.mark.parametrize("hq,new", [(300, 1), (300, 2), (520, 3)])
def test_groups_of_more_heads_than_a_tile_has_rows(hq, new):
    check_attn(po.make([(new, 70), (new, 130)], d=128, hq=hq, hkv=1, dtype=BF16, cache=E4M3))
    check_attn(po.make([(new, 70), (new, 330)], d=64, hq=hq, hkv=1, dtype=F16))


def test_many_lengths_out_of_range():
    """Lengths of the largest int for many sequences count as the table's capacity, in the work's division too."""
    p = po.make([(2, 90)] * 300 + [(40, 60)], d=64, page=16, dtype=F16)
    p.lengths[:] = 2 ** 31 - 1
    check_attn(p)
    check_attn(p, causal=False, max_new=2)


@pytest.mark.parametrize("new", [1, 90])
def test_two_calls_at_once(new):
    """Calls that overlap on two streams, over one cache: each has a workspace of its own."""
    p = po.make([(new, 2000), (new, 1500)], d=128, hq=8, hkv=2, dtype=BF16)
    g = p.to("cuda")
    other = torch.randn_like(g.q.float()).to(BF16)
    want = [cuda_attn.paged_attn(q, *g.cache(), g.cu, max_new=new) for q in (g.q, other)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, q in enumerate((g.q, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append(cuda_attn.paged_attn(q, *g.cache(), g.cu, max_new=new))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
