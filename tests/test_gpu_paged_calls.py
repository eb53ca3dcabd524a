"""Calls of the paged cache operators as programs make them: memory that is shared, calls that overlap, large ones."""
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
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, E4M3)], ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 6, 90])
def test_queries_and_result_in_one_buffer(dtype, cache, d, new):
    """q and out as heads of one tensor, rows of the one between rows of the other."""
    p = po.make([(new, 90), (new, 300)], d=d, hq=4, dtype=dtype, cache=cache)
    g = p.to("cuda")
    want = cuda_attn.paged_attn(g.q, *g.cache(), g.cu, **g.scales)
    for q_at, o_at in ((0, 4), (5, 1)):
        both = torch.full((2 * new, 9, d), 7.0, dtype=dtype, device="cuda")
        both[:, q_at:q_at + 4] = g.q
        back = cuda_attn.paged_attn(both[:, q_at:q_at + 4], *g.cache(), g.cu, out=both[:, o_at:o_at + 4], **g.scales)
        assert torch.equal(back, want) and torch.equal(both[:, q_at:q_at + 4], g.q)
        rest = [h for h in range(9) if not q_at <= h < q_at + 4 and not o_at <= h < o_at + 4]
        assert bool((both[:, rest] == 7).all())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
def test_result_over_the_cache_is_refused(dtype):
    p = po.make([(16, 60)], d=64, hq=2, hkv=2, dtype=dtype).to("cuda")
    rows = p.v_cache[1].transpose(0, 1)   # (page_size, heads, d) of a page
    before = p.v_cache.clone()
    with pytest.raises(RuntimeError, match="must not share memory with the cache"):
        cuda_attn.paged_attn(p.q, *p.cache(), p.cu, out=rows)
    torch.cuda.synchronize()
    assert torch.equal(p.v_cache.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
def test_a_page_copied_to_another(dtype, d):
    """cache_write of rows that lie in the cache: a page of a prefix that a sequence is about to change."""
    p = po.make([(0, 90)], hkv=3, hq=3, d=d, page=16, dtype=dtype, spare=3, stale=0.0).to("cuda")
    want_k, want_v = p.k_cache.clone(), p.v_cache.clone()
    src, dst = int(p.table[0, 2]), next(i for i in range(p.k_cache.shape[0]) if i not in p.table[0].tolist())
    want_k[dst], want_v[dst] = want_k[src], want_v[src]
    table = torch.tensor([[dst]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([16], dtype=torch.int32, device="cuda")
    cuda_attn.cache_write(p.k_cache[src].transpose(0, 1), p.v_cache[src].transpose(0, 1), p.k_cache, p.v_cache, table, lengths)
    assert torch.equal(p.k_cache, want_k) and torch.equal(p.v_cache, want_v)


def whole(p, causal=True):
    """(output, bound) of long chunks in float64, all rows of a head at once; the bound is paged_oracle.attn's."""
    tokens, hq, d = p.q.shape
    group, u = hq // p.k_cache.shape[1], po.HALF_STEP[p.q.dtype]
    out, bound = torch.zeros(p.q.shape, dtype=torch.float64), torch.zeros(p.q.shape, dtype=torch.float64)
    for s, (first, count, length) in enumerate(po.layout(p, tokens)):
        k, v, here = po.rows(p, s, length)
        assert bool(here.all())
        hidden = torch.arange(length)[None, :] > (length - count + torch.arange(count))[:, None] if causal else \
            torch.zeros(count, length, dtype=torch.bool)
        for h in range(hq):
            kh, vh, q = k[h // group], v[h // group], p.q[first:first + count, h].double()
            sc = ((q @ kh.t()) / math.sqrt(d)).masked_fill(hidden, -math.inf)
            w = torch.exp(sc - sc.amax(-1, keepdim=True))
            l = w.sum(-1, keepdim=True)
            o, a = (w @ vh) / l, (w @ vh.abs()) / l
            es = 2 * ((d + 8) * 2.0 ** -24 * (q.abs() @ kh.abs().t()).amax(-1, keepdim=True) / math.sqrt(d) + 2.0 ** -20)
            low = 2.0 ** -25 * (~hidden).sum(-1, keepdim=True) * vh.abs().max() / l if p.q.dtype == F16 else 0.0
            out[first:first + count, h] = o
            bound[first:first + count, h] = (2 * u + es) * a + low + u * o.abs() + 2.0 ** -25
    return out, bound


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3)], ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks_cut_over_many_workgroups(dtype, cache, d, causal):
    """Thousands of new tokens, most tiles shared by several workgroups, beside a single token."""
    p = po.make([(3001, 3700), (1, 2500)], hq=2, hkv=1, d=d, dtype=dtype, cache=cache)
    ref, bound = whole(p, causal)
    g = p.to("cuda")
    got = cuda_attn.paged_attn(g.q, *g.cache(), g.cu, causal=causal, **g.scales).double().cpu()
    assert bool(((got - ref).abs() <= bound).all()), float(((got - ref).abs() / bound).max())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
def test_64_dims_past_32_bit_offsets(dtype):
    """A 16-bit cache of 64 dims of a little over 4 GiB (chunks of it are read from 64-bit addresses), pages in use at
    both ends."""
    page, d = 128, 64
    pages = 2 ** 32 // (page * d * 2) + 64
    kc = torch.zeros((pages, 1, page, d), dtype=dtype, device="cuda")
    vc = torch.zeros_like(kc)
    p = po.make([(100, 300), (3, 200), (1, 90)], d=d, hq=2, hkv=1, page=page, dtype=dtype, stale=0.0)
    where = torch.tensor([pages - 1, 1, pages - 2, pages // 2, 0, pages - 3, pages - 4, 2])[:p.k_cache.shape[0]]
    kc[where.cuda()], vc[where.cuda()] = p.k_cache.cuda(), p.v_cache.cuda()
    table = torch.where(p.table >= 0, where[p.table.clamp(min=0).long()].to(torch.int32), p.table).cuda()
    lengths, cu = p.lengths.cuda(), p.cu.cuda()
    cuda_attn.cache_write(p.k.cuda(), p.v.cuda(), kc, vc, table, lengths, cu)
    p.k_cache, p.v_cache, _ = po.written(p)
    assert torch.equal(kc[where.cuda()].cpu(), p.k_cache) and torch.equal(vc[where.cuda()].cpu(), p.v_cache)
    ref, bound = whole(p)
    got = cuda_attn.paged_attn(p.q.cuda(), kc, vc, table, lengths, cu).double().cpu()
    assert bool(((got - ref).abs() <= bound).all())
    k, _ = cuda_attn.cache_read(kc, vc, table, lengths, max_len=300)
    assert torch.equal(k.double().cpu(), po.read(p, 300)[0])


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, E4M3)], ids=IDS)
def test_an_eager_call_beside_a_replay(new, dtype, cache):
    """An eager call on one stream while a captured one replays on another: both give what they give alone."""
    make = lambda seed: po.make([(new, 1400), (new, 900), (new, 260)], d=128, hq=8, hkv=2, dtype=dtype, cache=cache,  # noqa: E731
                                seed=seed, stale=0.0).to("cuda")
    a, b = make(1), make(2)
    call = lambda x: cuda_attn.paged_attn(x.q, *x.cache(), x.cu, max_new=new, **x.scales)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(a)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call(a)
    torch.cuda.synchronize()
    for replay in range(4):
        for x in (a, b):
            x.lengths -= 13 * replay
            x.q.copy_(torch.randn_like(x.q.float()).to(dtype))
        want_a, want_b = call(a), call(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        beside = [call(b) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(out, want_a)
        assert all(torch.equal(x, want_b) for x in beside)
