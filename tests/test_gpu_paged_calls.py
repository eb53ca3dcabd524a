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
