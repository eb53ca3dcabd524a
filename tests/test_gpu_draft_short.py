"""Trees of drafted tokens over short sequences, beside a page table that promises long ones, on the GPU against the plain
float64 form (tests/draft_oracle.py): tiles of fewer units than a cut is worth, one a workgroup."""
import os
import random
import sys

import pytest
import torch

import cuda_attn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import draft_oracle as do  # noqa: E402
import paged_oracle as po  # noqa: E402
from test_gpu_draft import BF16, F16, IDS, I8, MANY, TYPES, check_attn, tree_masks  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,n", [(64, 24), (128, 24), (128, 48)])
@pytest.mark.parametrize("kind", ["alike", "any", "one long"])
def test_short_sequences(dtype, cache, d, n, kind):
    rng = random.Random(n + d)
    if kind == "alike":
        seqs = [(n, n + 60)] * 20
    elif kind == "any":
        seqs = [(c := rng.randint(1, n), c + rng.randint(0, 250)) for _ in range(24)] + [(0, 30), (0, 0)]
    else:
        seqs = [(c := rng.randint(1, n), c + rng.randint(0, 60)) for _ in range(15)] + [(n, 1200)]
    p = po.make(seqs, hq=8, hkv=2, d=d, page=16, dtype=dtype, cache=cache, columns=MANY)
    check_attn(p, tree_masks(seqs, seed=n), max_new=n)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, I8)], ids=IDS)
@pytest.mark.parametrize("d,n,lengths", [(64, 256, (0, 0)), (64, 250, (0, 7)), (128, 200, (0, 40)), (128, 190, (10, 66))])
def test_short_tables(dtype, cache, d, n, lengths):
    """At most 256 positions a sequence: tiles are not cut, more of them than the least share allows workgroups."""
    rng = random.Random(n)
    seqs = [(n, n + rng.randint(*lengths)) for _ in range(6)] + [(n // 3, n // 2), (1, 9)]
    check_attn(po.make(seqs, hq=4, hkv=1, d=d, page=16, dtype=dtype, cache=cache), tree_masks(seqs, seed=n), max_new=n)


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,n,columns", [(64, 40, MANY), (128, 24, MANY), (128, 64, MANY), (128, 16, None)])
def test_same_results_every_time(dtype, cache, d, n, columns):
    """Parts of a cut tile are joined in one order: the same bits from call to call, and in a graph beside eager calls."""
    seqs = [(n, n + 900), (n // 2, 333), (n, n + 64), (3, 1700)]
    p = po.make(seqs, hq=8, hkv=2, d=d, page=16, dtype=dtype, cache=cache, columns=columns).to("cuda")
    mask = tree_masks(seqs, seed=n).cuda()
    call = lambda: cuda_attn.paged_tree_attn(p.q, *p.cache(), mask, p.cu, max_new=n, **p.scales)  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(4):
        assert torch.equal(call(), first)
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, first)
