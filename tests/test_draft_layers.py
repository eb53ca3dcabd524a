"""A step over the caches of several layers, as its documentation writes it."""
import os
import random
import sys
import textwrap
import types

import pytest
import torch

import cuda_attn
from cuda_attn import draft

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import draft_oracle as do  # noqa: E402
import paged_oracle as po  # noqa: E402


def documented_keep(module, caches, **names):
    """Runs the documented lines that keep the accepted rows of all caches; returns the lengths after them."""
    lines = draft.__doc__.split("draft_probs=draft_probs, max_new=n)\n")[1].split("\n\n")[0]
    scope = {"cuda_attn": module, "caches": caches, **names}
    if "caches:" not in lines:   # (one call for each)
        for k_cache, v_cache in caches:
            scope.update(k_cache=k_cache, v_cache=v_cache)
            exec(textwrap.dedent(lines), scope)
        return scope["lengths"]
    exec(textwrap.dedent(lines), scope)
    return scope["lengths"]


def test_every_layer_keeps_rows_by_the_same_lengths():
    seen = []

    def keep(k, v, table, lengths, path, accepted, cu):
        seen.append((k, v, lengths))
        return lengths - 7
    after = documented_keep(types.SimpleNamespace(cache_keep=keep), [("k0", "v0"), ("k1", "v1"), ("k2", "v2")], page_table=None, lengths=50,
                            path=None, accepted=None, cu_seqlens=None)
    assert seen == [("k0", "v0", 50), ("k1", "v1", 50), ("k2", "v2", 50)] and after == 43


@pytest.mark.gpu
def test_three_layers():
    seqs, rng = [(12, 40), (30, 77), (1, 9), (40, 300)], random.Random(3)
    paths, kept = [], []
    for n, _ in seqs:
        k = rng.randint(1, n)
        paths.append([0] + sorted(rng.sample(range(1, n), k - 1)) + [-1] * (40 - k))
        kept.append(k)
    path, accepted = torch.tensor(paths, dtype=torch.int32), torch.tensor(kept, dtype=torch.int32)
    layers = [po.make(seqs, hq=2, hkv=2, d=64, page=16, dtype=torch.bfloat16) for _ in range(3)]
    for i, p in enumerate(layers):
        p.k_cache, p.v_cache = p.k_cache * (i + 1), p.v_cache * (i + 1)
    want = [do.keep(p, path, accepted, p.cu) for p in layers]
    on = [p.to("cuda") for p in layers]
    _, _, table, lengths = on[0].cache()
    after = documented_keep(cuda_attn, [p.cache()[:2] for p in on], page_table=table, lengths=lengths, path=path.cuda(), accepted=accepted.cuda(),
                            cu_seqlens=on[0].cu)
    bits = lambda x: x.cpu().view(torch.int16)  # noqa: E731
    for p, (held, lengths) in zip(on, want):
        assert torch.equal(after.cpu(), lengths)
        assert torch.equal(bits(p.k_cache), bits(held["k_cache"])) and torch.equal(bits(p.v_cache), bits(held["v_cache"]))
