"""The operators around drafted tokens together, as a server's step calls them: eagerly, on streams, in graphs."""
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

pytestmark = pytest.mark.gpu

F16, BF16, I8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731
HQ, HKV, D, VOCAB, MOST = 4, 2, 64, 501, 12


class Step:
    """One layer and a head: tokens' rows from an embedding, attention, probabilities from the result."""

    def __init__(self, dtype, cache, seqs, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.seqs = dtype, seqs
        self.embed = torch.randn(VOCAB, (HQ + 2 * HKV) * D, generator=g).to(dtype).cuda()
        self.head = (torch.randn(HQ * D, VOCAB, generator=g) / 4).to(dtype).cuda()
        self.freqs = cuda_attn.rope_frequencies(D, device="cuda")[0]
        pages, page = 10 * len(seqs), 16
        held = torch.int8 if cache == E4M3 else cache
        make = lambda: torch.zeros(pages, HKV, page, D, dtype=held, device="cuda").view(cache)  # noqa: E731
        self.kc, self.vc = make(), make()
        self.scales = {} if cache == dtype else {n: torch.zeros(pages, HKV, page, device="cuda") for n in ("k_scale", "v_scale")}
        self.table = torch.randperm(pages, generator=g).to(torch.int32).view(len(seqs), 10).cuda()

    def rows(self, tokens, positions):
        both = self.embed[tokens].view(-1, HQ + 2 * HKV, D)
        cuda_attn.rope(both[:, :HQ], both[:, HQ:HQ + HKV], positions, self.freqs, inplace=True)
        return both[:, :HQ], both[:, HQ:HQ + HKV], both[:, HQ + HKV:]

    def prompts(self, lengths, g):
        """The sequences' earlier tokens, by a causal call; lengths as they are behind it."""
        cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
        tokens = torch.randint(VOCAB, (sum(lengths),), generator=g).cuda()
        positions = torch.cat([torch.arange(n) for n in lengths]).cuda()
        _, k, v = self.rows(tokens, positions)
        cuda_attn.cache_write(k, v, self.kc, self.vc, self.table, torch.tensor(lengths, dtype=torch.int32).cuda(), cu, **self.scales)

    def __call__(self, tokens, parents, lengths, cu, uniform, q):
        mask, positions = cuda_attn.draft_tree(parents, lengths, cu, max_new=MOST)
        qr, k, v = self.rows(tokens, positions)
        cuda_attn.cache_write(k, v, self.kc, self.vc, self.table, lengths, cu, **self.scales)
        o = cuda_attn.paged_tree_attn(qr, self.kc, self.vc, self.table, lengths, mask, cu, max_new=MOST, **self.scales)
        probs = torch.softmax((o.reshape(o.shape[0], -1) @ self.head).float(), -1)
        path, kept, nxt = cuda_attn.verify_draft(tokens, parents, probs, uniform, cu, draft_probs=q, max_new=MOST)
        after = cuda_attn.cache_keep(self.kc, self.vc, self.table, lengths, path, kept, cu, **self.scales)
        return mask, positions, o, probs, path, kept, nxt, after


def inputs(seqs, drawn, seed):
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    trees = [do.random_tree(n, 3, rng) for n in seqs]
    total = sum(seqs)
    q = torch.softmax(torch.randn(total, VOCAB, generator=g), -1) if drawn else None
    return (torch.randint(VOCAB, (total,), generator=g).cuda(), torch.tensor([x for t in trees for x in t], dtype=torch.int32).cuda(),
            torch.rand(total, generator=g).cuda(), None if q is None else q.cuda())


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (BF16, I8), (F16, E4M3)], ids=IDS)
@pytest.mark.parametrize("drawn", [True, False])
def test_step_is_its_tokens_one_after_another(dtype, cache, drawn):
    """After a step, what the cache holds and the probabilities at the last accepted token are those of the accepted tokens
    fed one at a time to a cache of their own; each part agrees with its oracle on the way."""
    seqs, before = [12, 1, 7], [33, 5, 60]
    step = Step(dtype, cache, seqs)
    step.prompts(before, torch.Generator().manual_seed(1))
    chain = Step(dtype, cache, seqs)
    chain.prompts(before, torch.Generator().manual_seed(1))
    cu = torch.tensor([0] + seqs).cumsum(0).to(torch.int32).cuda()
    lengths = torch.tensor([b + n for b, n in zip(before, seqs)], dtype=torch.int32).cuda()
    tokens, parents, uniform, q = inputs(seqs, drawn, 3)
    tokens[1], uniform[1] = 7, 0.0   # (accepted: some path is longer than its root)
    if drawn:
        q[0, 7] = 1e-6
    mask, positions, o, probs, path, kept, nxt, after = step(tokens, parents, lengths, cu, uniform, q)
    want = do.verify(tokens.cpu(), parents.cpu(), probs.cpu(), uniform.cpu(), cu.cpu(), None if q is None else q.cpu(), MOST)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((path, kept, nxt), want))
    assert int(kept[0]) > 1 and after.tolist() == [b + int(k) for b, k in zip(before, kept)]
    for s, b in enumerate(before):
        ids = [int(i) for i in path[s, :int(kept[s])]]
        for j, i in enumerate(ids):
            row = int(cu[s]) + i
            qr, k, v = chain.rows(tokens[row:row + 1], torch.tensor([b + j]).cuda())
            now = torch.tensor([b + j + 1], dtype=torch.int32).cuda()
            cache_ = (chain.kc, chain.vc, chain.table[s:s + 1], now)
            cuda_attn.cache_write(k, v, *cache_, **chain.scales)
            single = cuda_attn.paged_attn(qr, *cache_, **chain.scales)
            # The same keys and values in another order: each result is within half a rounding of P and of itself of the
            # exact one: paged_oracle's bound, (2 u + es) A + u |o| with A = sum p |v| and es below u for scores below 50,
            # is at most 4 u times the largest value. Two such errors apart.
            u = po.HALF_STEP[dtype]
            size = (cuda_attn.cache_read(*cache_, dtype=dtype, max_len=b + j + 1, **chain.scales)[1][0].float().abs().amax())
            assert float((single[0].float() - o[row].float()).abs().max()) <= 2 * (4 * u * float(size) + 2.0 ** -24)
    a = cuda_attn.cache_read(step.kc, step.vc, step.table, after, dtype=dtype, **step.scales)
    b = cuda_attn.cache_read(chain.kc, chain.vc, chain.table, after, dtype=dtype, **chain.scales)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("drawn", [True, False])
def test_steps_in_a_graph(drawn):
    """A captured step replayed over new inputs, lengths and offsets, with eager work between the replays; every replay is the
    eager step's result."""
    seqs = [12, 5, 9]
    step, plain = Step(BF16, BF16, seqs), Step(BF16, BF16, seqs)
    for s in (step, plain):
        s.prompts([40, 20, 70], torch.Generator().manual_seed(1))
    start = (step.kc.clone(), step.vc.clone())
    tokens, parents, uniform, q = inputs(seqs, drawn, 0)
    cu = torch.tensor([0] + seqs).cumsum(0).to(torch.int32).cuda()
    lengths = torch.tensor([52, 25, 79], dtype=torch.int32).cuda()
    held = [t for t in (tokens, parents, uniform, q, cu, lengths) if t is not None]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(tokens, parents, lengths, cu, uniform, q)
    torch.cuda.current_stream().wait_stream(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(tokens, parents, lengths, cu, uniform, q)
    for replay, counts in enumerate(([12, 5, 9], [3, 12, 11], [1, 1, 12], [12, 5, 9])):
        new = inputs(counts, drawn, 10 + replay)
        total = sum(counts)
        for t, x in zip((tokens, parents, uniform, q), new):
            if t is not None:
                t[:total] = x
        cu.copy_(torch.tensor([0] + counts).cumsum(0))
        lengths.copy_(torch.tensor([b + n for b, n in zip((40, 20, 70), counts)]))
        for s in (step, plain):
            s.kc.copy_(start[0])
            s.vc.copy_(start[1])
        graph.replay()
        torch.cuda.synchronize()
        want = plain(*(t.clone() if t is not None else None for t in (tokens, parents, lengths, cu, uniform, q)))
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            a, b = (x[:total] if i < 4 else x for x in (a, b))   # (rows behind the last sequence are not set)
            assert torch.equal(a, b), (replay, i)
        assert torch.equal(step.kc, plain.kc) and torch.equal(step.vc, plain.vc)
    assert len(held) >= 5


def test_steps_on_two_streams():
    """Two servers' steps that overlap: each call has a workspace of its own."""
    seqs = [12, 5, 9]
    runs = []
    for seed in (0, 1):
        s = Step(BF16, BF16, seqs, seed)
        s.prompts([40, 20, 70], torch.Generator().manual_seed(seed))
        tokens, parents, uniform, q = inputs(seqs, True, seed)
        cu = torch.tensor([0] + seqs).cumsum(0).to(torch.int32).cuda()
        runs.append((s, (tokens, parents, torch.tensor([52, 25, 79], dtype=torch.int32).cuda(), cu, uniform, q)))
    start = [(s.kc.clone(), s.vc.clone()) for s, _ in runs]
    want = [s(*args) for s, args in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = [None, None]
        for (s, _), (k, v) in zip(runs, start):
            s.kc.copy_(k)
            s.vc.copy_(v)
        torch.cuda.synchronize()
        for i, (s, args) in enumerate(runs):
            with torch.cuda.stream(streams[i]):
                got[i] = s(*args)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
