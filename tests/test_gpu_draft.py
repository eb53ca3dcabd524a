"""The operators around drafted tokens on the GPU against their plain float64 forms (tests/draft_oracle.py)."""
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

F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
TYPES = [(F16, F16), (BF16, BF16), (F16, I8), (BF16, I8), (F16, E4M3), (BF16, E4M3)]
IDS = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def offsets(counts):
    return torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32)


def flat(trees):
    return torch.tensor([x for t in trees for x in t], dtype=torch.int32)


def bits(t):
    return t.view(torch.int8) if t.dtype == E4M3 else t.view(torch.int16) if t.dtype in (F16, BF16) else t


# ---------------------------------------------------------------- masks and positions
def check_tree(parents, lengths, cu, max_new=None, words=None):
    masks, positions = do.draft_tree(parents, lengths, cu, max_new or min(len(parents), 1024))
    got, pos = cuda_attn.draft_tree(parents.cuda(), lengths.cuda(), cu.cuda(), max_new=max_new)
    rows = [i for i, m in enumerate(masks) if m is not None]
    want = do.words([masks[i] for i in rows], got.shape[1])
    assert got.shape == (len(parents), -(-(max_new or min(len(parents), 1024)) // 32)) and got.dtype == pos.dtype == torch.int32
    assert torch.equal(got.cpu()[rows], want) and pos.cpu()[rows].tolist() == [positions[i] for i in rows]


@pytest.mark.parametrize("counts", [[1], [2], [31], [32], [33], [64, 1, 65], [5, 0, 0, 9], [256, 100, 3], [1024], [1000, 24]])
@pytest.mark.parametrize("branch", [1, 4])
def test_tree(counts, branch):
    rng = random.Random(sum(counts) + branch)
    parents = flat([do.random_tree(n, branch, rng) if n else [] for n in counts])
    lengths = torch.tensor([n + rng.randint(0, 5000) for n in counts], dtype=torch.int32)
    check_tree(parents, lengths, offsets(counts), max_new=max(counts))
    check_tree(parents, lengths, offsets(counts))


def test_tree_of_any_parents():
    """Entries that are no earlier token, more tokens than max_new, lengths and offsets out of range, rows of no sequence."""
    g = torch.Generator().manual_seed(1)
    parents = torch.randint(-3, 90, (120,), generator=g).to(torch.int32)
    parents[7], parents[8] = 2 ** 31 - 1, -2 ** 31
    lengths = torch.tensor([70, -5, 2 ** 31 - 1], dtype=torch.int32)
    check_tree(parents, lengths, torch.tensor([0, 60, 90, 120], dtype=torch.int32))
    check_tree(parents, lengths, torch.tensor([0, 60, 90, 120], dtype=torch.int32), max_new=33)
    check_tree(parents, lengths, torch.tensor([-4, 50, 50, 110], dtype=torch.int32), max_new=64)
    check_tree(parents, lengths, torch.tensor([100, 999, 20, 10], dtype=torch.int32))
    flat_rows = parents.repeat(20)   # more tokens than a tree may have
    check_tree(flat_rows, lengths[:1], torch.tensor([0, 2400], dtype=torch.int32), max_new=1024)


def test_tree_without_offsets():
    parents = flat([[-1, 0, 1, 0, 2]] * 3)
    lengths = torch.tensor([5, 50, 7], dtype=torch.int32)
    a = cuda_attn.draft_tree(parents.cuda(), lengths.cuda())
    b = cuda_attn.draft_tree(parents.cuda(), lengths.cuda(), offsets([5, 5, 5]).cuda(), max_new=5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------- rotary positions
def check_rope(q, k, positions, freqs, scale=1.0, inplace=False, **kw):
    """Tensors on the CPU as the caller has them; both layouts against the oracle's (tokens, heads, d)."""
    dense = q.dim() == 4
    gq, gk = (None if x is None else (x.cuda() if not inplace else x) for x in (q, k))
    want = []
    for x in (q, k):
        if x is None:
            continue
        y, pos = x.cpu(), positions.cpu()
        if dense:
            b, h, n, d = y.shape
            y = y.transpose(1, 2).reshape(b * n, h, d)
            pos = pos.expand(b, n).reshape(-1)
        want.append(do.rope(y, pos, freqs, kw.get("interleaved", False), scale, kw.get("inverse", False)))
    got = cuda_attn.rope(gq, gk, positions.cuda(), freqs.cuda(), scale=scale, inplace=inplace, **kw)
    assert (got[1] is None) == (k is None)
    for x, src, (ref, err) in zip((t for t in got if t is not None), (t for t in (gq, gk) if t is not None), want):
        assert x.shape == src.shape and x.dtype == src.dtype
        y = x.double().cpu()
        if dense:
            y = y.transpose(1, 2).reshape(ref.shape)
        wrong = (y - ref).abs() > err
        assert not bool(wrong.any()), (int(wrong.sum()), float((y - ref).abs()[wrong].max()))
    return got


def freqs_of(r, base=10000.0):
    return cuda_attn.rope_frequencies(r, base)[0]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(128, 128), (64, 32), (80, 80), (96, 24), (128, 6), (66, 66), (33, 32), (2, 2), (1024, 1024), (256, 100)])
def test_rope(dtype, interleaved, d, r):
    g = torch.Generator().manual_seed(d + r)
    tokens = 7
    q, k = (torch.randn(tokens, h, d, generator=g).to(dtype) for h in (5, 2))
    positions = torch.tensor([0, 1, 77, 4095, 100003, 2 ** 31 - 1, -12], dtype=torch.int32)
    check_rope(q, k, positions, freqs_of(r), interleaved=interleaved)
    check_rope(q, None, positions.long(), freqs_of(r), scale=1.25, inverse=True, interleaved=interleaved)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_dense(dtype, interleaved):
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(3, h, 50, 64, generator=g).to(dtype) for h in (4, 1))
    f = freqs_of(48)
    check_rope(q, k, torch.arange(50), f, interleaved=interleaved)
    check_rope(q, k, torch.randint(0, 10 ** 6, (3, 50), generator=g).to(torch.int32), f, interleaved=interleaved, inverse=True)
    check_rope(q, k, torch.randint(0, 9999, (50, 3), generator=g).t(), f, interleaved=interleaved)
    check_rope(q.transpose(1, 2).contiguous().transpose(1, 2), k[:, :, :, :].expand(3, 6, 50, 64), torch.arange(0, 100, 2), f)


@pytest.mark.parametrize("shape", [(1, 1, 1, 64), (2, 3, 1, 64), (1, 2, 9, 96), (3, 1, 5, 2)])
def test_rope_dense_shapes(shape):
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(shape, generator=g), torch.randn(shape[0], 2, *shape[2:], generator=g)
    f = freqs_of(shape[3])
    check_rope(q, k, torch.full((1,), 7).expand(shape[2]), f)   # (a stride of 0)
    check_rope(q, k, torch.full((1, 1), 7).expand(shape[0], shape[2]), f, interleaved=True)
    both = torch.randn(shape[0], shape[2], shape[1] + 3, shape[3], generator=g).cuda().transpose(1, 2)   # of one projection
    q, k = both[:, :shape[1]], both[:, shape[1]:shape[1] + 2]
    before, positions = both.clone(), torch.arange(shape[2]).cuda()
    want = cuda_attn.rope(q.clone(), k.clone(), positions, f.cuda())
    cuda_attn.rope(q, k, positions, f.cuda(), inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(both[:, -1], before[:, -1])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_past_32_bits(interleaved):
    """More than 2^31 elements, in place; the last rows are those of a small call."""
    tokens = 2 ** 31 // (64 * 128) + 100
    q = torch.zeros(tokens, 64, 128, dtype=F16, device="cuda")
    q[-50:] = torch.randn(50, 64, 128, device="cuda").to(F16)
    positions, f = torch.arange(tokens, device="cuda"), freqs_of(128).cuda()
    want = cuda_attn.rope(q[-50:].clone(), None, positions[-50:], f, interleaved=interleaved)[0]
    cuda_attn.rope(q, None, positions, f, interleaved=interleaved, inplace=True)
    assert torch.equal(q[-50:], want) and not bool(q[-100:-50].any()) and not bool(q[:50].any())


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 3), (2, 2), (4, 4), (8, 8)])
def test_rope_strides_and_alignment(dtype, shift, pad):
    """Rows at any element, in place, between others that stay as they are."""
    tokens, d = 9, 64
    room = torch.randn(tokens * 7 * (d + pad) + shift + 8, generator=torch.Generator().manual_seed(shift)).to(dtype).cuda()
    rows = room[shift:shift + tokens * 7 * (d + pad)].view(tokens, 7, d + pad)
    before = room.clone()
    kept = before[shift:shift + tokens * 7 * (d + pad)].view(tokens, 7, d + pad)
    q, k, positions = rows[:, 1:4, :d], rows[:, 5:6, :d], torch.arange(50, 50 + tokens)
    f = freqs_of(64)
    want = cuda_attn.rope(kept[:, 1:4, :d], kept[:, 5:6, :d], positions.cuda(), f.cuda())
    check_rope(kept[:, 1:4, :d].cpu(), kept[:, 5:6, :d].cpu(), positions, f)
    got = cuda_attn.rope(q, k, positions.cuda(), f.cuda(), inplace=True)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    untouched = torch.ones(7, d + pad, dtype=torch.bool, device="cuda")
    untouched[1:4, :d] = untouched[5:6, :d] = False
    assert torch.equal(rows[:, untouched], kept[:, untouched])
    assert torch.equal(room[:shift], before[:shift]) and torch.equal(room[-8:], before[-8:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(interleaved):
    """inverse is the gradient: against differences of the operator (it is linear, so that any step will do: its rounding
    errors are the oracle's bounds) and against autograd of the formula in float64."""
    g = torch.Generator().manual_seed(5)
    x, v, dy = (torch.randn(11, 3, 64, generator=g) for _ in range(3))
    positions, f, scale = torch.arange(1000, 1011), freqs_of(32), 1.5
    turn = lambda t, **kw: cuda_attn.rope(t.cuda(), None, positions.cuda(), f.cuda(), interleaved=interleaved, scale=scale, **kw)[0].double().cpu()  # noqa: E731
    dx = turn(dy, inverse=True)
    x64 = x.double().requires_grad_()
    theta = positions.double()[:, None] * f
    c, s = (scale * theta.cos())[:, None], (scale * theta.sin())[:, None]
    a, b = (x64[..., 0:32:2], x64[..., 1:32:2]) if interleaved else (x64[..., :16], x64[..., 16:32])
    turned = (torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2) if interleaved else torch.cat((a * c - b * s, a * s + b * c), -1))
    torch.cat((turned, x64[..., 32:]), -1).backward(dy.double())
    _, err = do.rope(dy, positions, f, interleaved, scale, True)
    assert bool(((dx - x64.grad).abs() <= err).all())
    plus, minus = x + v, x - v
    slope = ((turn(plus) - turn(minus)) * dy.double()).sum() / 2
    step = (plus.double() - minus.double()) / 2   # what the rounded inputs differ by
    room = sum((do.rope(t, positions, f, interleaved, scale)[1] * dy.double().abs()).sum() for t in (plus, minus)) / 2
    assert abs(float(slope - (dx * step).sum())) <= float(room + (err * step.abs()).sum())


def test_rope_on_another_stream_and_many_tokens():
    q = torch.randn(5000, 3, 64, device="cuda").to(BF16)
    positions, f = torch.arange(5000, device="cuda"), freqs_of(64).cuda()
    want = cuda_attn.rope(q, None, positions, f)[0]
    ref, err = do.rope(q.cpu(), positions.cpu(), f.cpu())
    assert bool(((want.double().cpu() - ref).abs() <= err).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cuda_attn.rope(q, None, positions, f)[0]
    side.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------- attention
def check_attn(p, mask, **kw):
    ref, bound, mine = do.attn(p, mask)
    g = p.to("cuda")
    got = cuda_attn.paged_tree_attn(g.q, *g.cache(), mask.cuda(), g.cu, **kw, **g.scales).double().cpu()
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(got[mine]), bad[mine])
    err = (got - ref).abs()
    fine = ((err <= bound) | bad)[mine]
    assert bool(fine.all()), (int((~fine).sum()), float(err[mine][~fine].max()), float(bound[mine][~fine].max()))
    return got


def tree_masks(seqs, branch=3, seed=0, width=None):
    rng = random.Random(seed)
    sets = [set(do.ancestors(t, i)) for n, _ in seqs for t in [do.random_tree(n, branch, rng) if n else []] for i in range(n)]
    return do.words(sets, width or max(1, -(-max(n for n, _ in seqs) // 32)))


SEQS = {
    "one": [(1, 1), (1, 2), (1, 64), (1, 200)],
    "few": [(5, 5), (3, 130), (7, 64), (2, 33), (16, 500)],
    "tree": [(40, 40), (64, 77), (33, 301), (64, 64), (17, 63)],
    "large": [(130, 400), (1, 70), (100, 130)],
    "holes": [(0, 40), (2, 2), (0, 0), (3, 1), (4, 0), (40, 30), (17, 90)],   # none new, none held, more new than held
    "long": [(6, 1500), (33, 1031)],
}


# A page table of many columns lets the launcher expect long sequences: it then takes tiles of as many rows as a tree has.
MANY = 60000


@pytest.mark.parametrize("kind", list(SEQS))
@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,hq,hkv,page", [(64, 4, 2, 16), (128, 8, 1, 24), (128, 3, 3, 64)])
def test_attention(kind, dtype, cache, d, hq, hkv, page):
    check_attn(po.make(SEQS[kind], hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, cache=cache), tree_masks(SEQS[kind]))


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [9, 16, 17, 32, 33, 50, 64, 70, 130])
def test_tiles_of_every_size(dtype, cache, d, n):
    """4 query heads a key/value head: 36 to 520 rows, beside trees with fewer and sequences with none."""
    seqs = [(n, n + 700), (1, 333), (0, 20), (n // 2, 64 + n // 2), (n, n), (3, 129)]
    check_attn(po.make(seqs, hq=8, hkv=2, d=d, page=16, dtype=dtype, cache=cache, columns=MANY), tree_masks(seqs, seed=n), max_new=n)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F16, E4M3), (BF16, I8)], ids=IDS)
@pytest.mark.parametrize("d,n", [(64, 14), (64, 40), (128, 14), (128, 30), (128, 60)])
def test_tiles_of_many_sequences(dtype, cache, d, n):
    g = torch.Generator().manual_seed(n)
    r = lambda k: int(torch.randint(k, (1,), generator=g))  # noqa: E731
    seqs = [(0, r(50)) if i % 7 == 3 else (c := 1 + r(n), c + r(400)) for i in range(40)]
    check_attn(po.make(seqs, hq=4, hkv=1, d=d, page=16, dtype=dtype, cache=cache, columns=MANY), tree_masks(seqs), max_new=n)


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,hq", [(64, 2), (128, 8)])
@pytest.mark.parametrize("width", [1, 2, 5])
@pytest.mark.parametrize("columns", [None, MANY])
def test_any_mask(dtype, cache, d, hq, width, columns):
    """Bits of no tree: rows that see later tokens, not themselves, or nothing; fewer and more words than tokens."""
    seqs = [(70, 70), (40, 333), (9, 9), (1, 1), (3, 90)]
    g = torch.Generator().manual_seed(width)
    mask = torch.randint(-2 ** 31, 2 ** 31, (123, width), generator=g).to(torch.int32)
    mask[:5], mask[111:113] = 0, 0          # (rows of sequences without earlier keys: nothing to see)
    mask[20:25] = -1
    got = check_attn(po.make(seqs, hq=hq, hkv=2, d=d, dtype=dtype, cache=cache, columns=columns), mask)
    assert bool((got[:5] == 0).all()) and bool((got[111:113] == 0).all())


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, E4M3)], ids=IDS)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (12, 4), (16, 1), (40, 2), (96, 1), (300, 1)])
@pytest.mark.parametrize("columns", [None, MANY])
def test_head_groups(dtype, cache, hq, hkv, columns):
    seqs = [(1, 70), (4, 100), (19, 40)]
    for bound in (None, 19):
        check_attn(po.make(seqs, hq=hq, hkv=hkv, d=128, dtype=dtype, cache=cache, columns=columns), tree_masks(seqs), max_new=bound)


@pytest.mark.parametrize("page", [1, 7, 16, 48, 256])
def test_page_sizes(page):
    seqs = [(1, 70), (12, 513), (90, 300)]
    check_attn(po.make(seqs, d=64, page=page, dtype=BF16), tree_masks(seqs))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("uniform", [1, 5, 40])
def test_without_offsets(dtype, uniform):
    seqs = [(uniform, 300), (uniform, 64), (uniform, uniform)]
    check_attn(po.make(seqs, d=128, dtype=dtype, uniform=True), tree_masks(seqs))


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("max_new", [1, 8, 100000])
def test_max_new_is_a_hint(dtype, cache, max_new):
    seqs = [(1, 70), (40, 513), (100, 300)]
    check_attn(po.make(seqs, d=64, hq=8, dtype=dtype, cache=cache), tree_masks(seqs), max_new=max_new)


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("n,d", [(20, 64), (20, 128), (120, 64), (120, 128)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("columns", [None, MANY])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(dtype, cache, n, d, bad, columns):
    """A value (8 bits: its scale) of one drafted token: rows that do not see it keep their results."""
    seqs = [(n, n + 70), (3, 50)]
    rng = random.Random(7)
    sets = [set(do.ancestors(t, i)) for c, _ in seqs for t in [do.random_tree(c, 3, rng)] for i in range(c)]
    mask = do.words(sets, -(-n // 32))
    for which in ("v", "k"):
        p = po.make(seqs, d=d, hq=4, hkv=2, dtype=dtype, cache=cache, columns=columns)
        pg, rw = po.slot(p, 0, 70 + 4)
        if p.scales:
            p.scales[which + "_scale"][pg, :, rw] = bad
        else:
            getattr(p, which + "_cache")[pg, :, rw, 9] = bad
        ref, bound, _ = do.attn(p, mask)
        g = p.to("cuda")
        got = cuda_attn.paged_tree_attn(g.q, *g.cache(), mask.cuda(), g.cu, **g.scales).double().cpu()
        sees = torch.tensor([i < n and 4 in s for i, s in enumerate(sets)])
        assert sees.any() and not sees.all()
        assert bool(((got - ref).abs() <= bound)[~sees].all())
        if which == "v" and not p.scales:   # its own dim only, as the formula has it
            assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
        elif which == "v":
            assert not torch.isfinite(got[sees]).any()


def test_a_chain_is_causal_attention():
    seqs = [(5, 80), (40, 200), (1, 7)]
    p = po.make(seqs, d=128, hq=8, dtype=BF16)
    mask = tree_masks(seqs, branch=1)
    check_attn(p, mask)
    ref, bound, _ = po.attn(p)
    g = p.to("cuda")
    got = cuda_attn.paged_tree_attn(g.q, *g.cache(), mask.cuda(), g.cu).double().cpu()
    assert bool(((got - ref).abs() <= bound).all())


@pytest.mark.parametrize("columns", [None, MANY])
def test_pages_lengths_and_offsets_out_of_range(columns):
    seqs = [(2, 40), (30, 64), (20, 50)]
    mask = tree_masks(seqs)
    p = po.make(seqs, d=64, page=16, dtype=F16, columns=columns)
    p.table[0, 2], p.table[1, 3], p.table[1, 0] = -1, p.k_cache.shape[0], 2 ** 31 - 1
    check_attn(p, mask)
    p.table[2, :] = -5   # nothing to see
    check_attn(p, mask)
    p = po.make(seqs, d=64, page=16, dtype=F16, columns=columns)
    p.lengths[:] = torch.tensor([-7, 2 ** 31 - 1 if columns is None else 5000, 90], dtype=torch.int32)   # 90: past the table's columns
    check_attn(p, mask)
    p.cu[:] = torch.tensor([-3, 2, 1, 99], dtype=torch.int32)
    check_attn(p, mask)


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("n", [20, 40])
def test_absent_pages_in_every_tile(dtype, cache, page, n):
    """80 and 160 rows of 128 dims; pages that begin and end inside a tile are absent, one by one and in a row."""
    seqs = [(n, n + 300), (3, 200), (n - 1, 2 * n)]
    p = po.make(seqs, d=128, hq=8, hkv=2, page=page, dtype=dtype, cache=cache, columns=MANY)
    p.table[0, 2], p.table[0, 5:8], p.table[1, 0], p.table[1, 9], p.table[2, 1] = -1, -3, p.k_cache.shape[0], 2 ** 31 - 1, -1
    p.table[0, (n + 299) // page] = -1   # the last one
    check_attn(p, tree_masks(seqs, seed=n), max_new=n)
    p.table[0] = -1
    check_attn(p, tree_masks(seqs, seed=n), max_new=n)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, I8)], ids=IDS)
@pytest.mark.parametrize("new", [3, 70])
def test_out_mask_strides_and_rows_behind(dtype, cache, new):
    p = po.make([(new, 90), (new, 300)], d=64, hq=4, dtype=dtype, cache=cache)
    mask = tree_masks([(new, 90), (new, 300)])
    ref, bound, _ = do.attn(p, mask)
    g = p.to("cuda")
    tokens, w = 2 * new, mask.shape[1]
    both = torch.randn(tokens + 3, 9, 64, device="cuda").to(dtype)
    both[:tokens, 2:6] = g.q
    wide = torch.full((tokens + 3, w + 4), -1, dtype=torch.int32, device="cuda")
    wide[:tokens, 1:1 + w] = mask.cuda()
    room = torch.full((tokens + 3, 6, 64), 7.0, device="cuda", dtype=dtype)
    back = cuda_attn.paged_tree_attn(both[:, 2:6], *g.cache(), wide[:, 1:1 + w], g.cu, out=room[:, 1:5], **g.scales)
    assert bool(((back[:tokens].double().cpu() - ref).abs() <= bound).all())
    assert bool((room[tokens:] == 7).all()) and bool((room[:, 0] == 7).all()) and bool((room[:, 5] == 7).all())
    with pytest.raises(RuntimeError, match="share memory with the mask"):
        shared = torch.zeros(tokens * 4 * 64, dtype=dtype, device="cuda")
        view = shared[:tokens * w * 2].view(torch.int32).view(tokens, w)
        cuda_attn.paged_tree_attn(g.q, *g.cache(), view, g.cu, out=shared.view(tokens, 4, 64), **g.scales)


@pytest.mark.parametrize("d,n", [(64, 60), (128, 70), (64, 6)])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, I8)], ids=IDS)
def test_offsets_past_32_bits(dtype, cache, d, n):
    """A cache of a little over 4 GiB, pages in use at both ends."""
    page, hkv, size = 128, 1, 1 if cache == I8 else 2
    pages = 2 ** 32 // (page * hkv * d * size) + 64
    kc = torch.zeros((pages, hkv, page, d), dtype=cache, device="cuda")
    vc = torch.zeros_like(kc)
    seqs = [(n, 300), (3, 200)]
    p = po.make(seqs, d=d, hq=4, hkv=hkv, page=page, dtype=dtype, cache=cache, stale=0.0)
    where = torch.tensor([pages - 1, 1, pages - 2, pages // 2, 0, pages - 3, pages - 4, 2], device="cuda")[:p.k_cache.shape[0]]
    kc[where], vc[where] = p.k_cache.cuda(), p.v_cache.cuda()
    scales = {}
    for name, s in p.scales.items():
        scales[name] = torch.zeros((pages, hkv, page), device="cuda")
        scales[name][where] = s.cuda()
    table = torch.where(p.table >= 0, where.cpu()[p.table.clamp(min=0).long()].to(torch.int32), p.table).cuda()
    mask = tree_masks(seqs)
    ref, bound, _ = do.attn(p, mask)
    got = cuda_attn.paged_tree_attn(p.q.cuda(), kc, vc, table, p.lengths.cuda(), mask.cuda(), p.cu.cuda(), **scales)
    assert bool(((got.double().cpu() - ref).abs() <= bound).all())
    path = torch.tensor([[0, 2, n - 1], [0, 1, 2]], dtype=torch.int32)
    kept, lengths = do.keep(p, path, torch.tensor([3, 3]), p.cu)
    after = cuda_attn.cache_keep(kc, vc, table, p.lengths.cuda(), path.cuda(), torch.full((2,), 3, dtype=torch.int32, device="cuda"),
                                 p.cu.cuda(), **scales)
    assert torch.equal(after.cpu(), lengths)
    assert torch.equal(bits(kc[where]).cpu(), bits(kept["k_cache"])) and torch.equal(bits(vc[where]).cpu(), bits(kept["v_cache"]))


# ---------------------------------------------------------------- verification
def check_verify(tokens, parents, p, u, cu, q, max_new=None, place=lambda x: x.cuda()):
    most = max_new or min(len(tokens), 1024)
    want = do.verify(tokens, parents, p, u, cu, q, most)
    got = cuda_attn.verify_draft(tokens.cuda(), parents.cuda(), place(p), u.cuda(), cu.cuda(),
                                 draft_probs=None if q is None else place(q), max_new=max_new)
    for name, a, b in zip(("path", "accepted", "next"), got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), (name, a.cpu().tolist(), b.tolist())


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("branch", [1, 3])
@pytest.mark.parametrize("vocab", [1, 7, 33, 255, 4095, 4096, 4097, 20011])
def test_verify(drawn, branch, vocab):
    seqs = [8, 1, 13, 2, 0, 5, 21] + [6] * 20
    for seed, near in ((0, 0.9), (1, 0.3)):
        check_verify(*do.drafts(seqs, vocab, branch, seed, drawn, near), max_new=21)


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_large(drawn):
    check_verify(*do.drafts([70, 3, 200], 1031, 4, 2, drawn, 0.8, 1.0))
    check_verify(*do.drafts([1, 4], 300000, 2, 3, drawn, 0.8, 1.0), max_new=4)
    check_verify(*do.drafts([1024, 10], 17, 30, 4, drawn, 0.9, 1.0), max_new=1024)
    check_verify(*do.drafts([4] * 300, 11, 2, 5, drawn), max_new=4)


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_rows_at_any_address(drawn):
    def place(x):
        room = torch.full((x.shape[0], x.shape[1] + 6), math.nan, device="cuda")
        room[:, 3:-3] = x.cuda()
        return room[:, 3:-3]
    check_verify(*do.drafts([5, 9, 4], 4099, 2, 1, drawn), place=place)


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("vocab", [3000, 70001])
def test_verify_one_row_for_all(drawn, vocab):
    """Rows that are the same memory (a stride of 0)."""
    tokens, parents, p, u, cu, q = do.drafts([5, 9, 4], vocab, 2, 1, drawn)
    p, q = p[:1].expand(18, vocab), None if q is None else q[:1].expand(18, vocab)
    one = lambda x: x[:1].cuda().expand(18, vocab)  # noqa: E731
    check_verify(tokens, parents, p, u, cu, q, max_new=9, place=one)


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_past_32_bits(drawn):
    """Probabilities of more than 2^31 elements, the sequences at their end."""
    vocab, rows = 128001, 2 ** 31 // 128001 + 30
    tokens, parents, p, u, cu, q = do.drafts([9, 4], vocab, 2, 1, drawn, 0.5)
    def place(x):
        room = torch.empty(rows, vocab, device="cuda")
        room[-13:] = x.cuda()
        return room
    wide = lambda x: torch.cat([torch.zeros(rows - 13, dtype=x.dtype), x]).cuda()  # noqa: E731
    got = cuda_attn.verify_draft(wide(tokens), wide(parents), place(p), wide(u), (cu + rows - 13).to(torch.int32).cuda(),
                                 draft_probs=None if q is None else place(q), max_new=9)
    for a, b in zip(got, do.verify(tokens, parents, p, u, cu, q, 9)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("drawn", [True, False])
def test_verify_unusual_rows(drawn):
    """One-hot rows, equal models, rows without mass, elements that are not finite or negative, drafts out of the vocabulary or
    twice the same, numbers at the ends of their range, entries of parents that are no earlier token."""
    tokens, parents, p, u, cu, q = do.drafts([6] * 24, 50, 2, 9, drawn, 0.8)
    hot = torch.zeros(50)
    hot[17] = 1.0
    p[0:6] = hot
    tokens[1] = 17
    if drawn:
        q[6:12] = p[6:12]                    # accepted always; nothing left where it is not
        q[12:18] = 0.0                       # drafts that their rows say cannot be
        q[18, :25], q[24:30] = math.nan, 2 * q[24:30]
        p[30:36] = q[30:36] * (u[30:36, None] > 0.5)
    p[36:42] = 0.0
    p[42:48] = math.nan
    p[48, :10], p[49, 10:20] = math.inf, -1.0
    tokens[55], tokens[56], tokens[57] = -1, 50, 2 ** 62
    tokens[61] = tokens[62] = tokens[63]
    parents[60:66] = torch.tensor([-1, 0, 0, 0, 0, 0], dtype=torch.int32)
    parents[66:72] = torch.tensor([-1, 5, 2, 0, -9, 0], dtype=torch.int32)
    u[72:78], u[78:84], u[84:90], u[90:96] = 0.0, 1.0 - 2.0 ** -24, 1.0, math.nan
    p[96:102] *= 2.0 ** -140                 # subnormal
    p[102:108] *= 2.0 ** 100
    check_verify(tokens, parents, p, u, cu, q, max_new=6)
    long = lambda x: x if x is None else torch.cat([x, torch.zeros(x.shape[0], 70000)], 1)  # noqa: E731
    check_verify(tokens, parents, long(p), u, cu, long(q), max_new=6)   # (a vocabulary that takes more than one launch)
    check_verify(tokens, parents, p, u, cu, q, max_new=4)   # the last two tokens of each are not looked at
    check_verify(tokens, parents, p, u, torch.tensor([-5, 6, 3, 20, 200], dtype=torch.int32), q, max_new=20)


@pytest.mark.parametrize("vocab", [8191, 8192, 16385, 25353, 70001])
@pytest.mark.parametrize("some", [1, 40])
def test_verify_rows_with_unusual_elements_anywhere(vocab, some):
    """Rejections behind which another draft is tried: sums over rows with elements that count as 0, in the first and last places too."""
    tokens, parents, p, u, cu, q = do.drafts([13] * 12, vocab, 3, vocab, True, 0.2)
    g = torch.Generator().manual_seed(vocab)
    odd = torch.tensor([math.nan, math.inf, -math.inf, -0.25, -0.0, 2.0 ** -140, -(2.0 ** -149)])
    for x in (p, q):
        for row in range(0, x.shape[0], 2):
            at = torch.randint(vocab, (some,), generator=g)
            at[0] = (0, vocab - 1, vocab // 2)[row % 3]
            x[row, at] = odd[torch.randint(len(odd), (some,), generator=g)]
    check_verify(tokens, parents, p, u, cu, q, max_new=13)


def test_verify_same_results_every_time():
    tokens, parents, p, u, cu, q = do.drafts([9] * 40, 30011, 3, 4, True, 0.5)
    call = lambda: cuda_attn.verify_draft(tokens.cuda(), parents.cuda(), p.cuda(), u.cuda(), cu.cuda(), draft_probs=q.cuda(), max_new=9)  # noqa: E731
    first = call()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(call(), first))


# ---------------------------------------------------------------- the accepted rows
def check_keep(p, path, accepted):
    held, lengths = do.keep(p, path, accepted, p.cu)
    g = p.to("cuda")
    after = cuda_attn.cache_keep(*g.cache(), path.cuda(), accepted.cuda(), g.cu, **g.scales)
    assert torch.equal(after.cpu(), lengths) and torch.equal(g.lengths.cpu(), p.lengths)
    for name, want in held.items():
        got = g.scales[name] if name in g.scales else getattr(g, name)
        a, b = got.cpu(), want
        same = (a == b) | (torch.isnan(a) & torch.isnan(b)) if a.dtype == F32 else bits(a) == bits(b)
        assert bool(same.all()), name


@pytest.mark.parametrize("dtype,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("d,hkv,page", [(64, 3, 16), (128, 1, 7), (128, 24, 64)])
def test_keep(dtype, cache, d, hkv, page):
    seqs = [(1, 40), (30, 77), (0, 9), (12, 12), (40, 300), (5, 90)]
    rng = random.Random(d)
    paths, kept = [], []
    for n, _ in seqs:
        k = rng.randint(1, n) if n else 0
        row = [0] + sorted(rng.sample(range(1, n), k - 1)) if n else []
        paths.append(row + [-1] * (40 - k))
        kept.append(k)
    check_keep(po.make(seqs, hq=hkv, hkv=hkv, d=d, page=page, dtype=dtype, cache=cache), torch.tensor(paths, dtype=torch.int32),
               torch.tensor(kept, dtype=torch.int32))


def test_keep_of_anything():
    """Counts, lengths, offsets and pages out of range; entries that are no new token leave their row."""
    seqs = [(8, 40), (8, 64), (8, 30), (8, 90)]
    paths = torch.tensor([[0, 3, 5, 7], [0, -1, 99, 7], [0, 1, 2, 3], [0, 2, 2 ** 31 - 1, 5]], dtype=torch.int32)
    for kept in ([4, 4, 4, 4], [-3, 99, 0, 2], [2 ** 31 - 1, -2 ** 31, 3, 1]):
        p = po.make(seqs, d=64, page=16, dtype=F16)
        p.table[3, 5], p.table[1, 3] = -1, p.k_cache.shape[0] + 4
        check_keep(p, paths, torch.tensor(kept, dtype=torch.int32))
        p = po.make(seqs, d=64, page=16, dtype=F16)
        p.lengths[:] = torch.tensor([-1, 2 ** 31 - 1, 5, 96], dtype=torch.int32)   # 5: fewer than are new
        check_keep(p, paths, torch.tensor(kept, dtype=torch.int32))
        p = po.make(seqs, d=64, page=16, dtype=F16)
        p.cu[:] = torch.tensor([3, -5, 9, 8, 2 ** 31 - 1], dtype=torch.int32)
        check_keep(p, paths, torch.tensor(kept, dtype=torch.int32))


def test_keep_takes_paths_with_strides():
    p = po.make([(8, 40), (8, 64)], d=64, page=16, dtype=BF16)
    wide = torch.full((2, 9), -7, dtype=torch.int32)
    wide[:, 2:5] = torch.tensor([[0, 3, 5], [0, 1, 6]])
    kept = torch.tensor([3, 3], dtype=torch.int32)
    held, _ = do.keep(p, wide[:, 2:5], kept, p.cu)
    g = p.to("cuda")
    cuda_attn.cache_keep(*g.cache(), wide.cuda()[:, 2:5], kept.cuda(), g.cu)
    assert torch.equal(bits(g.k_cache).cpu(), bits(held["k_cache"])) and torch.equal(bits(g.v_cache).cpu(), bits(held["v_cache"]))
