"""What the operators of speculative decoding are measured on: listed cases and a generator of more.

A server's step over drafted tokens: `draft_tree` makes the visibility masks and positions of each sequence's
tree of drafted tokens, `rope` turns queries and keys to their positions, `paged_tree_attn` is the attention of
the drafted tokens over the paged cache and their own ancestors, `verify_draft` accepts a path through the tree
by the target's probabilities and draws the token behind it, `cache_keep` leaves the accepted rows alone in the
cache. With `own` false the same results come from elementary torch operations, in 32 bits, and in 64 for angles
and for sums that a comparison or a choice depends on. Sizes are generic ones around this package's head dims
(64 and 128), its head counts (16 and 32) and the row lengths of its benchmark configurations.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8,
           "e4m3": torch.float8_e4m3fn}
_LARGEST = {"int8": 127.0, "e4m3": 448.0}


def _rope(dtype, b, n, hq, hkv, d, r, far, interleaved=False, inverse=False, dense=False, name=None):
    """b x n tokens; dense: (b, heads, n, d) tensors, else packed (b * n, heads, d). Positions end at `far`."""
    c = {"op": "rope", "dtype": dtype, "b": b, "n": n, "hq": hq, "hkv": hkv, "d": d, "r": r, "far": far,
         "interleaved": interleaved, "inverse": inverse, "dense": dense}
    return c if name is None else {"name": name, **c}


def _tree(s, n, ragged, branch, name=None):
    """s trees of n tokens (ragged: up to n), `branch` children a token (1: a chain)."""
    c = {"op": "tree", "s": s, "n": n, "ragged": ragged, "branch": branch}
    return c if name is None else {"name": name, **c}


def _attn(dtype, cache, s, n, ctx, hq, hkv, d, page, ragged, branch, name=None):
    c = {"op": "attn", "dtype": dtype, "cache": cache, "s": s, "n": n, "ctx": ctx, "hq": hq, "hkv": hkv, "d": d,
         "page": page, "ragged": ragged, "branch": branch}
    return c if name is None else {"name": name, **c}


def _verify(s, n, vocab, ragged, branch, drafted, near, name=None):
    """drafted: the drafts were drawn from given distributions; near: how alike the two models are, 0 to 1."""
    c = {"op": "verify", "s": s, "n": n, "vocab": vocab, "ragged": ragged, "branch": branch, "drafted": drafted,
         "near": near}
    return c if name is None else {"name": name, **c}


def _keep(cache, s, n, ctx, hkv, d, page, ragged, name=None):
    c = {"op": "keep", "cache": cache, "s": s, "n": n, "ctx": ctx, "hkv": hkv, "d": d, "page": page, "ragged": ragged}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # One generation step of 64 users far into long contexts: a few rows, where latency counts.
        _rope("bf16", 64, 1, 32, 8, 128, 128, 100000, name="rope_bf16_64x1"),
        # Gradients of a batch's queries and keys, in the layout of the dense kernels, half of each head turned.
        _rope("f16", 4, 4096, 32, 32, 128, 64, 4096, interleaved=True, inverse=True, dense=True, name="rope_grad_f16_4x4096"),
        # One user's tree of drafts: the smallest call.
        _tree(1, 26, False, 4, name="tree_1x26"),
        # A busy server's trees, some of them large.
        _tree(64, 256, True, 4, name="tree_64x256"),
        # One user's small tree over a short context: the smallest attention call.
        _attn("bf16", "bf16", 1, 16, 1000, 32, 8, 128, 16, False, 3, name="attn_bf16_1x16_over_1000"),
        # Trees of all sizes over contexts of all lengths, the cache in e4m3.
        _attn("f16", "e4m3", 24, 40, 4096, 16, 4, 64, 32, True, 3, name="attn_e4m3_d64_24x40_over_4096"),
        # Large trees of a busy server over long contexts: the largest call.
        _attn("bf16", "bf16", 32, 64, 8192, 32, 8, 128, 16, True, 4, name="attn_bf16_32x64_over_8192"),
        # One user's few proposals from a lookup (no distribution), over a small vocabulary.
        _verify(1, 5, 32000, False, 1, False, 0.7, name="verify_1x5_of_32000"),
        # Chains of a small model's drafts for many users, over a large vocabulary.
        _verify(48, 8, 128000, True, 1, True, 0.8, name="verify_drafted_48x8_of_128000"),
        # Trees with several drafts of one distribution beside each other.
        _verify(16, 21, 65537, True, 3, True, 0.5, name="verify_tree_16x21_of_65537"),
        # The accepted rows of a few users' trees in one layer's cache.
        _keep("bf16", 4, 32, 300, 8, 128, 16, False, name="keep_bf16_4x32"),
        # The same for many users, the cache in int8.
        _keep("int8", 64, 64, 700, 8, 128, 16, True, name="keep_int8_64x64"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random):
    op = rng.choices(["rope", "tree", "attn", "verify", "keep"], [3, 2, 7, 4, 2])[0]
    hkv = rng.choice([1, 2, 4, 8, 16])
    page, ragged = rng.choice([1, 8, 16, 16, 24, 32, 64]), rng.random() < 0.7
    branch = rng.choice([1, 2, 3, 4, 8])
    if op == "rope":
        dense = rng.random() < 0.4
        d = rng.choice([64, 80, 96, 128, 128, 256])
        r = rng.choice([d, d, d // 2, d // 4, 2 * rng.randint(1, d // 2)])
        hq = hkv * rng.choice([g for g in (1, 2, 4, 5, 8) if g * hkv <= 32])
        dtype = rng.choice(["f16", "bf16", "f32"])
        tokens = _spread(rng, 1, min(16384, 2 ** 27 // ((hq + hkv) * d * (2 if dtype == "f32" else 1))))
        b = _spread(rng, 1, min(64, tokens))
        return _rope(dtype, b, max(1, tokens // b), hq, hkv, d, r, _spread(rng, 16, 2 ** 20),
                     rng.random() < 0.5, rng.random() < 0.4, dense)
    if op == "tree":
        return _tree(_spread(rng, 1, 64), _spread(rng, 1, 256), ragged, branch)
    if op == "keep":
        s, n = _spread(rng, 1, 64), _spread(rng, 2, 64)
        return _keep(rng.choice(["f16", "bf16", "int8", "e4m3"]), s, n, _spread(rng, 1, 1000), min(hkv, 8), rng.choice([64, 128]), page,
                     ragged)
    n = _spread(rng, 1, 64)
    if op == "verify":
        vocab = _spread(rng, 1000, 160000)
        s = _spread(rng, 1, max(1, min(64, 48 * 8 * 128000 // (n * vocab))))
        drafted = rng.random() < 0.6
        return _verify(s, min(n, 24) if drafted else n, vocab, ragged, branch, drafted, rng.choice([0.0, 0.5, 0.7, 0.9]))
    dtype = rng.choice(["f16", "bf16"])
    cache = rng.choice([dtype, dtype, "int8", "e4m3"])
    d = rng.choice([64, 128])
    hq = hkv * rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if g * hkv <= 64])
    ctx = _spread(rng, 1, 16384)
    # At most 2^27 cached elements of keys and 2^35 products of a query's and a key's element.
    most = min(64.0, 2.0 ** 27 / ((ctx + n) * hkv * d), 2.0 ** 35 / (float(n) * (ctx + n) * hq * d) * (1 if ragged else 0.5))
    return _attn(dtype, cache, _spread(rng, 1, max(1, int(most))), n, ctx, hq, hkv, d, page, ragged, branch)


# ---------------------------------------------------------------- what a program has in hand
def _counts(case):
    """[(new tokens, tokens after the call)] of each sequence; the same for every seed."""
    rng = random.Random("%s %s %s" % (case["s"], case["n"], case.get("ctx", 0)))
    got = []
    for i in range(case["s"]):
        new, ctx = case["n"], case.get("ctx", 0)
        if case["ragged"] and i:
            new, ctx = rng.randint(max(1, new // 4), new), rng.randint(ctx // 16, ctx)
        got.append((new, new + ctx))
    return got


def _parents(case, seed):
    """Each sequence's tree, breadth first: the parent of each token among the sequence's, -1 for the first."""
    rng = random.Random("%s %s" % (case["branch"], seed))
    got = []
    for new, _ in _counts(case):
        got.append([-1] + [max(0, (i - 1) // case["branch"] - (rng.random() < 0.3 and case["branch"] > 1)) for i in range(1, new)])
    return got


def _ancestors(parents):
    """rows[i]: token i and its ancestors."""
    rows = []
    for i, p in enumerate(parents):
        rows.append([i] if p < 0 else rows[p] + [i])
    return rows


def _flat(lists, dtype=torch.int32):
    return torch.tensor([x for part in lists for x in part], dtype=dtype).cuda()


def _quantise(x, kind):
    amax = x.abs().amax(-1, keepdim=True)
    code = x * (_LARGEST[kind] / amax)
    return (code.round().to(torch.int8) if kind == "int8" else code.to(torch.float8_e4m3fn)), (amax / _LARGEST[kind]).squeeze(-1)


def _cache(case, st, g):
    lens, page = _counts(case), case["page"]
    pages_of = [-(-t // page) for _, t in lens]
    pages = sum(pages_of) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu()
    table = torch.full((case["s"], max(pages_of)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages_of):
        table[i, :n] = order[at:at + n]
        at += n
    st["table"], st["lengths"] = table.cuda(), _flat([[t] for _, t in lens])
    st["max_len"] = max(t for _, t in lens)
    held16 = _DTYPES[case["dtype"] if case["op"] == "attn" else case["cache"] if case["cache"] not in _LARGEST else "bf16"]
    for name in ("k", "v"):
        x = torch.randn((pages, case["hkv"], page, case["d"]), device="cuda", generator=g)
        x *= torch.exp(0.3 * torch.randn(x.shape[:-1] + (1,), device="cuda", generator=g))
        held, scale = _quantise(x.to(held16).float(), case["cache"]) if case["cache"] in _LARGEST else (x.to(held16), None)
        st[name + "_cache"], st[name + "_scale"] = held, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    st, op = {"case": case}, case["op"]
    if op == "rope":
        dtype, b, n, d = _DTYPES[case["dtype"]], case["b"], case["n"], case["d"]
        heads = case["hq"] + case["hkv"]
        if case["dense"]:
            st["q"] = torch.randn((b, case["hq"], n, d), device="cuda", generator=g).to(dtype)
            st["k"] = torch.randn((b, case["hkv"], n, d), device="cuda", generator=g).to(dtype)
            first = torch.randint(0, max(1, case["far"] - n) + 1, (b, 1), device="cuda", generator=g)
            st["positions"] = (first + torch.arange(n, device="cuda")).to(torch.int32)
        else:   # queries and keys as slices of one projection's output
            both = torch.randn((b * n, heads + case["hkv"], d), device="cuda", generator=g).to(dtype)
            st["q"], st["k"] = both[:, :case["hq"]], both[:, case["hq"]:heads]
            first = torch.randint(0, max(1, case["far"] - n) + 1, (b, 1), device="cuda", generator=g)
            st["positions"] = (first + torch.arange(n, device="cuda")).reshape(-1).to(torch.int32)
        # Frequencies for a context stretched to four times its length.
        i = torch.arange(0, case["r"], 2, dtype=torch.float64)
        st["freqs"] = (10000.0 ** (-i / case["r"]) / 4.0).cuda()
        return st
    lens = _counts(case)
    st["max_new"] = max(n for n, _ in lens)
    st["cu"] = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32).cuda()
    total = sum(n for n, _ in lens)
    if op == "tree":
        st["parents"], st["lengths"] = _flat(_parents(case, seed)), _flat([[t + 500 + i] for i, (_, t) in enumerate(lens)])
    elif op == "attn":
        _cache(case, st, g)
        st["q"] = torch.randn((total, case["hq"], case["d"]), device="cuda", generator=g).to(_DTYPES[case["dtype"]])
        words = -(-st["max_new"] // 32)
        masks = []
        for tree in _parents(case, 0):
            for row in _ancestors(tree):
                bits = sum(1 << j for j in row)
                masks.append([((bits >> 32 * w & 0xffffffff) ^ 0x80000000) - 0x80000000 for w in range(words)])
        st["mask"] = torch.tensor(masks, dtype=torch.int32).cuda()
    elif op == "verify":
        trees = _parents(case, seed)
        st["parents"] = _flat(trees)
        first = st["cu"].long()[:-1].repeat_interleave(st["cu"].diff().long())
        logits = 3.0 * torch.randn((total, case["vocab"]), device="cuda", generator=g)
        other = 3.0 * torch.randn((total, case["vocab"]), device="cuda", generator=g)
        other = torch.softmax(case["near"] * logits + math.sqrt(1 - case["near"] ** 2) * other, -1)
        st["p"] = torch.softmax(logits, -1)
        above = first + st["parents"].long().clamp(min=0)
        if case["drafted"]:   # each child drawn from its parent's row by itself
            cum = other.cumsum(-1, dtype=torch.float64)
            u = torch.rand(total, 1, device="cuda", dtype=torch.float64, generator=g)
            st["tokens"] = torch.searchsorted(cum[above], u * cum[above, -1:])[:, 0].clamp(max=case["vocab"] - 1)
        else:                 # the most likely ones of the row, each child another
            rank = torch.tensor([sum(1 for j in range(1, i) if t[j] == t[i]) for t in trees for i in range(len(t))]).cuda()
            st["tokens"] = torch.topk(other, min(case["vocab"], int(rank.max()) + 1), -1).indices[above, rank]
        st["q"] = other if case["drafted"] else None
        st["uniform"] = torch.rand(total, device="cuda", generator=g)
    else:
        _cache(case, st, g)
        rng = random.Random("%s %s" % (case["s"], seed))
        path, kept = [], []
        for (new, _), (accepted, in_place) in zip(lens, _accepted(case)):
            # The first `in_place` stand where they stay; the others come from behind the kept rows (so that a
            # pass can be repeated).
            behind = sorted(rng.sample(range(accepted, new), accepted - in_place))
            row = list(range(in_place)) + behind
            path.append(row + [-1] * (st["max_new"] - accepted))
            kept.append([accepted])
        st["path"], st["accepted"] = torch.tensor(path, dtype=torch.int32).cuda(), _flat(kept)
    return st


def _accepted(case):
    """[(kept tokens, those of them in place)] of each sequence; the same for every seed."""
    rng = random.Random("%s %s kept" % (case["s"], case["n"]))
    got = []
    for new, _ in _counts(case):
        accepted = rng.randint(1, min(new, 8))
        in_place = rng.randint(max(1, 2 * accepted - new), accepted)
        got.append((accepted, in_place))
    return got


# ---------------------------------------------------------------- the plain forms
def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _plain_rope(st):
    c = st["case"]
    angle = st["positions"].double()[..., None] * st["freqs"]
    if c["inverse"]:
        angle = -angle
    cos, sin = angle.cos().float(), angle.sin().float()
    axis = 1   # the heads': behind the batch in (B, H, N, d), behind the token in (tokens, H, d)
    cos, sin = cos.unsqueeze(axis), sin.unsqueeze(axis)
    return {"q": _turn(st["q"], cos, sin, c["interleaved"]), "k": _turn(st["k"], cos, sin, c["interleaved"])}


def _rows_of(st, total):
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(st["cu"][1:].long(), row, right=True)
    return seq, row - st["cu"].long()[seq]


def _plain_tree(st):
    total, n = st["parents"].shape[0], st["max_new"]
    seq, tok = _rows_of(st, total)
    first = st["cu"].long()[seq]
    seen = torch.zeros((total, 32 * -(-n // 32)), dtype=torch.bool, device="cuda")
    at, depth = tok.clone(), torch.zeros_like(tok)
    row = torch.arange(total, device="cuda")
    for _ in range(n):   # one step up each time; a root stays where it is
        seen[row, at] = True
        up = st["parents"].long()[first + at]
        depth += up >= 0
        at = torch.where(up >= 0, up, at)
    bit = torch.ones((), dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
    words = (seen.view(total, -1, 32) * bit).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words)
    before = st["lengths"].long() - st["cu"].diff().long()
    return {"mask": words.to(torch.int32), "positions": (before[seq] + depth).to(torch.int32)}


def _plain_rows(st, name, n):
    page = st["case"]["page"]
    pos = torch.arange(n, device="cuda")
    at = st["table"].long()[:, pos // page].clamp(min=0), pos % page
    held, scale = st[name + "_cache"], st[name + "_scale"]
    if held.dtype == torch.float8_e4m3fn:   # (gathered as bytes)
        x = held.view(torch.int8).transpose(1, 2)[at].view(torch.float8_e4m3fn).float()
    else:
        x = held.transpose(1, 2)[at].float()
    if scale is not None:
        x = x * scale.transpose(1, 2)[at][..., None]
    x = torch.where((pos < st["lengths"].long()[:, None])[..., None, None], x, torch.zeros((), device="cuda"))
    return x.transpose(1, 2).contiguous()


def _plain_attn(st):
    q, c = st["q"], st["case"]
    total, hq, d = q.shape
    n, length, group = st["max_new"], st["max_len"], hq // c["hkv"]
    seq, tok = _rows_of(st, total)
    pad = torch.zeros((c["s"], n, c["hkv"], group, d), device="cuda")
    pad[seq, tok] = q.float().view(total, c["hkv"], group, d)
    pad = pad.permute(0, 2, 3, 1, 4).reshape(c["s"], c["hkv"], group * n, d)
    scores = pad @ _plain_rows(st, "k", length).transpose(2, 3).contiguous()
    scores *= 1.0 / math.sqrt(d)
    scores = scores.view(c["s"], c["hkv"], group, n, length)
    key = torch.arange(length, device="cuda")
    lens = st["lengths"].long()
    before = lens - st["cu"].diff().long()
    bits = torch.zeros((c["s"], n, st["mask"].shape[1]), dtype=torch.int64, device="cuda")
    bits[seq, tok] = st["mask"].long()
    drafted = (key - before[:, None])[:, None].expand(-1, n, -1)   # which new token each key is
    inside = drafted.clamp(min=0, max=32 * bits.shape[2] - 1)
    set_ = (torch.gather(bits, 2, inside // 32) >> (inside % 32)) & 1
    sees = (drafted < 0) | (set_ > 0) & (key < lens[:, None])[:, None] & (drafted < 32 * bits.shape[2])
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    p /= p.sum(-1, keepdim=True)
    out = p.view(c["s"], c["hkv"], group * n, length) @ _plain_rows(st, "v", length)
    out = out.view(c["s"], c["hkv"], group, n, d).permute(0, 3, 1, 2, 4)
    return out[seq, tok].reshape(total, hq, d).to(q.dtype)


def _plain_verify(st):
    p, q, u, tokens, parents = st["p"], st["q"], st["uniform"].double(), st["tokens"], st["parents"].long()
    first, count = st["cu"].long()[:-1], st["cu"].diff().long()
    b, n, vocab = first.shape[0], st["max_new"], p.shape[1]
    seq = torch.arange(b, device="cuda")
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    path = torch.full((b, n), -1, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    accepted, cur = torch.ones_like(first), torch.zeros_like(first)
    taken = torch.zeros((b, vocab), dtype=torch.bool, device="cuda")   # tokens rejected at `cur`
    mass, off = torch.ones(b, dtype=torch.float64, device="cuda"), torch.zeros(b, dtype=torch.float64, device="cuda")
    for i in range(1, n):
        row = (first + i).clamp(max=tokens.shape[0] - 1)
        here, tok = (i < count) & (parents[row] == cur), tokens[row]
        if q is None:
            w = torch.where(taken[seq, tok], zero, p[first + cur, tok].double())
            yes = here & (u[row] * mass < w)
            no = here & ~yes
            mass = torch.where(no, (mass - w).clamp(min=0), mass)
            taken[seq, tok] |= no
        else:   # what is left of p after `off` times q
            left = (p[first + cur].double() - off[:, None] * q[first + cur].double()).clamp(min=0)
            size = torch.where(off == 0, torch.ones_like(off), left.sum(-1))
            yes = here & (u[row] * q[first + cur, tok].double() * size < left[seq, tok])
            off = torch.where(here & ~yes, off + size, off)
        off = torch.where(yes, zero, off)
        mass = torch.where(yes, torch.ones_like(mass), mass)
        taken &= ~yes[:, None]
        cur = torch.where(yes, i, cur)
        path[seq, accepted.clamp(max=n - 1)] = torch.where(yes, i, path[seq, accepted.clamp(max=n - 1)])
        accepted = accepted + yes
    w = p[first + cur].double()
    left = torch.where(taken, zero, w) if q is None else (w - off[:, None] * q[first + cur].double()).clamp(min=0)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
    upto = left.cumsum(-1)
    token = torch.searchsorted(upto, (u[first] * upto[:, -1])[:, None], right=True)[:, 0]
    last = torch.where(left > 0, torch.arange(vocab, device="cuda"), -1).amax(-1)
    return {"path": path.to(torch.int32), "accepted": accepted.to(torch.int32), "next": torch.minimum(token, last)}


def _plain_keep(st):
    page = st["case"]["page"]
    before = st["lengths"].long() - st["cu"].diff().long()
    seq, j = torch.nonzero(torch.arange(st["path"].shape[1], device="cuda") < st["accepted"][:, None], as_tuple=True)
    src, dst = before[seq] + st["path"].long()[seq, j], before[seq] + j
    src, dst = (st["table"].long()[seq, src // page], src % page), (st["table"].long()[seq, dst // page], dst % page)
    for name in ("k", "v"):
        held = st[name + "_cache"]
        held = held.view(torch.int8) if held.dtype == torch.float8_e4m3fn else held
        held.transpose(1, 2)[dst] = held.transpose(1, 2)[src]
        if st[name + "_scale"] is not None:
            st[name + "_scale"].transpose(1, 2)[dst] = st[name + "_scale"].transpose(1, 2)[src]
    return _kept(st, (before + st["accepted"]).to(torch.int32))


def _kept(st, lengths):
    """The caches as they are held (codes as whole numbers: they are moved, not computed)."""
    got = {"lengths": lengths}
    for name in ("k", "v"):
        held = st[name + "_cache"]
        got[name + "_cache"] = held.view(torch.int8) if held.dtype == torch.float8_e4m3fn else held
        if st[name + "_scale"] is not None:
            got[name + "_scale"] = st[name + "_scale"]
    return got


_PLAIN = {"rope": _plain_rope, "tree": _plain_tree, "attn": _plain_attn, "verify": _plain_verify, "keep": _plain_keep}


# ---------------------------------------------------------------- the framework's operators
if os.path.isdir(os.path.join(os.getcwd(), "phantom-a100_amd")) and os.path.join(os.getcwd(), "phantom-a100_amd") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "phantom-a100_amd"))


def _own(st):
    import cuda_attn

    c = st["case"]
    scales = {} if st.get("k_scale") is None else {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if c["op"] == "rope":
        q, k = cuda_attn.rope(st["q"], st["k"], st["positions"], st["freqs"], interleaved=c["interleaved"],
                              inverse=c["inverse"])
        return {"q": q, "k": k}
    if c["op"] == "tree":
        mask, positions = cuda_attn.draft_tree(st["parents"], st["lengths"], st["cu"], max_new=st["max_new"])
        return {"mask": mask, "positions": positions}
    if c["op"] == "attn":
        return cuda_attn.paged_tree_attn(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lengths"], st["mask"],
                                         st["cu"], max_new=st["max_new"], **scales)
    if c["op"] == "verify":
        path, accepted, token = cuda_attn.verify_draft(st["tokens"], st["parents"], st["p"], st["uniform"], st["cu"],
                                                       draft_probs=st["q"], max_new=st["max_new"])
        return {"path": path, "accepted": accepted, "next": token}
    lengths = cuda_attn.cache_keep(st["k_cache"], st["v_cache"], st["table"], st["lengths"], st["path"], st["accepted"],
                                   st["cu"], **scales)
    return _kept(st, lengths)


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    """Each element that the path cannot do without read or written once. Verification: the drafts, and one row of
    probabilities (two with the draft's) for each sequence's next token."""
    if case["op"] == "rope":
        size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
        tokens, heads = case["b"] * case["n"], case["hq"] + case["hkv"]
        return {"bytes": 2 * tokens * heads * case["d"] * size + 4 * tokens + 4 * case["r"], "flops": 3 * tokens * heads * case["r"]}
    lens = _counts(case)
    new, length = sum(n for n, _ in lens), sum(t for _, t in lens)
    words = -(-max(n for n, _ in lens) // 32)
    if case["op"] == "tree":
        return {"bytes": 4 * new * (2 + words) + 8 * len(lens), "flops": 0}
    if case["op"] == "verify":
        rows = (2 if case["drafted"] else 1) * len(lens)
        return {"bytes": 4 * rows * case["vocab"] + new * (20 if case["drafted"] else 16), "flops": 2 * rows * case["vocab"]}
    row = {"f16": 2, "bf16": 2, "int8": 1, "e4m3": 1}[case["cache"]] * case["d"] + (4 if case["cache"] in _LARGEST else 0)
    if case["op"] == "keep":
        moved = sum(a - here for a, here in _accepted(case))
        return {"bytes": 2 * 2 * moved * case["hkv"] * row + 8 * len(lens), "flops": 0}
    pairs = sum(n * (t - n) for n, t in lens) + sum(len(r) for tree in _parents(case, 0) for r in _ancestors(tree))
    return {"bytes": 2 * length * case["hkv"] * row + 2 * 2 * new * case["hq"] * case["d"] + 4 * new * words,
            "flops": 4 * pairs * case["hq"] * case["d"]}


# ---------------------------------------------------------------- 64 bits
def _exact_rope(st):
    c = st["case"]
    sign = -1.0 if c["inverse"] else 1.0
    theta = sign * torch.outer(st["positions"].reshape(-1).to(torch.float64), st["freqs"])
    turn = torch.polar(torch.ones_like(theta), theta)
    got = {}
    for name in ("q", "k"):
        x = st[name].double()
        if c["dense"]:
            b, h, n, d = x.shape
            x = x.transpose(1, 2).reshape(b * n, h, d)
        half = c["r"] // 2
        re = x[..., 0:c["r"]:2] if c["interleaved"] else x[..., :half]
        im = x[..., 1:c["r"]:2] if c["interleaved"] else x[..., half:c["r"]]
        z = torch.complex(re.contiguous(), im.contiguous()) * turn[:, None]
        y = x.clone()
        if c["interleaved"]:
            y[..., 0:c["r"]:2], y[..., 1:c["r"]:2] = z.real, z.imag
        else:
            y[..., :half], y[..., half:c["r"]] = z.real, z.imag
        got[name] = y.reshape(b, n, h, d).transpose(1, 2) if c["dense"] else y
    return got


def _exact_tree(st, seed):
    masks, positions = [], []
    words = -(-st["max_new"] // 32)
    for tree, length in zip(_parents(st["case"], seed), st["lengths"].tolist()):
        for row in _ancestors(tree):
            value = [0] * words
            for j in row:
                value[j // 32] |= 1 << j % 32
            masks.append([x - (1 << 32) if x >> 31 else x for x in value])
            positions.append(length - len(tree) + len(row) - 1)
    return {"mask": torch.tensor(masks, dtype=torch.int32), "positions": torch.tensor(positions, dtype=torch.int32)}


def _exact_cached(st, name, i):
    """Sequence i's cached rows, (H, length, d) in 64 bits."""
    n, page = int(st["lengths"][i]), st["case"]["page"]
    pages = st["table"][i, :-(-n // page)].long()
    if st[name + "_cache"].dtype == torch.float8_e4m3fn:
        x = st[name + "_cache"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).to(torch.float32).double()
    else:
        x = st[name + "_cache"][pages].double()
    if st[name + "_scale"] is not None:
        x = x * st[name + "_scale"][pages].double().unsqueeze(-1)
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n].contiguous()


def _exact_attn(st):
    case = st["case"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    group, first = case["hq"] // case["hkv"], 0
    for i, ((new, length), tree) in enumerate(zip(_counts(case), _parents(case, 0))):
        k, v = _exact_cached(st, "k", i), _exact_cached(st, "v", i)
        hidden = torch.ones((new, length), dtype=torch.bool)
        hidden[:, :length - new] = False
        for j, row in enumerate(_ancestors(tree)):
            hidden[j, [length - new + x for x in row]] = False
        hidden = hidden.cuda()
        for h in range(case["hq"]):
            s = st["q"][first:first + new, h].double() @ k[h // group].t().contiguous() / math.sqrt(case["d"])
            out[first:first + new, h] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1) @ v[h // group]
        first += new
    return out


def _exact_verify(st):
    tokens, parents, u = st["tokens"].tolist(), st["parents"].tolist(), st["uniform"].double().tolist()
    cu, paths, kept, drawn = st["cu"].tolist(), [], [], []
    for first, end in zip(cu, cu[1:]):
        node, path = 0, [0]
        while True:
            p = st["p"][first + node].double()
            q = None if st["q"] is None else st["q"][first + node].double()
            left, mass, chosen = p, 1.0, None
            for child in (i for i in range(node + 1, end - first) if parents[first + i] == node):
                t = tokens[first + child]
                if q is None:
                    if u[first + child] * mass < float(left[t]):
                        chosen = child
                        break
                    mass -= float(left[t])
                    left = left.clone()
                    left[t] = 0.0
                else:   # `left` is normalised after each rejection
                    if u[first + child] * float(q[t]) < float(left[t]):
                        chosen = child
                        break
                    left = (left - q).clamp(min=0.0)
                    left = left / left.sum()
            if chosen is None:
                break
            node = chosen
            path.append(node)
        if not float(left.sum()) > 0.0:
            left = p
        upto = torch.cumsum(left, 0)
        above = torch.nonzero(upto > u[first] * upto[-1])
        drawn.append(int(above[0]) if len(above) else int(torch.nonzero(left > 0)[-1]))
        kept.append(len(path))
        paths.append(path + [-1] * (st["max_new"] - len(path)))
    return {"path": torch.tensor(paths, dtype=torch.int32), "accepted": torch.tensor(kept, dtype=torch.int32),
            "next": torch.tensor(drawn, dtype=torch.int64)}


def _exact_keep(st):
    page, lengths = st["case"]["page"], []
    for i, (new, length) in enumerate(_counts(st["case"])):
        before, kept = length - new, int(st["accepted"][i])
        table, path = st["table"][i].tolist(), st["path"][i].tolist()
        for j in range(kept):   # (ascending: a source never lies before its destination)
            a, b = before + path[j], before + j
            for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
                held = st[name]
                if held is None:
                    continue
                held = held.view(torch.int8) if held.dtype == torch.float8_e4m3fn else held
                held[table[b // page], :, b % page] = held[table[a // page], :, a % page].clone()
        lengths.append(before + kept)
    return _kept(st, torch.tensor(lengths, dtype=torch.int32))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "tree":
        return _exact_tree(st, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "verify": _exact_verify, "keep": _exact_keep}[case["op"]](st)
