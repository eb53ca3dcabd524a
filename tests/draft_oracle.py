"""Plain float64 forms of the operators around drafted tokens, on the CPU. Nothing here uses the package."""
from __future__ import annotations

import math
import random

import numpy as np
import torch

import paged_oracle as po

TREE_MAX = 1024


def spans(cu, tokens):
    """[(first row, count)] of each sequence under the documented clamps."""
    got = []
    for b, e in zip(cu.tolist(), cu.tolist()[1:]):
        b = min(max(b, 0), tokens)
        got.append((b, min(max(e, b), tokens) - b))
    return got


def random_tree(n, branch, rng):
    """Parents of n tokens, breadth first with some disorder; -1 for the root."""
    return [-1] + [max(0, (i - 1) // branch - rng.randint(0, 1)) if branch > 1 else i - 1 for i in range(1, n)]


def ancestors(parents, i):
    """Token i and its ancestors; entries that are no earlier token end the way up."""
    got = [i]
    while 0 <= parents[i] < i:
        i = parents[i]
        got.append(i)
    return got


def draft_tree(parents, lengths, cu, max_new):
    """(mask as rows of Python sets, positions) for the rows of some sequence; others are None."""
    masks, positions = [None] * len(parents), [None] * len(parents)
    for s, (first, count) in enumerate(spans(cu, len(parents))):
        tree = parents[first:first + count].tolist()
        length = min(max(int(lengths[s]), 0), 2 ** 30)
        for i in range(count):
            up = ancestors(tree, i) if i < max_new else []
            masks[first + i] = set(up)
            positions[first + i] = length - count + max(len(up) - 1, 0)
    return masks, positions


def words(sets, n):
    """Rows of bit sets as an int32 tensor of n words (None: zeros)."""
    rows = []
    for bits in sets:
        value = sum(1 << j for j in bits or ())
        rows.append([(value >> 32 * w & 0xffffffff) - (1 << 32) * (value >> 32 * w + 31 & 1) for w in range(n)])
    return torch.tensor(rows, dtype=torch.int32)


def attn(p, mask):
    """(output, bound on a kernel's error, rows of exactly one sequence) with the mask's bits. The bound is
    paged_oracle.attn's: the same kernels and roundings."""
    tokens, hq, d = p.q.shape
    hkv, page = p.k_cache.shape[1], p.k_cache.shape[2]
    out = torch.zeros(p.q.shape, dtype=torch.float64)
    bound = torch.zeros(p.q.shape, dtype=torch.float64)
    claims = torch.zeros(tokens, dtype=torch.long)
    finite = lambda x: torch.where(torch.isfinite(x), x, torch.zeros((), dtype=x.dtype))  # noqa: E731
    u, width = po.HALF_STEP[p.q.dtype], 32 * mask.shape[1]
    shift = torch.arange(32)
    for s, (first, count, length) in enumerate(po.layout(p, tokens)):
        if count == 0:
            continue
        k, v, here = po.rows(p, s, min(length, p.table.shape[1] * page))
        claims[first:first + count] += 1
        n = k.shape[1]
        drafted = torch.arange(n) - (length - count)   # the new token that each key is
        bits = (mask[first:first + count].long()[..., None] >> shift & 1).reshape(count, width).bool()
        inside = (drafted >= 0) & (drafted < width)
        seen = (drafted < 0).expand(count, n).clone()
        seen[:, inside] = bits[:, drafted[inside]]
        seen &= here[None, :]
        for h in range(hq):
            kh, vh = k[h // (hq // hkv)], v[h // (hq // hkv)]
            kh = torch.where(here[:, None], kh, torch.zeros((), dtype=torch.float64))
            q = p.q[first:first + count, h].double()
            sc = (q @ kh.t()) / math.sqrt(d)
            for i in range(count):   # rows that see different keys: nothing of an unseen value may reach them
                use = seen[i]
                if not use.any():
                    continue
                w = torch.exp(sc[i, use] - sc[i, use].max())
                l = w.sum()
                out[first + i, h] = (w @ vh[use]) / l
                a = (w @ vh[use].abs()) / l
                size = (q[i].abs() @ kh[use].abs().t()).max() / math.sqrt(d)
                es = 2 * ((d + 8) * 2.0 ** -24 * size + 2.0 ** -20)
                low = 2.0 ** -25 * use.sum() * finite(vh[use]).abs().max() / l if p.q.dtype == torch.float16 else 0.0
                bound[first + i, h] = (2 * u + es) * a + low + u * out[first + i, h].abs() + 2.0 ** -25
    return out, bound, claims == 1


def counted(x):
    """Elements as the verification counts them."""
    x = x.double()
    return torch.where((x > 0) & (x < math.inf), x, torch.zeros((), dtype=torch.float64))


def verify(tokens, parents, p, uniform, cu, q=None, max_new=TREE_MAX):
    """(path, accepted, next), the walk of each sequence with its residual distribution held and normalised."""
    paths, kept, drawn = [], [], []
    vocab = p.shape[1]
    for first, count in spans(cu, len(tokens)):
        count = min(count, max_new)
        tree, tok = parents[first:first + count].tolist(), tokens[first:first + count].tolist()
        u = uniform[first:first + count].double().tolist()
        if count == 0:
            paths.append([-1] * max_new), kept.append(0), drawn.append(-1)
            continue
        node, path = 0, [0]
        while True:
            row = counted(p[first + node])
            left, mass, chosen = row.clone(), 1.0, None
            dist = None if q is None else counted(q[first + node])
            for i in range(node + 1, count):
                t = tok[i]
                if tree[i] != node or not 0 <= t < vocab:
                    continue
                if q is None:
                    if u[i] * mass < float(left[t]):
                        chosen = i
                        break
                    mass = max(mass - float(left[t]), 0.0)
                    left[t] = 0.0
                else:
                    if u[i] * float(dist[t]) < float(left[t]):
                        chosen = i
                        break
                    left = (left - dist).clamp(min=0.0)
                    total = float(left.sum())
                    if total > 0.0:
                        left /= total
            if chosen is None:
                break
            node = chosen
            path.append(node)
        left = left if float(left.sum()) > 0.0 else row
        upto = left.cumsum(0)
        above = torch.nonzero((upto > u[0] * upto[-1]) & (left > 0))
        some = torch.nonzero(left > 0)
        drawn.append(int(above[0]) if len(above) else int(some[-1]) if len(some) else -1)
        kept.append(len(path))
        paths.append(path + [-1] * (max_new - len(path)))
    return (torch.tensor(paths, dtype=torch.int32), torch.tensor(kept, dtype=torch.int32), torch.tensor(drawn, dtype=torch.int64))


def drafts(seqs, vocab, branch, seed=0, drawn=True, near=0.7, sharp=2.0):
    """A verification problem of trees of `seqs` tokens each: (tokens, parents, p, uniform, cu, q or None)."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    trees = [random_tree(n, branch, rng) if n else [] for n in seqs]
    total = sum(seqs)
    parents = torch.tensor([x for t in trees for x in t], dtype=torch.int32)
    cu = torch.tensor([0] + list(seqs)).cumsum(0).to(torch.int32)
    logits = sharp * torch.randn(total, vocab, generator=g)
    other = near * logits + math.sqrt(1 - near * near) * sharp * torch.randn(total, vocab, generator=g)
    p, q = torch.softmax(logits, -1), torch.softmax(other, -1)
    tokens = torch.zeros(total, dtype=torch.int64)
    for first, count in spans(cu, total):
        for i in range(1, count):
            up = first + max(int(parents[first + i]), 0)
            if drawn:
                tokens[first + i] = torch.multinomial(q[up].double(), 1, generator=g)
            else:
                rank = sum(int(parents[first + j]) == int(parents[first + i]) for j in range(1, i))
                tokens[first + i] = torch.argsort(q[up], descending=True)[min(rank, vocab - 1)]
    return tokens, parents, p, torch.rand(total, generator=g), cu, q if drawn else None


def keep(p, path, accepted, cu):
    """The caches and scales after cache_keep, and the lengths."""
    held = {"k_cache": p.k_cache.clone(), "v_cache": p.v_cache.clone(), **{n: t.clone() for n, t in p.scales.items()}}
    raw = {n: t.view(torch.int8) if t.dtype == torch.float8_e4m3fn else t for n, t in held.items()}
    lengths = []
    for s, (first, count) in enumerate(spans(cu, 2 ** 30)):
        length = min(max(int(p.lengths[s]), 0), 2 ** 30)
        kept = min(max(int(accepted[s]), 0), count, path.shape[1])
        for j in range(kept):
            i = int(path[s, j])
            src = po.slot(p, s, length - count + i) if 0 <= i < count else None
            dst = po.slot(p, s, length - count + j)
            if src is not None and dst is not None:
                for t in raw.values():
                    t[dst[0], :, dst[1]] = t[src[0], :, src[1]].clone()
        lengths.append(max(length - count + kept, 0))
    return held, torch.tensor(lengths, dtype=torch.int32)


def rope(x, positions, freqs, interleaved=False, scale=1.0, inverse=False):
    """(result, bound on a kernel's error) in float64, x (tokens, heads, d).

    The bound counts: cos and sin in fp32 of an angle whose fraction is rounded to 2^-28 of a turn (2.4e-8 rad), from
    functions good to 2 units in the last place of values below 1 (2 * 2^-24), times the scale (2^-24 more): below
    4 * 2^-24 of the scale; a product and a fused product and sum, 2 * 2^-24; the rounding of the result."""
    r = 2 * freqs.shape[0]
    # 64 bits would leave position 2^31 off by 2^-22: angles in numpy's longer type, a whole number of turns taken off.
    turn = 8 * np.arctan(np.longdouble(1))
    theta = np.multiply.outer(positions.numpy().astype(np.longdouble), freqs.double().numpy().astype(np.longdouble))
    theta = torch.from_numpy(np.fmod(theta, turn).astype(np.float64)) * (-1.0 if inverse else 1.0)
    c, s = (scale * theta.cos())[:, None], (scale * theta.sin())[:, None]
    y = x.double()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    out, err = y.clone(), torch.zeros_like(y)
    size = 6 * 2.0 ** -24 * scale * (a.abs() + b.abs())
    ends = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u = {torch.float32: 2.0 ** -24, **po.HALF_STEP}[x.dtype]
    for at, z in zip(ends, (a * c - b * s, a * s + b * c)):
        out[..., at] = z
        err[..., at] = size + u * (z.abs() + size) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    return out, err
