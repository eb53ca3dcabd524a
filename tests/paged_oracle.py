"""Plain float64 forms of the paged cache operators, on the CPU, and problems to run them on.

Nothing here uses the package. A problem holds the tensors of a call as the caller has them; the oracle reads
the same tensors, whatever is in them."""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
# Half a step of a value's rounding, relative to the value.
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def quantise(x: torch.Tensor, dtype: torch.dtype):
    """Codes and scales of rows x in fp32 arithmetic, the operator's documented formula."""
    x = x.float()
    amax = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    some = finite & (amax >= 2.0 ** -100)
    largest = torch.tensor(LARGEST[dtype])
    one = torch.ones(())
    inv = torch.where(some, largest / torch.where(some, amax, one), torch.zeros(()))
    y = torch.where(finite[..., None], x, torch.zeros(())) * inv[..., None]
    codes = y.round().to(torch.int8) if dtype == torch.int8 else y.to(dtype)
    scale = torch.where(some, amax / largest, torch.zeros(()))
    return codes, torch.where(finite, scale, torch.tensor(math.nan))


@dataclass
class Problem:
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    k_cache: torch.Tensor
    v_cache: torch.Tensor
    table: torch.Tensor
    lengths: torch.Tensor
    cu: torch.Tensor | None
    scales: dict = field(default_factory=dict)

    def to(self, device):
        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return Problem(*(move(t) for t in (self.q, self.k, self.v, self.k_cache, self.v_cache, self.table, self.lengths,
                                           self.cu)), {n: move(t) for n, t in self.scales.items()})

    def cache(self):
        return self.k_cache, self.v_cache, self.table, self.lengths


def make(seqs, *, hq=4, hkv=2, d=64, page=16, dtype=torch.float16, cache=None, seed=0, uniform=False, spare=2,
         qk_scale=1.0, stale=math.nan, columns=None) -> Problem:
    """seqs: [(new tokens, length)]. Slots that hold no token are `stale` (8-bit caches: their scales are)."""
    g = torch.Generator().manual_seed(seed)
    cache = cache or dtype
    need = [-(-max(n, 0) // page) for _, n in seqs]
    pages = sum(need) + spare
    cols = columns or max(1, max(need))
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(seqs), cols), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :min(n, cols)] = order[at:at + n].to(torch.int32)[:cols]
        at += n
    tokens = sum(c for c, _ in seqs)
    draw = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q = (draw(tokens, hq, d) * qk_scale).to(dtype)
    k = (draw(tokens, hkv, d) * qk_scale).to(dtype)
    v = draw(tokens, hkv, d).to(dtype)
    caches, scales = [], {}
    for name in ("k", "v"):
        x = draw(pages, hkv, page, d) * (qk_scale if name == "k" else 1.0)
        x = (x * torch.exp(0.5 * draw(pages, hkv, page, 1))).to(dtype)
        used = torch.zeros(pages, page, dtype=torch.bool)
        for i, (_, n) in enumerate(seqs):
            pos = torch.arange(min(max(n, 0), cols * page))
            used[table[i].long()[pos // page], pos % page] = True
        hole = ~used[:, None].expand(pages, hkv, page)
        if cache in LARGEST:
            codes, scale = quantise(x, cache)
            scale[hole] = stale
            caches.append(codes)
            scales[name + "_scale"] = scale
        else:
            x[hole] = stale
            caches.append(x)
    cu = None if uniform else torch.tensor([0] + [c for c, _ in seqs]).cumsum(0).to(torch.int32)
    return Problem(q, k, v, *caches, table, torch.tensor([n for _, n in seqs], dtype=torch.int32), cu, scales)


def layout(p: Problem, tokens: int):
    """[(first row, count, length)] under the documented clamps."""
    got = []
    for s in range(p.table.shape[0]):
        if p.cu is None:
            each = tokens // p.table.shape[0]
            b, e = s * each, (s + 1) * each
        else:
            b = min(max(int(p.cu[s]), 0), tokens)
            e = min(max(int(p.cu[s + 1]), b), tokens)
        got.append((b, e - b, min(max(int(p.lengths[s]), 0), 2 ** 30)))
    return got


def slot(p: Problem, s: int, pos: int):
    """(page, row) of a position, None if it has none."""
    page = p.k_cache.shape[2]
    if pos < 0 or pos >= p.table.shape[1] * page:
        return None
    at = int(p.table[s, pos // page])
    return (at, pos % page) if 0 <= at < p.k_cache.shape[0] else None


def rows(p: Problem, s: int, n: int):
    """K and V of positions 0 .. n - 1 in float64, (heads, n, d), and which of them have a page."""
    slots = [slot(p, s, i) for i in range(n)]
    here = torch.tensor([x is not None for x in slots], dtype=torch.bool)
    pg = torch.tensor([0 if x is None else x[0] for x in slots], dtype=torch.long)
    rw = torch.tensor([0 if x is None else x[1] for x in slots], dtype=torch.long)
    out = []
    for name in ("k", "v"):
        held = getattr(p, name + "_cache")
        held = held.float() if held.dtype == torch.float8_e4m3fn else held
        x = held[pg, :, rw].double()
        if p.scales:
            x = x * p.scales[name + "_scale"][pg, :, rw].double()[..., None]
        out.append(x.transpose(0, 1))
    return out[0], out[1], here


def written(p: Problem):
    """The caches and scales after cache_write."""
    kc, vc = p.k_cache.clone(), p.v_cache.clone()
    scales = {n: t.clone() for n, t in p.scales.items()}
    for s, (first, count, length) in enumerate(layout(p, p.k.shape[0])):
        for i in range(count):
            at = slot(p, s, length - count + i)
            if at is None:
                continue
            for x, c, name in ((p.k, kc, "k_scale"), (p.v, vc, "v_scale")):
                row = x[first + i]
                if scales:
                    row, scale = quantise(row, c.dtype)
                    scales[name][at[0], :, at[1]] = scale
                if c.dtype == torch.float8_e4m3fn:
                    c.view(torch.int8)[at[0], :, at[1]] = row.view(torch.int8)
                else:
                    c[at[0], :, at[1]] = row
    return kc, vc, scales


def read(p: Problem, n: int):
    """K and V laid out as (B, heads, n, d) in float64; zeros where there is no row."""
    out = []
    for which in (0, 1):
        x = torch.zeros((p.table.shape[0], p.k_cache.shape[1], n, p.k_cache.shape[3]), dtype=torch.float64)
        for s in range(p.table.shape[0]):
            m = min(max(int(p.lengths[s]), 0), n)
            got = rows(p, s, m)
            x[s, :, :m] = torch.where(got[2][None, :, None], got[which], torch.zeros((), dtype=torch.float64))
        out.append(x)
    return out


def attn(p: Problem, causal: bool = True):
    """(output, bound on a kernel's error, rows of exactly one sequence) in float64. (Offsets out of order can
    give a row to two sequences: such a row may hold either's result.)

    The bound counts the roundings of a kernel with 16-bit matrix operands and fp32 sums, u half a step of the
    inputs' type, A = sum_j p_j |v_j| / l:
      * p rounded once to the type: u A; below fp16's normal range an absolute 2^-25 of each p (and, for 8-bit
        caches, of p times the value's scale over the largest scale): 2^-25 sum_j max|v| / l
        (max over the finite values: an output that is a number sums no others)
      * the output rounded: u |o|, or half a subnormal fp16 step
      * scores in fp32: d products summed, |ds| <= (d + 8) 2^-24 sum |q k| / sqrt(d); and 2^-20 for the
        exponentials and the sums; twice, for the numerator and the sum l.
    A second rounding of p as l's summand would be of the same size and is allowed for: 2 u A."""
    tokens, hq, d = p.q.shape
    hkv, page = p.k_cache.shape[1], p.k_cache.shape[2]
    out = torch.zeros(p.q.shape, dtype=torch.float64)
    bound = torch.zeros(p.q.shape, dtype=torch.float64)
    claims = torch.zeros(tokens, dtype=torch.long)
    finite = lambda x: torch.where(torch.isfinite(x), x, torch.zeros((), dtype=x.dtype))  # noqa: E731
    u = HALF_STEP[p.q.dtype]
    for s, (first, count, length) in enumerate(layout(p, tokens)):
        if count == 0:
            continue
        cap = p.table.shape[1] * page
        k, v, here = rows(p, s, min(length, cap))
        claims[first:first + count] += 1
        n = k.shape[1]
        seen = torch.arange(n)[None, :] <= (length - count + torch.arange(count))[:, None] if causal else \
            torch.ones(count, n, dtype=torch.bool)
        seen = seen & here[None, :]
        for h in range(hq):
            kh, vh = k[h // (hq // hkv)], v[h // (hq // hkv)]
            kh = torch.where(here[:, None], kh, torch.zeros((), dtype=torch.float64))
            q = p.q[first:first + count, h].double()
            sc = (q @ kh.t()) / math.sqrt(d)
            sc = torch.where(seen, sc, torch.tensor(-math.inf, dtype=torch.float64))
            some = seen.any(-1)
            top = torch.where(some, sc.amax(-1) if n else torch.zeros(count, dtype=torch.float64), torch.zeros((), dtype=torch.float64))
            w = torch.where(seen, torch.exp(sc - top[:, None]), torch.zeros((), dtype=torch.float64))
            l = torch.where(some, w.sum(-1), torch.ones((), dtype=torch.float64))[:, None]
            for i in range(count):   # rows that see different keys: nothing of an unseen value may reach them
                if some[i]:
                    use = seen[i]
                    out[first + i, h] = (w[i, use] @ vh[use]) / l[i]
                    a = (w[i, use] @ vh[use].abs()) / l[i]
                    size = (q[i].abs() @ kh[use].abs().t()).max() / math.sqrt(d)
                    es = 2 * ((d + 8) * 2.0 ** -24 * size + 2.0 ** -20)
                    low = 2.0 ** -25 * use.sum() * finite(vh[use]).abs().max() / l[i] if p.q.dtype == torch.float16 else 0.0
                    bound[first + i, h] = (2 * u + es) * a + low + u * out[first + i, h].abs() + 2.0 ** -25
    return out, bound, claims == 1
