"""What the serving operators over a paged key/value cache are measured on: listed cases and a generator of more.

Three operators: `cache_write` puts the keys and values of new tokens into pages, as they are or in 8 bits
with a scale for each token and head; `cache_read` lays a batch's pages out as the (B, H, N, d) tensors that
the other entry points take; `paged_attn` is the attention of each sequence's new tokens, one or a chunk of
them, over its pages. With `own` false the same results come from elementary torch operations in 32 bits.
Sizes are generic ones around this package's head dims (64 and 128), its head counts (16 and 32) and the row
lengths of its benchmark configurations.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_LARGEST = {"int8": 127.0, "e4m3": 448.0}
_TINY = 2.0 ** -100   # a token whose largest magnitude is below this is held as zeros in 8 bits


def _case(op, dtype, cache, s, hq, hkv, d, page, new, ctx, ragged=False, causal=True, name=None):
    """s sequences of `ctx` tokens before the call and `new` new ones (ragged: up to so many each)."""
    c = {"op": op, "dtype": dtype, "cache": cache, "s": s, "hq": hq, "hkv": hkv, "d": d, "page": page,
         "new": new, "ctx": ctx, "ragged": ragged, "causal": causal}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # One generation step's keys and values of 32 users: a handful of rows, where latency counts.
        _case("write", "bf16", "bf16", 32, 32, 8, 128, 16, 1, 700, ragged=True, name="write_bf16_32x1"),
        # A batch of prompts' keys and values as they are, chunks of odd lengths behind what is there.
        _case("write", "f16", "f16", 8, 16, 16, 64, 64, 2048, 500, ragged=True, name="write_f16_d64_8x2048"),
        # Prompts quantised into an int8 cache and laid out again for the dense entry points.
        _case("write_read", "bf16", "int8", 4, 32, 8, 128, 16, 4096, 0, ragged=True, name="write_read_int8_4x4096"),
        # The same for one short prompt in e4m3: a call where latency counts.
        _case("write_read", "f16", "e4m3", 1, 16, 16, 64, 32, 333, 0, name="write_read_e4m3_1x333"),
        # Long contexts of many users taken out of an e4m3 cache (moved, or attended by a dense kernel).
        _case("read", "bf16", "e4m3", 16, 32, 8, 128, 16, 0, 8192, ragged=True, name="read_e4m3_16x8192"),
        # One user's next token over a short context: the smallest attention call.
        _case("attn", "bf16", "bf16", 1, 32, 8, 128, 16, 1, 1030, name="attn_bf16_1x1_over_1031"),
        # One generation step of a busy server: a token each over contexts of all lengths.
        _case("attn", "bf16", "bf16", 64, 32, 8, 128, 16, 1, 8192, ragged=True, name="attn_bf16_64x1_over_8192"),
        # The same with few key/value heads and the cache in e4m3.
        _case("attn", "f16", "e4m3", 32, 32, 4, 128, 64, 1, 16384, ragged=True, name="attn_e4m3_32x1_over_16384"),
        # Verification of a few proposed tokens for each user, the cache in int8.
        _case("attn", "f16", "int8", 16, 16, 4, 64, 16, 5, 4096, ragged=True, name="attn_int8_d64_16x5_over_4096"),
        # A scheduler's mixed step: single tokens and chunks of prompts in one call.
        _case("attn", "bf16", "e4m3", 24, 32, 8, 128, 32, 700, 4096, ragged=True, name="attn_e4m3_mixed_24x700"),
        # Whole prompts at once, no context, one key/value head for each query head.
        _case("attn", "f16", "f16", 4, 16, 16, 64, 64, 2048, 0, name="attn_f16_d64_4x2048"),
        # A large chunk of a long document: the largest call.
        _case("attn", "bf16", "bf16", 1, 32, 8, 128, 16, 4096, 28672, name="attn_bf16_1x4096_over_32768"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random):
    op = rng.choices(["write", "write_read", "read", "attn"], [2, 2, 2, 8])[0]
    dtype = rng.choice(["f16", "bf16"])
    cache = rng.choice(["int8", "e4m3"]) if op == "write_read" else rng.choice([dtype, dtype, "int8", "e4m3"])
    if op == "write":
        cache = dtype   # (written in 8 bits: read back by write_read)
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8, 16])
    hq = hkv * rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if g * hkv <= 64])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    ragged = rng.random() < 0.7
    causal = op != "attn" or rng.random() < 0.85
    if op != "attn":
        tokens = _spread(rng, 1, 32768)
        s = _spread(rng, 1, min(64, tokens))
        per = max(1, tokens // s)
        if op == "read":
            return _case(op, dtype, cache, s, hq, hkv, d, page, 0, per, ragged)
        return _case(op, dtype, cache, s, hq, hkv, d, page, per, 0 if op == "write_read" else _spread(rng, 1, 2000), ragged)
    form = rng.choice(["single", "single", "few", "chunk", "chunk", "prompt"])
    new = {"single": 1, "few": rng.randint(2, 16), "chunk": _spread(rng, 17, 4096), "prompt": _spread(rng, 1, 4096)}[form]
    ctx = 0 if form == "prompt" else _spread(rng, 1, 32768)
    # At most 2^27 cached elements, 2^40 operations and 2^32 scores over the padded batch.
    pad = float(new + ctx)
    most = min(128.0, 2.0 ** 27 / (pad * hkv * d), 2.0 ** 40 / (4.0 * new * pad * hq * d), 2.0 ** 32 / (new * pad * hq))
    s = _spread(rng, 1, max(1, int(most)))
    return _case("attn", dtype, cache, s, hq, hkv, d, page, new, ctx, ragged, causal)


def _lengths(case):
    """[(new tokens, tokens after the call)] of each sequence; the same for every seed."""
    rng = random.Random("%(s)d %(new)d %(ctx)d %(page)d" % case)
    got = []
    for i in range(case["s"]):
        new, ctx = case["new"], case["ctx"]
        if case["ragged"]:
            ctx = rng.randint(ctx // 16, ctx) if i else ctx
            if new > 16:   # a third single tokens beside a context, the others chunks of any length
                new = 1 if ctx and rng.random() < 0.34 and i else rng.randint(max(1, new // 4), new)
            elif new > 1:
                new = rng.randint(1, new) if i else new
        got.append((new, new + ctx))
    return got


def _draw_rows(shape, g, spread=0.0):
    x = torch.randn(shape, device="cuda", generator=g)
    if spread:   # tokens of unlike size, as keys and values of a network are
        x *= torch.exp(spread * torch.randn(shape[:-1] + (1,), device="cuda", generator=g))
    return x


def _quantise(x, kind):
    """x in 8 bits and the scale of each row, in 32 bits: scale = amax / largest, code = round(x * (largest / amax))."""
    most = _LARGEST[kind]
    amax = x.abs().amax(-1, keepdim=True)
    some = amax >= _TINY
    code = x * torch.where(some, most / amax, torch.zeros_like(amax))
    code = code.round().to(torch.int8) if kind == "int8" else code.to(torch.float8_e4m3fn)
    return code, torch.where(some, amax / most, torch.zeros_like(amax)).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, cache, page, d = _DTYPES[case["dtype"]], case["cache"], case["page"], case["d"]
    lens = _lengths(case)
    total = sum(n for n, _ in lens)
    pages_of = [-(-n // page) for _, n in lens]
    columns, pages = max(pages_of), sum(pages_of) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((case["s"], columns), -1, dtype=torch.int32)
    at = 0
    host_order = order.cpu()
    for i, n in enumerate(pages_of):
        table[i, :n] = host_order[at:at + n]
        at += n
    cu = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32)
    uniform = len({n for n, _ in lens}) == 1
    st = {"case": case, "table": table.cuda(), "lengths": torch.tensor([n for _, n in lens], dtype=torch.int32).cuda(),
          "cu": cu.cuda(), "uniform": uniform, "max_new": max(n for n, _ in lens), "max_len": max(n for _, n in lens),
          "k_scale": None, "v_scale": None, "dtype": dtype}
    shape = (pages, case["hkv"], page, d)
    for name in ("k", "v"):
        if case["op"] in ("write", "write_read"):
            held = torch.zeros(shape, dtype=_DTYPES[cache], device="cuda")
            scale = torch.zeros(shape[:3], device="cuda") if cache in _LARGEST else None
        else:
            x = _draw_rows(shape, g, 0.3)
            held, scale = _quantise(x.to(dtype).float(), cache) if cache in _LARGEST else (x.to(dtype), None)
        st[name + "_cache"], st[name + "_scale"] = held, scale
    if case["op"] in ("write", "write_read"):
        # keys and values as slices of one projection's output
        both = _draw_rows((total, 2 * case["hkv"], d), g, 0.3).to(dtype)
        st["k"], st["v"] = both[:, :case["hkv"]], both[:, case["hkv"]:]
    elif case["op"] == "attn":
        st["q"] = _draw_rows((total, case["hq"], d), g).to(dtype)
    return st


# ---------------------------------------------------------------- the plain forms
def _rows_of(st, total):
    """For each new token its sequence and its index among that sequence's new tokens."""
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(st["cu"][1:].long(), row, right=True)
    return seq, row - st["cu"].long()[seq]


def _plain_write(st):
    cu, page = st["cu"].long(), st["case"]["page"]
    seq, tok = _rows_of(st, st["k"].shape[0])
    pos = st["lengths"].long()[seq] - (cu[1:] - cu[:-1])[seq] + tok
    at = st["table"].long()[seq, pos // page], pos % page
    for name in ("k", "v"):
        x = st[name]
        if st[name + "_scale"] is not None:
            x, scale = _quantise(x.float(), st["case"]["cache"])
            st[name + "_scale"].transpose(1, 2)[at] = scale
            if x.dtype != torch.int8:   # (moved as bytes)
                st[name + "_cache"].view(torch.int8).transpose(1, 2)[at] = x.view(torch.int8)
                continue
        st[name + "_cache"].transpose(1, 2)[at] = x


def _plain_rows(st, name, n):
    """The first n cached rows of every sequence, (S, H, n, d) in 32 bits; zeros behind its last token."""
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
    if c["causal"]:
        new = (st["cu"][1:] - st["cu"][:-1]).long()
        seen = (lens - new)[:, None] + torch.arange(n, device="cuda") + 1
    else:
        seen = lens[:, None].expand(-1, n)
    hidden = key >= torch.minimum(seen, lens[:, None])[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    p /= p.sum(-1, keepdim=True)
    out = p.view(c["s"], c["hkv"], group * n, length) @ _plain_rows(st, "v", length)
    out = out.view(c["s"], c["hkv"], group, n, d).permute(0, 3, 1, 2, 4)
    return out[seq, tok].reshape(total, hq, d).to(q.dtype)


def _plain(st):
    op = st["case"]["op"]
    if op == "attn":
        return _plain_attn(st)
    if op != "read":
        _plain_write(st)
    if op == "write":
        return {"k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    got = {name: _plain_rows(st, name, st["max_len"]).to(st["dtype"]) for name in ("k", "v")}
    if op == "write_read":
        got.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    return got


# ---------------------------------------------------------------- the framework's operators
if os.path.isdir(os.path.join(os.getcwd(), "phantom-a100_amd")) and os.path.join(os.getcwd(), "phantom-a100_amd") not in sys.path:
    sys.path.insert(0, os.path.join(os.getcwd(), "phantom-a100_amd"))


def _own(st):
    import cuda_attn

    op, cu = st["case"]["op"], None if st["uniform"] else st["cu"]
    scales = {} if st["k_scale"] is None else {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if op == "attn":
        return cuda_attn.paged_attn(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lengths"], cu,
                                    causal=st["case"]["causal"], max_new=st["max_new"], **scales)
    if op != "read":
        cuda_attn.cache_write(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["lengths"], cu, **scales)
    if op == "write":
        return {"k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    k, v = cuda_attn.cache_read(st["k_cache"], st["v_cache"], st["table"], st["lengths"], max_len=st["max_len"],
                                dtype=st["dtype"], **scales)
    got = {"k": k, "v": v}
    if op == "write_read":
        got.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    return got


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    """Each visible row of the cache read once, each new row read or written once; 4 d operations per visible
    (query, key) pair of a head."""
    lens = _lengths(case)
    new, length = sum(n for n, _ in lens), sum(n for _, n in lens)
    row = {"f16": 2, "bf16": 2, "int8": 1, "e4m3": 1}[case["cache"]] * case["d"] + (4 if case["cache"] in _LARGEST else 0)
    if case["op"] == "attn":
        if case["causal"]:
            pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in lens)
        else:
            pairs = sum(n * t for n, t in lens)
        return {"bytes": 2 * length * case["hkv"] * row + 2 * 2 * new * case["hq"] * case["d"],
                "flops": 4 * pairs * case["hq"] * case["d"]}
    got = 0
    if case["op"] != "read":
        got += 2 * new * case["hkv"] * (2 * case["d"] + row)
    if case["op"] != "write":   # (the rows behind a sequence's last are written as zeros)
        got += 2 * case["hkv"] * (length * row + len(lens) * max(t for _, t in lens) * 2 * case["d"])
    return {"bytes": got, "flops": 0}


# ---------------------------------------------------------------- 64 bits
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


def _exact_round(x, kind):
    """Rows of x as their 8 bits stand for them, and their scales, in 64 bits."""
    most = _LARGEST[kind]
    top = x.abs().max(-1, keepdim=True).values
    top = torch.where(top < _TINY, torch.zeros_like(top), top)
    y = torch.where(top > 0, x / torch.where(top > 0, top, torch.ones_like(top)) * most, torch.zeros_like(x))
    if kind == "int8":
        y = torch.round(y)
    else:   # e4m3: 3 bits behind the leading one, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = torch.round(y / step) * step
    return y * (top / most), (top / most).squeeze(-1)


def exact(case, seed):
    st = prepare(case, seed)
    lens = _lengths(case)
    if case["op"] == "write":   # each row behind the ones that its sequence had
        got = {}
        for name in ("k", "v"):
            held = st[name + "_cache"].double()
            first = 0
            for i, (new, length) in enumerate(lens):
                pos = torch.arange(length - new, length, device="cuda")
                held[st["table"][i].long()[pos // case["page"]], :, pos % case["page"]] = st[name][first:first + new].double()
                first += new
            got[name + "_cache"] = held
        return got
    if case["op"] == "attn":
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        group, first = case["hq"] // case["hkv"], 0
        for i, (new, length) in enumerate(lens):
            k, v = _exact_cached(st, "k", i), _exact_cached(st, "v", i)
            key = torch.arange(length, device="cuda")
            for h in range(case["hq"]):
                kt = k[h // group].t().contiguous()
                for r in range(0, new, 2048):
                    m = min(2048, new - r)
                    s = st["q"][first + r:first + r + m, h].double() @ kt / math.sqrt(case["d"])
                    if case["causal"]:
                        last = length - new + torch.arange(r, r + m, device="cuda")
                        s = s.masked_fill(key[None, :] > last[:, None], -math.inf)
                    out[first + r:first + r + m, h] = torch.softmax(s, dim=-1) @ v[h // group]
            first += new
        return out
    got = {}
    width = max(t for _, t in lens)
    for name in ("k", "v"):
        got[name] = torch.zeros((case["s"], case["hkv"], width, case["d"]), dtype=torch.float64, device="cuda")
        if case["op"] == "read":
            for i, (_, length) in enumerate(lens):
                got[name][i, :, :length] = _exact_cached(st, name, i)
            continue
        scale = torch.zeros(st[name + "_scale"].shape, dtype=torch.float64, device="cuda")
        first = 0
        for i, (new, length) in enumerate(lens):
            rows, sizes = _exact_round(st[name][first:first + new].double(), case["cache"])
            got[name][i, :, length - new:length] = rows.transpose(0, 1)
            pos = torch.arange(length - new, length, device="cuda")
            scale[st["table"][i].long()[pos // case["page"]], :, pos % case["page"]] = sizes
            first += new
        got[name + "_scale"] = scale
    return got
