"""Where paged_attn may write: `out` against q and the call's other tensors (host checks, no GPU)."""
import itertools

import pytest
import torch

from cuda_attn import _checks

F16 = torch.float16


def bytes_of(t):
    """The addresses of a tensor's elements."""
    at = [t.data_ptr() + t.element_size() * sum(i * s for i, s in zip(index, t.stride()))
          for index in itertools.product(*(range(n) for n in t.shape))]
    return set(at)


def accepted(q, out, *others):
    try:
        _checks.check_out("paged_attn", q, out, *others)
    except RuntimeError as e:
        assert "share memory" in str(e)
        return False
    return True


def test_slices_of_one_projection():
    """q and out as heads, or as tokens, of one buffer, in either order."""
    both = torch.zeros(6, 12, 64, dtype=F16)
    assert accepted(both[:, :4], both[:, 4:8])
    assert accepted(both[:, 4:8], both[:, :4])
    assert accepted(both[:, :4], both[:, 8:])
    assert accepted(both[::2, :4], both[1::2, :4])
    assert accepted(both[:, ::2], both[:, 1::2])
    wide = torch.zeros(6, 4, 128, dtype=F16)
    assert accepted(wide[..., :64], wide[..., 64:])
    for a, b in ((both[:, :4], both[:, 3:7]), (both[:, 4:8], both[:, 1:5]), (both[:4, :4], both[2:, :4]), (both, both),
                 (wide[..., :64], wide[..., 8:72]), (wide[..., :64], wide[..., 56:120]), (both[0:5:2, :4], both[2:7:2, :4])):
        if a.shape == b.shape:
            assert not accepted(a, b)


def test_one_token_and_one_head():
    """A stride of a dimension of one does not matter."""
    both = torch.zeros(1, 8, 64, dtype=F16)
    assert accepted(both[:, :4], both[:, 4:])
    assert not accepted(both[:, :4], both[:, 3:7])
    heads = torch.zeros(8, 2, 64, dtype=F16)
    assert accepted(heads[:, :1], heads[:, 1:])
    assert not accepted(heads[:, :1], heads[:, :1])
    one = torch.zeros(3, 64, dtype=F16)
    assert accepted(one[:1].view(1, 1, 64), one[1:2].view(1, 1, 64).as_strided((1, 1, 64), (8, 16, 1), 64))


@pytest.mark.parametrize("seed", range(4))
def test_agrees_with_the_addresses(seed):
    """Slices of one buffer at equal strides: refused iff an element of the one is one of the other."""
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: lo + int(torch.randint(hi - lo + 1, (1,), generator=g))  # noqa: E731
    seen = {True: 0, False: 0}
    for _ in range(150):
        tokens, heads, d = r(1, 4), r(1, 4), 16
        strides = (8 * r(2, 12), 8 * r(2, 12), 1)
        buffer = torch.zeros(4000, dtype=F16)
        a = buffer.as_strided((tokens, heads, d), strides, 8 * r(0, 60))
        b = buffer.as_strided((tokens, heads, d), strides, 8 * r(0, 60))
        try:
            _checks.check_out("paged_attn", a, b)
            ok = True
        except RuntimeError as e:
            if "must not overlap" in str(e):   # (out's own rows)
                continue
            ok = False
        assert ok == bytes_of(a).isdisjoint(bytes_of(b)), (a.shape, strides, a.storage_offset(), b.storage_offset())
        seen[ok] += 1
    assert min(seen.values()) > 10


def test_unlike_strides():
    """Rows of unlike strides must lie apart altogether."""
    buffer = torch.zeros(4096, dtype=F16)
    a = buffer[:1536].view(6, 4, 64)
    assert accepted(a, buffer[1536:3072].view(4, 6, 64).transpose(0, 1))
    assert not accepted(a, buffer[1472:3008].view(4, 6, 64).transpose(0, 1))


def test_the_calls_other_tensors():
    """out over the cache, its scales, the page table, the lengths or the offsets."""
    arena = torch.zeros(1 << 16, dtype=torch.uint8)
    q = torch.zeros(6, 4, 64, dtype=F16)
    size = 2 * q.numel()
    out = arena[4096:4096 + size].view(F16).view(6, 4, 64)
    free = arena[:4096], arena[4096 + size:]
    cache = free[1][:10240].view(torch.int8).view(5, 2, 16, 64)
    assert accepted(q, out, cache, None, free[0][:64].view(torch.int32))
    for at in (4096, 4096 + size - 16, 4080):
        assert not accepted(q, out, arena[at:at + 32].view(torch.int32))
    assert not accepted(q, out, None, arena[1024:1024 + 20480].view(F16).view(5, 2, 16, 64))
    table = arena[:8192].view(torch.int32).view(4, 512)[:, :3]   # (rows of a wider table; the last lie in out)
    assert not accepted(q, out, table)
