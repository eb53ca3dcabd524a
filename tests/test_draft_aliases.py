"""Results of the operators around drafted tokens that share memory with what a call reads are refused (no GPU): other
workgroups may read it after it has been written."""
import ctypes

import pytest

from cuda_attn import _native

V = ctypes.c_void_p
MB = 1 << 20


def cache(**change):
    c = _native.PagedCacheArgs(1 * MB, 2 * MB, None, None, 3 * MB, 4 * MB, 5, 16, 2, 64, 3, 2, 2, _native.DTYPE_F16)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def keep(after, c=cache(), path=5 * MB, stride=4, accepted=6 * MB, cu=7 * MB, width=4):
    return _native.lib().pa_cache_keep(c, V(path), width, stride, V(accepted), V(cu), V(after), None)


ROWS = 5 * 2 * 16   # pages x heads x rows of a page


@pytest.mark.parametrize("after", [4 * MB, 4 * MB + 8, 4 * MB - 8, 6 * MB, 6 * MB + 8, 7 * MB + 12, 5 * MB + 44, 5 * MB - 8, 3 * MB + 20,
                                   1 * MB, 1 * MB + ROWS * 128 - 4, 2 * MB + 64])
def test_keep_refuses_new_lengths_over_what_it_reads(after):
    assert keep(after) == -1 and "new_lengths must share no memory" in _native.last_error()


@pytest.mark.parametrize("after", [8 * MB, 8 * MB + ROWS * 4 - 4, 9 * MB])
def test_keep_refuses_new_lengths_over_scales(after):
    c = cache(dtype=_native.DTYPE_I8, k_scale=8 * MB, v_scale=9 * MB)
    assert keep(after, c) == -1 and "new_lengths must share no memory" in _native.last_error()


def test_keep_refuses_new_lengths_between_rows_of_a_path():
    assert keep(5 * MB + 1000 * 4, stride=900) == -1 and "new_lengths must share no memory" in _native.last_error()
    assert keep(2 ** 50, stride=2 ** 62) == -1 and "new_lengths must share no memory" in _native.last_error()


def tree(mask=1 * MB, positions=2 * MB, parents=3 * MB, lengths=4 * MB, cu=5 * MB):
    return _native.lib().pa_draft_tree(V(parents), V(lengths), V(cu), 100, 3, 40, V(mask), V(positions), None)


@pytest.mark.parametrize("where", [{"positions": 3 * MB}, {"positions": 3 * MB + 396}, {"positions": 4 * MB + 8}, {"positions": 5 * MB + 12},
                                   {"mask": 3 * MB - 796}, {"mask": 4 * MB}, {"mask": 2 * MB - 4}, {"positions": 1 * MB + 796}])
def test_draft_tree_refuses_results_over_what_it_reads(where):
    assert tree(**where) == -1 and "share no memory" in _native.last_error()


def verify(path=1 * MB, accepted=2 * MB, drawn=3 * MB, ws=4 * MB, vocab=100000, q=None, stride=100000):
    return _native.lib().pa_verify_draft(V(10 * MB), V(11 * MB), V(100 * MB), stride, q and V(q), stride, V(12 * MB), V(13 * MB), 20, 3, vocab, 8,
                                         V(path), V(accepted), V(drawn), ws and V(ws), 1 << 16, None)


@pytest.mark.parametrize("where", [{"path": 10 * MB + 152}, {"path": 11 * MB}, {"path": 11 * MB - 92}, {"accepted": 12 * MB + 76}, {"drawn": 13 * MB + 8},
                                   {"path": 100 * MB + 8000000 - 16}, {"path": 300 * MB, "q": 300 * MB}, {"accepted": 1 * MB + 92}, {"drawn": 2 * MB + 8},
                                   {"ws": 11 * MB}, {"ws": 1 * MB + 64}, {"path": 100 * MB + 16, "vocab": 100, "stride": 0}])
def test_verify_draft_refuses_results_over_what_it_reads(where):
    assert verify(**where) == -1 and "share no memory" in _native.last_error()
