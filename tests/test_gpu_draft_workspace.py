"""The C entry of verify_draft with its results right behind its workspace, of which the caller says that it is larger than it is."""
import ctypes
import os
import sys

import pytest
import torch

from cuda_attn import _native

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import draft_oracle as do  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("vocab", [300, 70001])
def test_results_behind_the_workspace(drawn, vocab):
    tokens, parents, p, u, cu, q = do.drafts([5, 9, 4], vocab, 2, 1, drawn)
    lib, seqs, most = _native.lib(), 3, 9
    need = lib.pa_verify_draft_workspace(seqs, vocab, int(drawn))
    room = torch.zeros(need + 1024, dtype=torch.uint8, device="cuda")
    at = lambda n: ctypes.c_void_p(room.data_ptr() + need + n)  # noqa: E731
    on = [x.cuda() for x in (tokens, parents, p, u, cu)]
    gq = q.cuda() if drawn else None
    ptr = lambda x: None if x is None else ctypes.c_void_p(x.data_ptr())  # noqa: E731
    assert need % 8 == 0
    rc = lib.pa_verify_draft(ptr(on[0]), ptr(on[1]), ptr(on[2]), vocab, ptr(gq), vocab, ptr(on[3]), ptr(on[4]), len(tokens), seqs, vocab, most,
                             at(0), at(512), at(768), ptr(room), 1 << 40, None)
    assert rc == 0, _native.last_error()
    torch.cuda.synchronize()
    out = room[need:].cpu()
    path, accepted, drawn_next = out[:4 * seqs * most].view(torch.int32).view(seqs, most), out[512:512 + 4 * seqs].view(torch.int32), \
        out[768:768 + 8 * seqs].view(torch.int64)
    for a, b in zip((path, accepted, drawn_next), do.verify(tokens, parents, p, u, cu, q, most)):
        assert torch.equal(a, b)
