"""rope in place beside autograd: what it would not see is refused, and what it has saved is known to have changed."""

import pytest
import torch

import cuda_attn
from cuda_attn import _checks


def check(q, k=None, inplace=True):
    _checks.check_rope("rope", q, k, torch.zeros(6, dtype=torch.int32), torch.ones(8, dtype=torch.float64), inplace, require_cuda=False)


def test_in_place_refuses_tensors_that_require_a_gradient():
    plain, leaf = torch.zeros(6, 4, 64), torch.zeros(6, 4, 64, requires_grad=True)
    for q, k in ((leaf, None), (plain, leaf), (leaf * 2, plain), (plain, leaf[:, :2])):
        with pytest.raises(RuntimeError, match="require a gradient"):
            check(q, k)
        check(q, k, inplace=False)
        with torch.no_grad():
            check(q, k)
    check(plain, torch.zeros(6, 2, 64))


@pytest.mark.gpu
def test_autograd_sees_rows_turned_in_place():
    f, positions = cuda_attn.rope_frequencies(64, device="cuda")[0], torch.arange(6, device="cuda")
    for both in (False, True):
        q, k = torch.randn(6, 4, 64, device="cuda"), torch.randn(6, 2, 64, device="cuda")
        w = torch.ones(64, device="cuda", requires_grad=True)
        kept = (w * (k if both else q)).sum()   # saves the rows for w's gradient
        cuda_attn.rope(q, k if both else None, positions, f, inplace=True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
    with torch.inference_mode():
        q = torch.randn(6, 4, 64, device="cuda")
        want = cuda_attn.rope(q, None, positions, f)[0]
        cuda_attn.rope(q, None, positions, f, inplace=True)
        assert torch.equal(q, want)
    leaf = torch.randn(6, 4, 64, device="cuda", requires_grad=True)
    before = leaf.detach().clone()
    with pytest.raises(RuntimeError, match="require a gradient"):
        cuda_attn.rope(leaf, None, positions, f, inplace=True)
    assert torch.equal(leaf, before) and not cuda_attn.rope(leaf, None, positions, f)[0].requires_grad
