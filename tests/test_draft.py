"""Host-side checks of the operators around drafted tokens (no GPU): refusals, the C entry points' argument checks, the
mask's index arithmetic and the oracle that the GPU tests use."""
import ctypes
import math
import os
import random
import shutil
import subprocess
import sys

import pytest
import torch

import cuda_attn
from cuda_attn import _checks, _native

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
sys.path.insert(0, HERE)
import draft_oracle as do  # noqa: E402

I32, I64 = torch.int32, torch.int64


def ints(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


# ---------------------------------------------------------------- refusals
def test_cpu_tensors_are_refused():
    f16 = torch.float16
    cache = (torch.zeros(5, 2, 16, 64, dtype=f16), torch.zeros(5, 2, 16, 64, dtype=f16), ints(3, 2), ints(3))
    q, probs, cu = torch.zeros(6, 4, 64, dtype=f16), torch.zeros(6, 10), ints(4)
    for call in (lambda: cuda_attn.draft_tree(ints(6), ints(3)), lambda: cuda_attn.paged_tree_attn(q, *cache, ints(6, 1)),
                 lambda: cuda_attn.verify_draft(ints(6, dtype=I64), ints(6), probs, torch.zeros(6), cu),
                 lambda: cuda_attn.cache_keep(*cache, ints(3, 2), ints(3), cu),
                 lambda: cuda_attn.rope(q, None, ints(6), torch.ones(32, dtype=torch.float64))):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()


def tree(parents, seqs, cu=None, max_new=None):
    return _checks.check_tree("draft_tree", parents, seqs, cu, max_new, require_cuda=False)


def test_trees():
    assert tree(ints(6), 3) == 2 and tree(ints(6), 3, ints(4)) == 6 and tree(ints(6), 3, ints(4), 4) == 4
    assert tree(ints(5000), 3, ints(4)) == 1024
    for args, match in (((ints(6, dtype=I64), 3), "parents"), ((ints(6, 2), 3), "parents"), ((ints(12)[::2], 3), "parents"),
                        ((ints(0), 3), "non-empty"), ((ints(6), 0), "non-empty"), ((ints(7), 3), "divide evenly"),
                        ((ints(6), 3, ints(3)), "cu_seqlens"), ((ints(6), 3, ints(4, dtype=I64)), "cu_seqlens"),
                        ((ints(6), 3, torch.zeros(4, dtype=I32, device="meta")), "same device"),
                        ((ints(6), 3, None, 0), "max_new"), ((ints(6), 3, None, 1025), "max_new"), ((ints(6), 3, None, True), "max_new"),
                        ((ints(6), 3, None, 2.0), "max_new"), ((ints(4096), 2), "at most 1024")):
        with pytest.raises(RuntimeError, match=match):
            tree(*args)


def test_masks_probabilities_and_paths():
    q = torch.zeros(6, 4, 64, dtype=torch.float16)
    _checks.check_mask("paged_tree_attn", ints(6, 3), q)
    _checks.check_mask("paged_tree_attn", ints(6, 9)[:, 2:5], q)
    for m, match in ((ints(5, 3), "mask"), (ints(6), "mask"), (ints(6, 0), "mask"), (ints(6, 3, dtype=I64), "mask"), (ints(3, 6).t(), "mask"),
                     (torch.zeros(6, 3, dtype=I32, device="meta"), "same device")):
        with pytest.raises(RuntimeError, match=match):
            _checks.check_mask("paged_tree_attn", m, q)
    both = torch.zeros(64, dtype=I32)
    with pytest.raises(RuntimeError, match="share memory with the mask"):
        _checks.check_no_overlap("paged_tree_attn", both[:40], both[39:], "the mask")
    _checks.check_no_overlap("paged_tree_attn", both[:40], both[40:], "the mask")
    cpu = q.device
    probs = lambda x, vocab=None: _checks.check_probs("verify_draft", "target_probs", x, 6, cpu, vocab, require_cuda=False)  # noqa: E731
    probs(torch.zeros(6, 11))
    probs(torch.zeros(6, 20)[:, 3:14], 11)
    for x, vocab, match in ((torch.zeros(5, 11), None, "target_probs"), (torch.zeros(6, 11).half(), None, "target_probs"),
                            (torch.zeros(11, 6).t(), None, "target_probs"), (torch.zeros(6), None, "target_probs"),
                            (torch.zeros(6, 0), None, "non-empty"), (torch.zeros(6, 11), 12, "one vocabulary"),
                            (torch.zeros(6, 11, device="meta"), None, "same device")):
        with pytest.raises(RuntimeError, match=match):
            probs(x, vocab)
    _checks.check_path("cache_keep", ints(3, 8)[:, :5], 3, cpu)
    for x, match in ((ints(4, 5), "path"), (ints(3), "path"), (ints(3, 0), "path"), (ints(3, 5, dtype=I64), "path"), (ints(5, 3).t(), "path"),
                     (torch.zeros(3, 5, dtype=I32, device="meta"), "same device")):
        with pytest.raises(RuntimeError, match=match):
            _checks.check_path("cache_keep", x, 3, cpu)
    for x, size, match in ((ints(5), 6, "vector of 6"), (ints(6, dtype=I64), 6, "vector"), (ints(12)[::2], 6, "vector"), (ints(0), None, "non-empty")):
        with pytest.raises(RuntimeError, match=match):
            _checks.check_vector("verify_draft", "accepted", x, I32, size, cpu, require_cuda=False)


def rope(q, k=None, positions=None, freqs=None, inplace=False):
    n = q.shape[0] if q.dim() == 3 else q.shape[-2]
    positions = ints(n) if positions is None else positions
    freqs = torch.ones(8, dtype=torch.float64) if freqs is None else freqs
    _checks.check_rope("rope", q, k, positions, freqs, inplace, require_cuda=False)


def test_rope_arguments():
    q, dense = torch.zeros(6, 4, 64), torch.zeros(2, 4, 6, 64)
    rope(q)
    rope(q, torch.zeros(6, 2, 64), ints(6, dtype=I64))
    rope(dense, torch.zeros(2, 1, 6, 64))
    rope(dense, None, ints(2, 6))
    rope(q, None, ints(12)[::2], torch.ones(32, dtype=torch.float64))
    rope(torch.zeros(6, 4, 33))
    f64 = lambda n: torch.ones(n, dtype=torch.float64)  # noqa: E731
    for args, match in (((q[0],), "shaped"), ((q.double(),), "float32, float16 or bfloat16"), ((q.int(),), "float32, float16 or bfloat16"),
                        ((q[:0],), "non-empty"), ((q, torch.zeros(6, 0, 64)), "non-empty"), ((q, q.half()), "share a dtype"),
                        ((q, torch.zeros(5, 4, 64)), "same tokens"), ((q, torch.zeros(6, 4, 32)), "same tokens"), ((q, dense), "same tokens"),
                        ((dense, torch.zeros(2, 4, 7, 64)), "same tokens"), ((torch.zeros(6, 1, 1025),), "up to 1024"),
                        ((q.transpose(1, 2),), "rows must be contiguous"), ((q, None, ints(5)), "positions"), ((q, None, ints(6, 1)), "positions"),
                        ((dense, None, ints(2)), "positions"), ((dense, None, ints(12)), "positions"), ((q, None, torch.zeros(6)), "int32 or int64"),
                        ((q, None, None, torch.ones(8)), "float64"), ((q, None, None, f64(33)), "d / 2"), ((q, None, None, f64(0)), "d / 2"),
                        ((q, None, None, f64(16)[::2]), "float64"), ((q, None, torch.zeros(6, dtype=I32, device="meta")), "same device"),
                        ((torch.zeros(1, 4, 64).expand(6, 4, 64), None, None, None, True), "must not overlap"),
                        ((torch.zeros(6, 1, 64).expand(6, 4, 64), None, None, None, True), "must not overlap"),
                        ((q, q, None, None, True), "share memory"), ((q[:, :3], q[:, 2:], None, None, True), "share memory")):
        with pytest.raises(RuntimeError, match=match):
            rope(*args)


def test_rope_in_place_takes_slices_of_one_projection():
    both = torch.zeros(6, 9, 64)
    rope(both[:, :4], both[:, 4:6], inplace=True)
    rope(both[:, 5:9], both[:, 1:2], inplace=True)
    rope(both[:3], both[3:], inplace=True)
    dense = torch.zeros(2, 6, 9, 64).transpose(1, 2)   # (B, heads, N, d) of a (B, N, heads, d) projection
    rope(dense[:, :4], dense[:, 4:], inplace=True)
    rope(dense[:, 6:], dense[:, 2:6], inplace=True)
    with pytest.raises(RuntimeError, match="share memory"):
        rope(dense[:, :4], dense[:, 3:], inplace=True)
    with pytest.raises(RuntimeError, match="share memory"):
        rope(both[0:4, :4], both[2:6, 1:2], inplace=True)


def test_rope_frequencies():
    f, scale = cuda_attn.rope_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and scale == 1.0
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * p / 64) for p in range(32)], dtype=torch.float64), rtol=1e-14)
    lin, _ = cuda_attn.rope_frequencies(64, scaling="linear", factor=4.0)
    assert torch.allclose(lin, f / 4, rtol=1e-14)
    ntk, _ = cuda_attn.rope_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    smooth, _ = cuda_attn.rope_frequencies(64, scaling="smooth", factor=8.0, original=8192, low=1.0, high=4.0)
    turns = 8192 * f / (2 * math.pi)
    assert torch.allclose(smooth[turns > 4], f[turns > 4], rtol=1e-14) and torch.allclose(smooth[turns < 1], f[turns < 1] / 8, rtol=1e-14)
    between = (turns > 1) & (turns < 4)
    assert between.any() and bool(((smooth < f) & (smooth > f / 8))[between].all())
    parts, scale = cuda_attn.rope_frequencies(64, scaling="parts", factor=16.0, original=4096)
    assert math.isclose(scale, 0.1 * math.log(16) + 1)
    assert torch.allclose(parts[turns / 2 > 40], f[turns / 2 > 40], rtol=1e-14) and math.isclose(float(parts[-1]), float(f[-1]) / 16, rel_tol=1e-12)
    for kw in (dict(dim=63), dict(dim=0), dict(dim=True), dict(dim=64, scaling="other"), dict(dim=64, factor=0.5), dict(dim=64, base=0.0),
               dict(dim=64, scaling="smooth", low=4.0, high=1.0)):
        with pytest.raises(RuntimeError, match="rope_frequencies"):
            cuda_attn.rope_frequencies(**kw)


# ---------------------------------------------------------------- the C entry points
P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)


def refused(rc, want, match):
    assert rc == want and match in _native.last_error(), (rc, _native.last_error())


def test_c_entries_refuse_trees_and_verification():
    lib = _native.lib()
    tree = lambda parents=P, lengths=P, tokens=6, seqs=3, most=4, mask=P, pos=P, cu=P: \
        lib.pa_draft_tree(parents, lengths, cu, tokens, seqs, most, mask, pos, None)  # noqa: E731
    for kw, rc, match in (({"parents": None}, -1, "null"), ({"pos": None}, -1, "null"), ({"tokens": 0}, -1, "non-empty"),
                          ({"seqs": 0}, -1, "non-empty"), ({"tokens": 2 ** 31}, -2, "2^30"), ({"seqs": 2 ** 23}, -2, "2^22"),
                          ({"most": 0}, -1, "max_new"), ({"most": 1025}, -1, "max_new"), ({"tokens": 7, "cu": None}, -1, "divide evenly")):
        refused(tree(**kw), rc, match)
    verify = lambda tokens=P, p=P, u=P, cu=P, n=6, seqs=3, vocab=100000, most=4, path=P, ws=P, room=2 ** 40, ps=100000, qs=0: \
        lib.pa_verify_draft(tokens, P, p, ps, None, qs, u, cu, n, seqs, vocab, most, path, P, P, ws, room, None)  # noqa: E731
    for kw, rc, match in (({"tokens": None}, -1, "null"), ({"p": None}, -1, "null"), ({"u": None}, -1, "null"), ({"cu": None}, -1, "null"),
                          ({"path": None}, -1, "null"), ({"n": 0}, -1, "non-empty"), ({"vocab": 0}, -1, "non-empty"),
                          ({"vocab": 2 ** 25}, -2, "2^24"), ({"seqs": 65536}, -2, "65535"), ({"most": 1025}, -1, "max_new"),
                          ({"ps": -1}, -1, "strides"), ({"qs": -1}, -1, "strides"), ({"ws": None}, -1, "workspace"), ({"ws": ODD}, -1, "workspace"),
                          ({"room": 8}, -1, "workspace"), ({"n": 2 ** 31}, -2, "2^30")):
        refused(verify(**kw), rc, match)
    assert lib.pa_verify_draft_workspace(3, 100, 1) == 0 and lib.pa_verify_draft_workspace(3, 100000, 0) > 0
    assert lib.pa_verify_draft_workspace(0, 100, 0) == -1 and lib.pa_verify_draft_workspace(3, 2 ** 25, 0) == -2


def native_cache(**change):
    c = _native.PagedCacheArgs(256, 256, None, None, 256, 256, 5, 16, 2, 64, 3, 2, 2, _native.DTYPE_F16)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def test_c_entries_refuse_tree_attention_and_keep():
    lib, f16 = _native.lib(), _native.DTYPE_F16
    attn = lambda cache=native_cache(), q=P, mask=P, words=1, stride=1, h=4, room=2 ** 40, ws=P: \
        lib.pa_paged_tree_attn_fwd(cache, q, P, f16, 6, h, 256, 64, 256, 64, None, 0, mask, words, stride, ws, room, None)  # noqa: E731
    for kw, rc, match in (({"cache": None}, -1, "null cache"), ({"q": None}, -1, "null"), ({"mask": None}, -1, "null"), ({"words": 0}, -1, "mask"),
                          ({"words": 2 ** 26}, -1, "mask"), ({"stride": -1}, -1, "mask"), ({"h": 3}, -1, "multiple"), ({"room": 1}, -1, "workspace"),
                          ({"ws": None}, -1, "workspace"), ({"cache": native_cache(d=96)}, -2, "head dimension")):
        refused(attn(**kw), rc, match)
    keep = lambda cache=native_cache(), path=P, width=4, stride=4, acc=P, cu=P, after=P: \
        lib.pa_cache_keep(cache, path, width, stride, acc, cu, after, None)  # noqa: E731
    for kw, rc, match in (({"cache": None}, -1, "null cache"), ({"path": None}, -1, "null"), ({"cu": None}, -1, "null"), ({"after": None}, -1, "null"),
                          ({"width": 0}, -1, "path"), ({"stride": -4}, -1, "path"), ({"cache": native_cache(dtype=_native.DTYPE_I8)}, -1, "k_scale"),
                          ({"cache": native_cache(dtype=_native.DTYPE_F32)}, -2, "float16 or bfloat16"), ({"cache": native_cache(pages=0)}, -1, "non-empty")):
        refused(keep(**kw), rc, match)


def test_c_entries_refuse_rope():
    lib, f16 = _native.lib(), _native.DTYPE_F16
    rows = lambda **kw: _native.RopeRows(*(kw.get(n, v) for n, v in zip(  # noqa: E731
        ("i", "o", "ib", "inn", "ih", "ob", "on", "oh", "heads"), (256, 256, 0, 256, 64, 0, 256, 64, 4))))
    ref = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    rope = lambda q=rows(), k=None, dt=f16, b=1, n=6, d=64, pos=P, f=P, pairs=32: \
        lib.pa_rope(ref(q), ref(k), dt, b, n, d, pos, 0, 0, 1, f, pairs, 0, 0, 1.0, None)  # noqa: E731
    for kw, rc, match in (({"q": None}, -1, "null"), ({"pos": None}, -1, "null"), ({"f": None}, -1, "null"), ({"q": rows(i=None)}, -1, "null"),
                          ({"k": rows(o=None)}, -1, "null"), ({"dt": _native.DTYPE_I8}, -2, "float32"), ({"n": 0}, -1, "non-empty"),
                          ({"pairs": 0}, -1, "non-empty"), ({"d": 2048}, -2, "1024"), ({"pairs": 33}, -1, "more pairs"), ({"b": 2 ** 20, "n": 2 ** 20}, -2, "2^30"),
                          ({"q": rows(heads=0)}, -1, "heads"), ({"k": rows(ih=-64)}, -1, "negative"), ({"q": rows(i=257)}, -1, "aligned")):
        refused(rope(**kw), rc, match)


def test_mask_window(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    exe = tmp_path / "mask_window_check"
    build = subprocess.run([hipcc, "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                            "-packed-fp32-ops", "-I", os.path.join(REPO, "phantom-a100_amd", "csrc"),
                            os.path.join(HERE, "native", "mask_window_check.cpp"), "-o", str(exe)],
                           capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr


# ---------------------------------------------------------------- the oracle
def test_oracle_masks():
    parents = torch.tensor([-1, 0, 0, 1, 3, 7, -5], dtype=I32)   # 5's is no earlier token
    masks, positions = do.draft_tree(parents, torch.tensor([20]), torch.tensor([0, 7]), 6)
    assert masks == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 3, 4}, {5}, set()]
    assert positions == [13, 14, 14, 15, 16, 13, 13]
    assert do.words([{0, 31, 33}, None], 2).tolist() == [[-2 ** 31 + 1, 2], [0, 0]]


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("branch", [1, 3])
def test_oracle_keeps_the_targets_distribution(drawn, branch):
    """The token behind the root, accepted draft or drawn, has the target's distribution whatever the drafts are: 8000
    sequences, each count within five standard deviations of its mean."""
    n, vocab, runs, width = 4, 5, 8000, 1 + branch
    g = torch.Generator().manual_seed(branch)
    p, q = torch.softmax(torch.randn(vocab, generator=g), -1), torch.softmax(torch.randn(vocab, generator=g), -1)
    tokens = torch.zeros(runs, width, dtype=I64)
    if drawn:
        tokens[:, 1:] = torch.multinomial(q.expand(runs, vocab), branch, replacement=True, generator=g)
    else:
        tokens[:, 1:] = torch.argsort(q, descending=True)[:branch]
    parents = torch.tensor([-1] + [0] * branch, dtype=I32).repeat(runs)
    cu = torch.arange(0, runs * width + 1, width, dtype=I32)
    rows = p.expand(runs * width, vocab)
    path, kept, nxt = do.verify(tokens.view(-1), parents, rows, torch.rand(runs * width, generator=g), cu,
                                q.expand(runs * width, vocab) if drawn else None, n)
    first = torch.where(kept > 1, tokens[torch.arange(runs), path[:, 1].long().clamp(min=0)], nxt)
    count = torch.bincount(first, minlength=vocab).double()
    mean = runs * p.double()
    assert bool(((count - mean).abs() <= 5 * (mean * (1 - p.double())).sqrt()).all()), (count, mean)


def test_oracle_verification_by_hand():
    p = torch.tensor([[0.5, 0.25, 0.25], [0.0, 1.0, 0.0], [0.25, 0.5, 0.25]])
    tokens, parents, cu = torch.tensor([9, 0, 2]), torch.tensor([-1, 0, 0], dtype=I32), torch.tensor([0, 3], dtype=I32)
    u = lambda *x: torch.tensor(x)  # noqa: E731
    path, kept, nxt = do.verify(tokens, parents, p, u(0.9, 0.49, 0.0), cu)     # 0.49 < 0.5: the first draft
    assert path[0, :3].tolist() == [0, 1, -1] and int(kept) == 2 and int(nxt) == 1
    path, kept, nxt = do.verify(tokens, parents, p, u(0.9, 0.5, 0.49), cu)     # rejected; 0.49 * 0.5 < 0.25: the second
    assert path[0, :3].tolist() == [0, 2, -1] and int(nxt) == 2
    path, kept, nxt = do.verify(tokens, parents, p, u(0.9, 0.5, 0.5), cu)      # both rejected: only token 1 is left
    assert int(kept) == 1 and int(nxt) == 1
    q = torch.tensor([[0.75, 0.125, 0.125]] * 3)
    path, kept, nxt = do.verify(tokens, parents, p, u(0.6, 0.66, 0.0), cu, q)  # 0.66 * 0.75 < 0.5
    assert path[0, :2].tolist() == [0, 1]
    path, kept, nxt = do.verify(tokens, parents, p, u(0.6, 0.67, 0.99), cu, q)   # rejected: left is (0, 1/2, 1/2), q(2) = 1/8
    assert path[0, :2].tolist() == [0, 2]


def test_oracle_rope_turns_by_the_angle():
    x = torch.randn(3, 2, 8, generator=torch.Generator().manual_seed(1))
    f = torch.tensor([1.0, 0.25], dtype=torch.float64)
    y, _ = do.rope(x, torch.tensor([0, 1, 5]), f)
    assert torch.equal(y[0], x[0].double()) and torch.equal(y[..., 4:], x[..., 4:].double())
    a, b = x[2, 1, 1].double(), x[2, 1, 3].double()
    assert math.isclose(float(y[2, 1, 1]), float(a * math.cos(1.25) - b * math.sin(1.25)), rel_tol=1e-12)
    z, _ = do.rope(x, torch.tensor([0, 1, 5]), f, interleaved=True)
    assert math.isclose(float(z[1, 0, 3]), float(x[1, 0, 2].double() * math.sin(0.25) + x[1, 0, 3].double() * math.cos(0.25)), rel_tol=1e-12)
    back, _ = do.rope(y.float(), torch.tensor([0, 1, 5]), f, inverse=True)
    assert torch.allclose(back, x.double(), atol=1e-6)


@pytest.mark.parametrize("change", [
    {}, {"parents": ints(6, dtype=I64)}, {"parents": ints(12)[::2]}, {"parents": ints(0)}, {"tokens": ints(5, dtype=I64)}, {"tokens": ints(6)},
    {"uniform": torch.zeros(6).double()}, {"uniform": torch.zeros(12)[::2]}, {"cu": ints(4, dtype=I64)}, {"cu": ints(8)[::2]}, {"most": 0},
    {"most": 1025}, {"most": True}, {"most": 2.0}, {"p": torch.zeros(5, 9)}, {"p": torch.zeros(6, 9).half()}, {"p": torch.zeros(9, 6).t()},
    {"p": torch.zeros(6, 0)}, {"q": torch.zeros(6, 8)}, {"q": torch.zeros(6, 9).double()}, {"q": None}, {"p": torch.zeros(6, 20)[:, 3:12]},
    {"parents": torch.zeros(6, dtype=I32, device="meta")}, {"q": torch.zeros(6, 9, device="meta")}])
def test_one_pass_acceptance_agrees_with_the_checks(change):
    """trees_ok and probs_ok accept what the checks one by one accept (on CPU tensors that say they are on the GPU)."""
    class OnGpu(torch.Tensor):
        is_cuda = True
    t = {"parents": ints(6), "tokens": ints(6, dtype=I64), "uniform": torch.zeros(6), "cu": ints(4), "p": torch.zeros(6, 9), "q": torch.zeros(6, 9)}
    t.update({n: x for n, x in change.items() if n != "most"})
    t = {n: x if x is None else x.as_subclass(OnGpu) for n, x in t.items()}
    most = change.get("most", 4)

    def one_by_one():
        try:
            device, n = t["parents"].device, t["parents"].shape[0]
            _checks.check_tree("verify_draft", t["parents"], 3, t["cu"], most)
            _checks.check_vector("verify_draft", "tokens", t["tokens"], I64, n, device)
            _checks.check_vector("verify_draft", "uniform", t["uniform"], torch.float32, n, device)
            _checks.check_probs("verify_draft", "target_probs", t["p"], n, device)
            if t["q"] is not None:
                _checks.check_probs("verify_draft", "draft_probs", t["q"], n, device, t["p"].shape[1])
        except RuntimeError:
            return False
        return True
    shape = t["parents"].shape
    ok = _checks.trees_ok(t["parents"], ((t["tokens"], I64, shape), (t["uniform"], torch.float32, shape), (t["cu"], I32, torch.Size([4]))), most) and all(
        x is None or _checks.probs_ok(x, shape[0], t["parents"].device, t["p"].shape[1]) for x in (t["p"], t["q"]))
    assert ok == one_by_one(), change


@pytest.mark.parametrize("change", [
    {}, {"k": None}, {"q": torch.zeros(6, 4, 64, dtype=torch.float64)}, {"q": torch.zeros(6, 4)}, {"q": torch.zeros(0, 4, 64)},
    {"q": torch.zeros(6, 64, 4).transpose(1, 2)}, {"k": torch.zeros(6, 2, 32)}, {"k": torch.zeros(5, 2, 64)}, {"k": torch.zeros(6, 2, 64).half()},
    {"positions": ints(5)}, {"positions": torch.zeros(6)}, {"positions": ints(12)[::2]}, {"positions": ints(6, dtype=I64)}, {"freqs": torch.ones(33, dtype=torch.float64)},
    {"freqs": torch.ones(8)}, {"freqs": torch.ones(16, dtype=torch.float64)[::2]}, {"freqs": torch.ones(0, dtype=torch.float64)},
    {"q": torch.zeros(2, 4, 6, 64), "k": torch.zeros(2, 1, 6, 64)}, {"q": torch.zeros(2, 4, 6, 64), "k": None, "positions": ints(2, 6)},
    {"q": torch.zeros(2, 4, 6, 64), "k": None, "positions": ints(6, 2)}, {"k": torch.zeros(6, 2, 64, device="meta")}])
def test_one_pass_acceptance_of_rope_agrees_with_its_check(change):
    class OnGpu(torch.Tensor):
        is_cuda = True
    t = {"q": torch.zeros(6, 4, 64), "k": torch.zeros(6, 2, 64), "positions": ints(6), "freqs": torch.ones(16, dtype=torch.float64)}
    t.update(change)
    t = {n: x if x is None else x.as_subclass(OnGpu) for n, x in t.items()}
    try:
        _checks.check_rope("rope", t["q"], t["k"], t["positions"], t["freqs"], False)
        fine = True
    except RuntimeError:
        fine = False
    assert _checks.rope_ok(t["q"], t["k"], t["positions"], t["freqs"]) == fine


@pytest.mark.parametrize("dtype,d,new,rows,wgs", [
    ("f16", 128, 4, 16, 512), ("f16", 128, 8, 32, 256), ("f16", 128, 9, 128, 256), ("f16", 128, 16, 128, 256), ("f16", 128, 17, 128, 256),
    ("f16", 128, 32, 128, 256), ("f16", 128, 33, 256, 256), ("f16", 128, 200, 256, 256), ("f16", 64, 8, 32, 512), ("f16", 64, 17, 128, 512),
    ("f16", 64, 64, 128, 512), ("i8", 128, 8, 32, 512), ("i8", 128, 17, 128, 512), ("i8", 128, 64, 256, 256), ("i8", 64, 17, 128, 512)])
def test_rows_of_a_tile(dtype, d, new, rows, wgs):
    """The tile that a call of long sequences takes (4 query heads a key/value head), by the workspace that it asks for."""
    lib = _native.lib()
    c = native_cache(heads=8, d=d, seqs=32, pages=40000, page_size=16, table_cols=40000, table_stride=40000)
    if dtype == "i8":
        c.dtype, c.k_scale, c.v_scale = _native.DTYPE_I8, 256, 256
    need = lib.pa_paged_tree_attn_workspace(c, _native.DTYPE_F16, 32 * new, 32, P, new)
    assert need == -(-wgs * 16 // 256) * 256 + wgs * 2 * rows * (d + 2) * 4, (need - wgs * 16) / (wgs * 2 * (d + 2) * 4)
    # short ones: as few as there are
    c.table_cols = 20
    assert lib.pa_paged_tree_attn_workspace(c, _native.DTYPE_F16, 32 * new, 32, P, new) <= max(need + 256 * 16, wgs * (16 + 64 * (d + 2) * 4) + 256)
