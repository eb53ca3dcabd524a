"""Host-side checks of the paged cache operators (no GPU): refusals, the C entry points' argument checks, the
index arithmetic of the kernels and the oracle that the GPU tests use."""
import ctypes
import math
import os
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
import paged_oracle as po  # noqa: E402


def tensors(dtype=torch.float16, cache=None, d=64, hkv=2):
    cache = cache or dtype
    t = {"rows": torch.zeros(6, 4, d, dtype=dtype), "k_cache": torch.zeros(5, hkv, 16, d, dtype=cache),
         "v_cache": torch.zeros(5, hkv, 16, d, dtype=cache), "page_table": torch.zeros(3, 2, dtype=torch.int32),
         "lengths": torch.zeros(3, dtype=torch.int32), "k_scale": None, "v_scale": None}
    if cache in _checks.EIGHT_BIT:
        t["k_scale"], t["v_scale"] = torch.zeros(5, hkv, 16), torch.zeros(5, hkv, 16)
    return t


def paged(**t):
    _checks.check_paged("paged_attn", **t, require_cuda=False)


def test_cpu_tensors_are_refused():
    t = tensors()
    cache = (t["k_cache"], t["v_cache"], t["page_table"], t["lengths"])
    for call in (lambda: cuda_attn.paged_attn(t["rows"], *cache), lambda: cuda_attn.cache_read(*cache),
                 lambda: cuda_attn.cache_write(t["rows"][:, :2], t["rows"][:, 2:], *cache)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cache", [None, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("d", [64, 128])
def test_valid_caches_pass(dtype, cache, d):
    paged(**tensors(dtype, cache, d))


@pytest.mark.parametrize("change,match", [
    ({"k_cache": torch.zeros(5, 2, 16, 32, dtype=torch.float16)}, "both alike"),
    ({"k_cache": torch.zeros(5, 2, 64, 16, dtype=torch.float16).transpose(2, 3)}, "contiguous"),
    ({"v_cache": torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)}, "share a dtype"),
    ({"k_cache": torch.zeros(5, 2, 16, 64), "v_cache": torch.zeros(5, 2, 16, 64)}, "cache's dtype must be float16"),
    ({"rows": torch.zeros(6, 4, 64)}, "float16 or bfloat16 only"),
    ({"rows": torch.zeros(6, 4, 64, dtype=torch.bfloat16)}, "the inputs' or an 8-bit one"),
    ({"k_cache": torch.zeros(5, 2, 16, 96, dtype=torch.float16), "v_cache": torch.zeros(5, 2, 16, 96, dtype=torch.float16)},
     "head dimension"),
    ({"k_cache": torch.zeros(0, 2, 16, 64, dtype=torch.float16), "v_cache": torch.zeros(0, 2, 16, 64, dtype=torch.float16)},
     "non-empty"),
    ({"page_table": torch.zeros(3, 0, dtype=torch.int32)}, "non-empty"),
    ({"page_table": torch.zeros(3, 2, dtype=torch.int64)}, "page_table"),
    ({"page_table": torch.zeros(2, 3, dtype=torch.int32).t()}, "page_table"),
    ({"lengths": torch.zeros(2, dtype=torch.int32)}, "lengths"),
    ({"lengths": torch.zeros(3, dtype=torch.int64)}, "lengths"),
    ({"k_scale": torch.zeros(5, 2, 16)}, "8-bit caches"),
    ({"lengths": torch.zeros(3, dtype=torch.int32, device="meta")}, "same device"),
])
def test_refused_caches(change, match):
    t = tensors()
    t.update(change)
    with pytest.raises(RuntimeError, match=match):
        paged(**t)


@pytest.mark.parametrize("change", [{"k_scale": None}, {"v_scale": torch.zeros(5, 2, 8)},
                                    {"v_scale": torch.zeros(5, 2, 16).half()}, {"k_scale": torch.zeros(5, 16, 2).transpose(1, 2)}])
def test_refused_scales(change):
    t = tensors(cache=torch.int8)
    t.update(change)
    with pytest.raises(RuntimeError, match="k_scale and v_scale"):
        paged(**t)


def test_refused_rows():
    t = tensors()
    cache, lengths = t["k_cache"], t["lengths"]
    rows = lambda x, cu=None: _checks.check_rows("paged_attn", x, cache, lengths, cu)  # noqa: E731
    rows(t["rows"])
    rows(torch.zeros(6, 9, 64, dtype=torch.float16)[:, 3:7])
    rows(torch.zeros(4, 6, 64, dtype=torch.float16).transpose(0, 1))
    for x, match in ((t["rows"][0], "shaped"), (torch.zeros(6, 4, 128, dtype=torch.float16), "shaped"),
                     (t["rows"][:0], "non-empty"), (t["rows"].transpose(1, 2).contiguous().transpose(1, 2), "16-byte steps"),
                     (torch.zeros(6, 4, 68, dtype=torch.float16)[..., :64], "16-byte steps"),
                     (torch.zeros(6 * 256 + 1, dtype=torch.float16)[1:].view(6, 4, 64), "aligned"),
                     (torch.zeros(7, 4, 64, dtype=torch.float16), "divide evenly")):
        with pytest.raises(RuntimeError, match=match):
            rows(x)
    rows(torch.zeros(7, 4, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int32))
    for cu in (torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32)[::2]):
        with pytest.raises(RuntimeError, match="cu_seqlens"):
            rows(t["rows"], cu)


def test_refused_heads_out_and_numbers():
    t = tensors()
    k = t["rows"][:, :2]
    _checks.check_same_rows("cache_write", k, k.clone(), t["k_cache"])
    for a, b in ((k, k[:, :1]), (k, k.bfloat16()), (t["rows"], t["rows"])):
        with pytest.raises(RuntimeError, match="share shape"):
            _checks.check_same_rows("cache_write", a, b, t["k_cache"])
    with pytest.raises(RuntimeError, match="multiple of the cache's heads"):
        _checks.check_query_heads("paged_attn", t["rows"][:, :3], t["k_cache"])
    q = t["rows"]
    _checks.check_out("paged_attn", q, torch.empty_like(q))
    _checks.check_out("paged_attn", q, torch.empty(4, 6, 64, dtype=q.dtype).transpose(0, 1))
    both = torch.zeros(12, 4, 64, dtype=torch.float16)
    _checks.check_out("paged_attn", both[:6], both[6:])
    for out, match in ((q.float(), "shape, dtype"), (q[:3], "shape, dtype"), (q, "share memory"), (both[4:10], "share memory"),
                       (torch.zeros(1, 4, 64, dtype=q.dtype).expand(6, 4, 64), "overlap"),
                       (torch.zeros(6, 1, 64, dtype=q.dtype).expand(6, 4, 64), "overlap")):
        with pytest.raises(RuntimeError, match=match):
            _checks.check_out("paged_attn", both[:6] if match == "share memory" and out is not q else q, out)
    assert _checks.check_max_new("paged_attn", 5) == 5
    for bad in (0, -1, 1.5, True, None):
        with pytest.raises(RuntimeError, match="max_new"):
            _checks.check_max_new("paged_attn", bad)
    for bad in (0, 2 ** 30 + 1, 2.0):
        with pytest.raises(RuntimeError, match="max_len"):
            _checks.check_max_len("cache_read", bad)
    assert _checks.read_dtype("cache_read", t["k_cache"], None) == torch.float16
    i8 = t["k_cache"].to(torch.int8)
    assert _checks.read_dtype("cache_read", i8, torch.bfloat16) == torch.bfloat16
    for cache, dtype in ((t["k_cache"], torch.bfloat16), (i8, None), (i8, torch.float32)):
        with pytest.raises(RuntimeError, match="dtype must be"):
            _checks.read_dtype("cache_read", cache, dtype)


# ---------------------------------------------------------------- the C entry points
def native_cache(**change):
    c = _native.PagedCacheArgs(256, 256, None, None, 256, 256, 5, 16, 2, 64, 3, 2, 2, _native.DTYPE_F16)
    for name, value in change.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("change,rc,match", [
    ({"k": None}, -1, "null"), ({"lengths": None}, -1, "null"), ({"dtype": _native.DTYPE_BF16}, -2, "tensors' dtype"),
    ({"dtype": _native.DTYPE_F32}, -2, "tensors' dtype"), ({"dtype": _native.DTYPE_I8}, -1, "k_scale"), ({"d": 96}, -2, "head dimension"),
    ({"pages": 0}, -1, "non-empty"), ({"page_size": -1}, -1, "non-empty"), ({"table_cols": 2 ** 27}, -2, "2\\^30 positions"),
    ({"pages": 2 ** 31 // 32}, -2, "2\\^31-1 rows"), ({"heads": 2 ** 40}, -2, "2\\^31-1 rows"), ({"page_size": 2 ** 62}, -2, "positions"),
    ({"seqs": 2 ** 25}, -2, "sequences"), ({"table_stride": -2}, -2, "stride"), ({"v": 264}, -1, "aligned")])
def test_c_entries_refuse_a_cache(change, rc, match):
    lib, c, p, f16 = _native.lib(), native_cache(**change), ctypes.c_void_p(256), _native.DTYPE_F16
    for got in (lambda: lib.pa_cache_write(c, p, p, f16, 6, 128, 64, 128, 64, None, None),
                lambda: lib.pa_cache_read(c, p, p, f16, 32, None),
                lambda: lib.pa_paged_attn_fwd(c, p, p, f16, 6, 4, 256, 64, 256, 64, None, 0, 1, p, 2 ** 40, None)):
        assert got() == rc
        assert __import__("re").search(match, _native.last_error()), _native.last_error()


def test_c_entries_refuse_arguments():
    lib, c, p, f16 = _native.lib(), native_cache(), ctypes.c_void_p(256), _native.DTYPE_F16
    odd = ctypes.c_void_p(264)
    attn = lambda cache=c, q=p, o=p, dt=f16, t=6, h=4, qs=256, qh=64, os_=256, oh=64, cu=None, ws=p, room=2 ** 40: \
        (lib.pa_paged_attn_fwd(cache, q, o, dt, t, h, qs, qh, os_, oh, cu, 0, 1, ws, room, None), _native.last_error())  # noqa: E731
    for kw, rc, match in (({"cache": None}, -1, "null cache"), ({"q": None}, -1, "null"), ({"dt": _native.DTYPE_F32}, -2, "bfloat16"),
                          ({"t": 0}, -1, "non-empty"), ({"t": 7}, -1, "divide evenly"), ({"t": 2 ** 31}, -2, "2^30"),
                          ({"h": 3}, -1, "multiple"), ({"h": 0}, -1, "multiple"), ({"q": odd}, -1, "aligned"), ({"qs": 4}, -1, "16-byte"),
                          ({"oh": -64}, -1, "16-byte"), ({"os_": 0, "oh": 0}, -1, "overlap"), ({"os_": 64, "oh": 64}, -1, "overlap")):
        got = attn(**kw)
        assert got[0] == rc and match in got[1], (kw, got)
    assert lib.pa_cache_write(c, None, p, f16, 6, 128, 64, 128, 64, None, None) == -1
    assert lib.pa_cache_write(c, p, odd, f16, 6, 128, 64, 128, 64, None, None) == -1
    assert lib.pa_cache_write(c, p, p, f16, 6, 128, 60, 128, 64, None, None) == -1
    assert lib.pa_cache_read(c, p, p, f16, 0, None) == -1
    assert lib.pa_cache_read(c, None, p, f16, 5, None) == -1
    assert lib.pa_cache_read(c, p, p, f16, 2 ** 31, None) == -2


def test_c_entries_refuse_more_work_than_they_can_count():
    """Offsets out of order could give every sequence all tokens: the worst case must fit the kernels' numbers."""
    lib, p, f16 = _native.lib(), ctypes.c_void_p(256), _native.DTYPE_F16
    c = native_cache(seqs=2 ** 24, heads=1, pages=1, table_cols=2 ** 25)
    for got in (lambda: lib.pa_paged_attn_workspace(c, f16, 2 ** 30, 1, p, 0),
                lambda: lib.pa_paged_attn_fwd(c, p, p, f16, 2 ** 30, 1, 64, 64, 64, 64, p, 0, 1, p, 2 ** 60, None)):
        assert got() == -2 and "2^62" in _native.last_error()
    c = native_cache(seqs=4096, heads=8, pages=2 ** 20, table_cols=2 ** 13)   # a large call
    assert lib.pa_paged_attn_workspace(c, f16, 2 ** 20, 64, p, 0) > 0


def test_index_arithmetic(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    exe = tmp_path / "paged_model_check"
    build = subprocess.run([hipcc, "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                            "-packed-fp32-ops", "-I", os.path.join(REPO, "phantom-a100_amd", "csrc"),
                            os.path.join(HERE, "native", "paged_model_check.cpp"), "-o", str(exe)],
                           capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr


# ---------------------------------------------------------------- the oracle
def test_oracle_attention_is_softmax_attention():
    p = po.make([(3, 10), (1, 7)], d=64, page=4, dtype=torch.float16)
    out, bound, mine = po.attn(p)
    k, v, here = po.rows(p, 0, 10)
    assert here.all() and mine.all()
    for i in range(3):
        s = (p.q[i, 3].double() @ k[1, :8 + i].t()) / 8.0
        assert torch.allclose(out[i, 3], torch.softmax(s, -1) @ v[1, :8 + i], rtol=1e-12, atol=1e-12)
    assert (bound > 0).all() and bound.max() < 0.02


def test_oracle_codes():
    x = torch.tensor([[1.0, -2.0, 0.5, 254.0], [0, 0, 0, 0], [1, math.inf, 0, 2], [2.0 ** -101, 0, 0, 0]])
    codes, scale = po.quantise(x, torch.int8)
    assert codes.tolist() == [[0, -1, 0, 127], [0] * 4, [0] * 4, [0] * 4]   # 0.5 and 0.25: to even
    assert scale[0] == 2 and scale[1] == 0 and math.isnan(scale[2]) and scale[3] == 0
    codes, scale = po.quantise(x, torch.float8_e4m3fn)
    assert codes.float()[0].tolist() == [1.75, -3.5, 0.875, 448.0] and scale[0] == torch.tensor(254.0) / 448


@pytest.mark.parametrize("change", [
    {}, {"k_cache": torch.zeros(5, 2, 64, 16, dtype=torch.float16).transpose(2, 3)}, {"v_cache": torch.zeros(5, 2, 16, 64)},
    {"v_cache": torch.zeros(4, 2, 16, 64, dtype=torch.float16)}, {"page_table": torch.zeros(3, 2, dtype=torch.int64)},
    {"page_table": torch.zeros(2, 3, dtype=torch.int32).t()}, {"lengths": torch.zeros(2, dtype=torch.int32)},
    {"lengths": torch.zeros(6, dtype=torch.int32)[::2]}, {"k_scale": torch.zeros(5, 2, 16)}, {"rows": torch.zeros(6, 4, 64)},
    {"rows": torch.zeros(6, 4, 68, dtype=torch.float16)[..., :64]}, {"rows": torch.zeros(7, 4, 64, dtype=torch.float16)}])
def test_one_pass_acceptance_agrees_with_the_checks(change, monkeypatch):
    """paged_ok accepts what the checks one by one accept (on CPU tensors that say they are on the GPU), nothing else."""
    class OnGpu(torch.Tensor):
        is_cuda = True
    t = tensors()
    t.update(change)
    t = {n: x if x is None else x.as_subclass(OnGpu) for n, x in t.items()}

    def one_by_one():
        try:
            _checks.check_paged("paged_attn", **t)
            _checks.check_rows("paged_attn", t["rows"], t["k_cache"], t["lengths"], None)
        except RuntimeError:
            return False
        return True
    ok = _checks.paged_ok(t["rows"], t["k_cache"], t["v_cache"], t["page_table"], t["lengths"], None, t["k_scale"], t["v_scale"])
    assert ok == one_by_one() == (not change)


def test_packed_arguments_are_the_structure():
    from cuda_attn import paged as pg
    t = tensors(cache=torch.int8)
    got = pg._cache_args(t["k_cache"], t["v_cache"], t["page_table"], t["lengths"], t["k_scale"], t["v_scale"])
    assert (got.k, got.v, got.k_scale, got.v_scale) == tuple(t[n].data_ptr() for n in ("k_cache", "v_cache", "k_scale", "v_scale"))
    assert (got.page_table, got.lengths) == (t["page_table"].data_ptr(), t["lengths"].data_ptr())
    assert (got.pages, got.page_size, got.heads, got.d, got.seqs, got.table_cols, got.table_stride, got.dtype) == \
        (5, 16, 2, 64, 3, 2, 2, _native.DTYPE_I8)
    assert pg._cache_args(t["k_cache"], t["v_cache"], t["page_table"], t["lengths"], None, None).k_scale is None
