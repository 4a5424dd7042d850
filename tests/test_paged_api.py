"""Refusals of the serving entry points (CPU: every check runs before device work).

Arguments are checked in the C ABI before a stream or device is touched, so
these calls pass addresses that are never read; the Python wrappers refuse
tensors that are not on a CUDA device.
"""
from __future__ import annotations

import pytest
import torch

from pyrite_b200 import _lib

TYPE, SHAPE, BUFFER = -1, -2, -3
A = 0x10000  # an aligned address; never read


@pytest.fixture(scope="module")
def lib():
    lib = _lib.load()
    assert lib is not None
    return lib


def tables(lib, **kw):
    a = dict(lens=A, new=A, n=4, ps=16, free=A, n_free=64, used=A, used_out=A, table=A, stride=8, width=8, row_stride=1,
             slots=A, pos=A, cap=4, starts=A, kv=A, ticket=A)
    a.update(kw)
    return lib.pyrite_cuda_page_tables(a["lens"], a["new"], a["n"], a["ps"], a["free"], a["n_free"], a["used"],
                                       a["used_out"], a["table"], a["stride"], a["width"], a["row_stride"], a["slots"],
                                       a["pos"], a["cap"], a["starts"], a["kv"], a["ticket"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(lens=None), BUFFER), (dict(ticket=None), BUFFER), (dict(row_stride=0, starts=None), BUFFER),
    (dict(used_out=None), BUFFER), (dict(n=0), SHAPE), (dict(n=4081, cap=4081), SHAPE), (dict(ps=8), SHAPE),
    (dict(ps=48), SHAPE), (dict(ps=512), SHAPE), (dict(n_free=0), SHAPE), (dict(width=0), SHAPE), (dict(stride=7), SHAPE),
    (dict(row_stride=-1), SHAPE), (dict(cap=5), SHAPE), (dict(cap=0, row_stride=0), SHAPE),
    (dict(n_free=1 << 28), SHAPE), (dict(width=1 << 28, stride=1 << 28), SHAPE)])
def test_page_tables_refuses(lib, kw, code):
    assert tables(lib, **kw) == code


def append(lib, **kw):
    a = dict(qkv=A, ldqkv=4 * 128, qn=None, kn=None, nq=2, nkv=1, hd=128, first=0, pos=A, slots=A, count=3, rope=A,
             max_ctx=64, q=A, ldq=256, k=A, v=A, t=0, pages=4, ps=16)
    a.update(kw)
    return lib.pyrite_cuda_qk_rope_kv_paged(a["qkv"], a["ldqkv"], a["qn"], a["kn"], a["nq"], a["nkv"], a["hd"], 1e-6,
                                            a["first"], a["pos"], a["slots"], a["count"], a["rope"], a["max_ctx"],
                                            a["q"], a["ldq"], a["k"], a["v"], a["t"], a["pages"], a["ps"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(t=8), TYPE), (dict(qkv=None), BUFFER), (dict(slots=None), BUFFER), (dict(v=None), BUFFER), (dict(hd=64), SHAPE),
    (dict(nq=3, nkv=2, ldqkv=8 * 128, ldq=512), SHAPE), (dict(nq=0), SHAPE), (dict(count=0), SHAPE),
    (dict(first=-1), SHAPE), (dict(ldqkv=511), SHAPE), (dict(ldq=254), SHAPE), (dict(ldq=257), SHAPE),
    (dict(qkv=A + 4), SHAPE), (dict(k=A + 8), SHAPE), (dict(pages=0), SHAPE), (dict(ps=17), SHAPE),
    (dict(pages=1 << 27, ps=16), SHAPE), (dict(max_ctx=0), SHAPE)])
def test_append_refuses(lib, kw, code):
    assert append(lib, **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(t=2), TYPE), (dict(k=None), BUFFER), (dict(slots=None), BUFFER), (dict(hd=256), SHAPE), (dict(ld=126), SHAPE),
    (dict(count=0), SHAPE), (dict(k=A + 4), SHAPE), (dict(kp=A + 8), SHAPE), (dict(ps=0), SHAPE)])
def test_store_refuses(lib, kw, code):
    a = dict(k=A, v=A, ld=128, slots=A, count=2, nkv=1, hd=128, kp=A, vp=A, t=0, pages=4, ps=16)
    a.update(kw)
    assert lib.pyrite_cuda_kv_store_paged(a["k"], a["v"], a["ld"], a["slots"], a["count"], a["nkv"], a["hd"], a["kp"],
                                          a["vp"], a["t"], a["pages"], a["ps"], None) == code


def attention(lib, **kw):
    a = dict(q=A, ldq=512, k=A, v=A, t=1, pages=8, ps=16, pre=A, plen=20, table=A, stride=4, width=4, lens=A, count=2,
             nq=4, nkv=2, hd=128, out=A, ldo=512, ws=A, wl=None)
    a.update(kw)
    if a["wl"] is None:
        a["wl"] = int(lib.pyrite_cuda_attention_paged_workspace_size(a["count"], a["nq"], a["nkv"], a["plen"], a["t"]))
    return lib.pyrite_cuda_attention_paged(a["q"], a["ldq"], a["k"], a["v"], a["t"], a["pages"], a["ps"], a["pre"],
                                           a["plen"], a["table"], a["stride"], a["width"], a["lens"], a["count"],
                                           a["nq"], a["nkv"], a["hd"], a["out"], a["ldo"], a["ws"], a["wl"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(t=12), TYPE), (dict(q=None), BUFFER), (dict(pre=None), BUFFER), (dict(lens=None), BUFFER),
    (dict(ws=None), BUFFER), (dict(wl=16), BUFFER), (dict(ws=A + 8), BUFFER), (dict(hd=64), SHAPE),
    (dict(nq=3), SHAPE), (dict(count=0), SHAPE), (dict(count=4097), SHAPE), (dict(plen=-1), SHAPE),
    (dict(width=0), SHAPE), (dict(stride=3), SHAPE), (dict(stride=-4), SHAPE), (dict(ldq=508), SHAPE),
    (dict(ldq=513), SHAPE), (dict(ldo=514), SHAPE), (dict(q=A + 4), SHAPE), (dict(out=A + 8), SHAPE),
    (dict(k=A + 2), SHAPE), (dict(ps=24), SHAPE), (dict(pages=0), SHAPE)])
def test_attention_refuses(lib, kw, code):
    assert attention(lib, **kw) == code


def test_attention_workspace_size(lib):
    f = lib.pyrite_cuda_attention_paged_workspace_size
    assert f(0, 4, 2, 0, 0) == 0 and f(4097, 4, 2, 0, 0) == 0 and f(2, 3, 2, 0, 0) == 0
    assert f(2, 4, 2, -1, 0) == 0 and f(2, 4, 2, 0, 2) == 0
    for t in (0, 1, 30):
        assert 0 < f(1, 8, 8, 0, t) < 1 << 24 and 0 < f(128, 64, 4, 8192, t) < 1 << 30


@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), BUFFER), (dict(u=None), BUFFER), (dict(t=None), BUFFER), (dict(ids=None), BUFFER),
    (dict(n=0), SHAPE), (dict(n=(1 << 20) + 1, ld=1 << 21), SHAPE), (dict(count=0), SHAPE), (dict(count=65536), SHAPE),
    (dict(ld=9), SHAPE)])
def test_sampling_refuses(lib, kw, code):
    a = dict(logits=A, ld=10, n=10, count=2, u=A, t=A, ids=A)
    a.update(kw)
    assert lib.pyrite_cuda_sample_rows(a["logits"], a["ld"], a["n"], a["count"], a["u"], a["t"], None, None, None,
                                       a["ids"], None, None) == code


@pytest.mark.parametrize("kw,code", [(dict(ids=None), BUFFER), (dict(limits=None), BUFFER), (dict(count=0), SHAPE),
                                     (dict(stride=0), SHAPE)])
def test_commit_refuses(lib, kw, code):
    a = dict(ids=A, count=2, stride=8, limits=A)
    a.update(kw)
    assert lib.pyrite_cuda_commit_tokens(a["ids"], a["count"], A, a["stride"], A, A, A, A, a["limits"], None) == code


def test_wrappers_refuse_host_tensors():
    from pyrite_b200.kernels import paged, sampling
    z = torch.zeros(2, 2, 16, 128)
    with pytest.raises(ValueError, match="CUDA"):
        paged.KVPool(z, z)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.page_tables(i, i, 16, i, i[:1], i[:, None], paged.TokenSlots.empty(2, row_stride=1, device="cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        sampling.sample_rows(torch.zeros(2, 8), torch.zeros(2), torch.zeros(2))
    with pytest.raises(ValueError, match="sizes"):
        paged.attention_workspace(2, 3, 2, device="cpu")


def test_native_calls_refuse_what_is_no_tensor():
    from pyrite_b200.kernels import _launch
    c = _launch.calls()
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="lens must be a tensor"):
        c.page_tables([1, 2], i, 16, i, i[:1], i[:, None], i[:1], i, i, i, i, i[:1], 1)
    with pytest.raises(ValueError, match="arguments"):
        c.store_kv(i, i)
    with pytest.raises(ValueError, match="q_norm must be a tensor"):
        c.append_kv(i, i, i, i, i, i, 2, 3, None, 1e-6, 0, None)
    with pytest.raises(TypeError):
        c.attention(i, i, i, i, i, None, 1.5, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        c.sample_rows(i, i, i, None, None, None, None, None)
    assert set(c.entries()) <= set(_lib.SIGNATURES)
    with pytest.raises(KeyError):
        c.bind("pyrite_matvec", 0)


def test_native_calls_are_loaded_once_by_many_threads():
    from concurrent.futures import ThreadPoolExecutor

    from pyrite_b200.kernels import _launch
    with ThreadPoolExecutor(8) as pool:
        assert len({id(f.result()) for f in [pool.submit(_launch.calls) for _ in range(32)]}) == 1


def test_a_launch_that_cuda_refuses_is_a_cuda_error():
    """Valid arguments without a device: PYRITE_E_CUDA from every entry point (in a process that sees no device)."""
    import os
    import subprocess
    import sys
    code = """
from tests.test_paged_api import A, _lib, append, attention, tables
lib = _lib.load()
assert lib.pyrite_cuda_device_count() <= 0
print(tables(lib), append(lib), attention(lib),
      lib.pyrite_cuda_kv_store_paged(A, A, 128, A, 2, 1, 128, A, A, 0, 4, 16, None),
      lib.pyrite_cuda_sample_rows(A, 10, 10, 2, A, A, None, None, None, A, None, None),
      lib.pyrite_cuda_commit_tokens(A, 2, A, 8, A, A, A, A, A, None),
      lib.pyrite_cuda_advance_pos(A, None), lib.pyrite_cuda_moe_combine_rows(A, A, 2, 32, 1, A, 32, None))
from pyrite_b200.kernels.cuda import _check
try:
    _check(lib.pyrite_cuda_commit_tokens(A, 2, A, 8, A, A, A, A, A, None), "commit tokens")
except RuntimeError as e:
    print(e)
"""
    run = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), text=True,
                         capture_output=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert run.returncode == 0, run.stderr
    lines = run.stdout.splitlines()
    assert lines[0].split() == ["-4"] * 8 and "CUDA error" in lines[1]


@pytest.mark.parametrize("word,says", [(0, ""), (1, "timed out"), (2, "expert id"), (4, "page or slot"),
                                       (5, "timed out, page or slot"), (-4, "CUDA runtime error")])
def test_check_status_names_what_happened(word, says):
    from types import SimpleNamespace

    from pyrite_b200.dense import DenseDecoder
    from pyrite_b200.model import MixedDecoder
    for cls in (MixedDecoder, DenseDecoder):
        dec = cls.__new__(cls)
        dec.lib = SimpleNamespace(pyrite_cuda_status=lambda clear: word)
        if word == 0:
            dec.check_status()
            continue
        with pytest.raises(RuntimeError) as e:
            dec.check_status()
        for part in ("timed out", "expert id", "page or slot", "CUDA runtime error"):
            assert (part in str(e.value)) == (part in says)
