"""Refusals of the operators around a decode step (CPU: every check runs before device work)."""
from __future__ import annotations

import ctypes

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


def chunks(lib, **kw):
    a = dict(q=A, ldq=512, k=A, v=A, t=1, pages=8, ps=16, pre=A, plen=20, table=A, stride=4, width=4, starts=A, lens=A,
             rows=9, n=2, nq=4, nkv=2, hd=128, out=A, ldo=512, ws=A, wl=1 << 40)
    a.update(kw)
    return lib.pyrite_cuda_attention_chunks(a["q"], a["ldq"], a["k"], a["v"], a["t"], a["pages"], a["ps"], a["pre"],
                                            a["plen"], a["table"], a["stride"], a["width"], a["starts"], a["lens"],
                                            a["rows"], a["n"], a["nq"], a["nkv"], a["hd"], a["out"], a["ldo"], a["ws"],
                                            a["wl"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(t=12), TYPE), (dict(q=None), BUFFER), (dict(pre=None), BUFFER), (dict(starts=None), BUFFER),
    (dict(lens=None), BUFFER), (dict(table=None), BUFFER), (dict(ws=None), BUFFER), (dict(wl=4), BUFFER),
    (dict(ws=A + 8), BUFFER), (dict(hd=64), SHAPE), (dict(nq=3), SHAPE), (dict(nq=1026, nkv=2, ldq=1 << 18, ldo=1 << 18), SHAPE),
    (dict(rows=0), SHAPE), (dict(rows=(1 << 20) + 1), SHAPE), (dict(n=0), SHAPE), (dict(n=4081), SHAPE),
    (dict(plen=-1), SHAPE), (dict(width=0), SHAPE), (dict(stride=3), SHAPE), (dict(stride=-4), SHAPE),
    (dict(width=1 << 27, stride=1 << 27), SHAPE), (dict(ldq=508), SHAPE), (dict(ldq=513), SHAPE), (dict(ldo=514), SHAPE),
    (dict(q=A + 4), SHAPE), (dict(out=A + 8), SHAPE), (dict(k=A + 2), SHAPE), (dict(ps=24), SHAPE), (dict(pages=0), SHAPE)])
def test_chunks_refuse(lib, kw, code):
    assert chunks(lib, **kw) == code


def test_chunks_workspace_size(lib):
    f = lib.pyrite_cuda_attention_chunks_workspace_size
    assert f(0, 1, 4, 2, 0) == 0 and f((1 << 20) + 1, 1, 4, 2, 0) == 0 and f(8, 0, 4, 2, 0) == 0
    assert f(8, 4081, 4, 2, 0) == 0 and f(8, 1, 3, 2, 0) == 0 and f(8, 1, 4, 2, 2) == 0 and f(8, 1, 2048, 2, 0) == 0
    for t in (0, 1, 30):
        assert 0 < f(1, 1, 8, 8, t) <= f(1 << 20, 4080, 64, 4, t) < 1 << 30


def release(lib, **kw):
    a = dict(lens=A, keep=A, n=4, ps=16, free=A, n_free=64, used=A, used_out=A, table=A, stride=8, width=8, shared=A,
             shared_out=A, pages=64, lens_out=A)
    a.update(kw)
    return lib.pyrite_cuda_release_pages(a["lens"], a["keep"], a["n"], a["ps"], a["free"], a["n_free"], a["used"],
                                         a["used_out"], a["table"], a["stride"], a["width"], a["shared"],
                                         a["shared_out"], a["pages"], a["lens_out"], None)


def fork(lib, **kw):
    a = dict(parents=A, lens=A, n=4, ps=16, free=A, n_free=64, used=A, used_out=A, table=A, stride=8, width=8, shared=A,
             shared_out=A, pages=64, src=A, dst=A, lens_out=A)
    a.update(kw)
    return lib.pyrite_cuda_fork_requests(a["parents"], a["lens"], a["n"], a["ps"], a["free"], a["n_free"], a["used"],
                                         a["used_out"], a["table"], a["stride"], a["width"], a["shared"],
                                         a["shared_out"], a["pages"], a["src"], a["dst"], a["lens_out"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(lens=None), BUFFER), (dict(shared=None), BUFFER), (dict(lens_out=None), BUFFER), (dict(used_out=None), BUFFER),
    (dict(n=0), SHAPE), (dict(n=4081), SHAPE), (dict(ps=8), SHAPE), (dict(ps=48), SHAPE), (dict(n_free=0), SHAPE),
    (dict(width=0), SHAPE), (dict(stride=7), SHAPE), (dict(width=1 << 28, stride=1 << 28), SHAPE), (dict(pages=0), SHAPE),
    (dict(pages=(1 << 20) + 1), SHAPE)])
def test_fork_and_release_refuse(lib, kw, code):
    assert release(lib, **kw) == code and fork(lib, **kw) == code


def test_fork_and_release_need_their_own(lib):
    assert release(lib, keep=None) == BUFFER
    assert fork(lib, parents=None) == BUFFER and fork(lib, src=None) == BUFFER and fork(lib, dst=None) == BUFFER


@pytest.mark.parametrize("kw,code", [
    (dict(t=8), TYPE), (dict(k=None), BUFFER), (dict(src=None), BUFFER), (dict(pools=0), SHAPE), (dict(pages=0), SHAPE),
    (dict(ps=20), SHAPE), (dict(nkv=0), SHAPE), (dict(hd=64), SHAPE), (dict(count=0), SHAPE), (dict(at=None), BUFFER),
    (dict(at=A + 8), SHAPE)])
def test_copy_refuses(lib, kw, code):
    a = dict(k=A, at=A, pools=2, t=1, pages=4, ps=16, nkv=1, hd=128, src=A, dst=A, count=3)
    a.update(kw)
    list_of = (ctypes.c_void_p * 2)(A, a["at"])
    assert lib.pyrite_cuda_copy_pages(list_of if a["k"] else None, list_of, a["pools"], a["t"], a["pages"], a["ps"],
                                      a["nkv"], a["hd"], a["src"], a["dst"], a["count"], None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), BUFFER), (dict(t=None), BUFFER), (dict(out=None), BUFFER), (dict(n=0), SHAPE),
    (dict(n=(1 << 20) + 1, ld=1 << 21, ldp=1 << 21), SHAPE), (dict(count=0), SHAPE), (dict(count=65536), SHAPE),
    (dict(ld=9), SHAPE), (dict(ldp=9), SHAPE), (dict(out=A + 2), SHAPE)])
def test_probs_refuse(lib, kw, code):
    a = dict(logits=A, ld=10, n=10, count=2, t=A, out=A, ldp=10)
    a.update(kw)
    assert lib.pyrite_cuda_token_probs(a["logits"], a["ld"], a["n"], a["count"], a["t"], None, None, None, a["out"],
                                       a["ldp"], None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(p=None), BUFFER), (dict(x=None), BUFFER), (dict(starts=None), BUFFER), (dict(u=None), BUFFER),
    (dict(counts=None), BUFFER), (dict(n=0), SHAPE), (dict(n=(1 << 20) + 1, ldp=1 << 21), SHAPE), (dict(rows=0), SHAPE),
    (dict(rows=(1 << 24) + 1), SHAPE), (dict(m=0), SHAPE), (dict(m=65536), SHAPE), (dict(ldp=9), SHAPE),
    (dict(q=A, ldq=9), SHAPE), (dict(q=A + 2, ldq=10), SHAPE)])
def test_verify_refuses(lib, kw, code):
    a = dict(p=A, ldp=10, n=10, rows=5, q=None, ldq=0, x=A, starts=A, m=2, u=A, pick=A, out=A, counts=A)
    a.update(kw)
    assert lib.pyrite_cuda_verify_drafts(a["p"], a["ldp"], a["n"], a["rows"], a["q"], a["ldq"], a["x"], a["starts"],
                                         a["m"], a["u"], a["pick"], a["out"], a["counts"], None) == code


def test_wrappers_refuse_host_tensors_and_what_is_no_tensor():
    from types import SimpleNamespace

    from pyrite_b200.kernels import paged, sampling
    i, f = torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    pool = SimpleNamespace(k=f, v=f)
    with pytest.raises(ValueError, match="CUDA"):
        paged.attention_chunks(torch.zeros(2, 256), pool, i[:, None], i, i[:1])
    with pytest.raises(ValueError, match="CUDA"):
        paged.fork_requests(i, i, 16, i, i[:1], i[:, None], i)
    with pytest.raises(ValueError, match="CUDA"):
        paged.release_pages(i, i, 16, i, i[:1], i[:, None], i)
    with pytest.raises(ValueError, match="CUDA"):
        paged.copy_pages([pool], i[None])
    with pytest.raises(ValueError, match="must be a tensor"):
        paged.copy_pages([pool], [1, 2])
    with pytest.raises(ValueError, match="CUDA"):
        sampling.token_probs(torch.zeros(2, 8), f)
    with pytest.raises(ValueError, match="CUDA"):
        sampling.verify_drafts(torch.zeros(2, 8), i, i, f, f[:1])
    with pytest.raises(ValueError, match="starts must be a tensor"):
        sampling.verify_drafts(torch.zeros(2, 8), i, [0, 2], f, f[:1])
    with pytest.raises(ValueError, match="sizes"):
        paged.chunks_workspace(2, 1, 3, 2, device="cpu")
    with pytest.raises(ValueError, match="sizes"):
        paged.chunks_workspace(2, 1, 4, 2, torch.float64, device="cpu")


def test_a_launch_that_cuda_refuses_is_a_cuda_error():
    """Valid arguments without a device: PYRITE_E_CUDA from every entry point (in a process that sees no device)."""
    import os
    import subprocess
    import sys
    code = """
import ctypes
from tests.test_serving_api import A, _lib, chunks, fork, release
lib = _lib.load()
assert lib.pyrite_cuda_device_count() <= 0
two = (ctypes.c_void_p * 2)(A, A)
print(chunks(lib), chunks(lib, t=0), fork(lib), release(lib),
      lib.pyrite_cuda_copy_pages(two, two, 2, 1, 4, 16, 1, 128, A, A, 3, None),
      lib.pyrite_cuda_token_probs(A, 10, 10, 2, A, None, None, None, A, 10, None),
      lib.pyrite_cuda_verify_drafts(A, 10, 10, 5, None, 0, A, A, 2, A, A, A, A, None))
"""
    run = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), text=True,
                         capture_output=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert run.returncode == 0, run.stderr
    assert run.stdout.split() == ["-4"] * 7


@pytest.mark.parametrize("kw,refused", [
    (dict(), False), (dict(out=A, ldo=1024), True), (dict(rows=1, out=A, ldo=1024), False), (dict(out=A + 16), True),
    (dict(out=A + 2048), True), (dict(out=A - 2048), True),  # a row further or back
    (dict(out=A + 9 * 2048), False), (dict(out=A + 9 * 2048 - 16), True), (dict(out=A - 9 * 2048), False),
    (dict(out=A - 9 * 2048 + 16), True),
    (dict(ldq=1024, ldo=1024, out=A + 2048), False), (dict(ldq=1024, ldo=1024, out=A + 2032), True),  # side by side
    (dict(ldq=1024, ldo=1024, out=A - 2048), False), (dict(ldq=1024, ldo=1024, out=A - 2032), True),
    (dict(ldq=1024, ldo=1024, out=A + 4096), True), (dict(ldq=1024, ldo=1024, out=A + 8 * 4096 + 2048), False),
    (dict(ldq=1024, ldo=1024, out=A + 3 * 4096 + 2064), True),
    (dict(ldq=2048, ldo=512, out=A + 2048, rows=3), False), (dict(ldq=2048, ldo=512, out=A + 2048, rows=4), True),
    (dict(ldq=512, ldo=2048, out=A - 2048, rows=3), False), (dict(ldq=512, ldo=2048, out=A - 2048, rows=4), True),
    (dict(ldq=516, ldo=1024, out=A + 9 * 2064 - 16), False)])
def test_chunks_refuse_an_output_over_the_queries(lib, kw, refused):
    """9 rows of 512 floats (2048 bytes) at A: the output is the queries themselves, or shares no value with them."""
    if lib.pyrite_cuda_device_count() > 0:
        pytest.skip("what is not refused would be launched")
    assert chunks(lib, **kw) == (BUFFER if refused else -4)


def test_chunks_refuse_every_output_that_shares_a_value(lib):
    """Random rows, strides and places against the sets of their values."""
    import random
    if lib.pyrite_cuda_device_count() > 0:
        pytest.skip("what is not refused would be launched")
    rng, seen = random.Random(0), [0, 0]
    for _ in range(600):
        rows, ldq, ldo, at = rng.randint(1, 6), *(4 * rng.choice([32, 33, 40, 64, 96, 200]) for _ in range(2)), 4 * rng.randint(-300, 300)
        q = {i * ldq + j for i in range(rows) for j in range(128)}
        out = {at + i * ldo + j for i in range(rows) for j in range(128)}
        refused = bool(q & out) and not (at == 0 and (ldq == ldo or rows == 1))
        seen[refused] += 1
        assert chunks(lib, rows=rows, nq=1, nkv=1, ldq=ldq, ldo=ldo, out=A + 4 * at) == (BUFFER if refused else -4)
    assert min(seen) > 100


@pytest.mark.parametrize("kw,refused", [(dict(out=A + 4), True), (dict(out=A + 16), True), (dict(out=A + 40), True),
                                        (dict(out=A + 80), False), (dict(out=A + 76), True), (dict(out=A, ldp=11), True),
                                        (dict(ld=20, ldp=20, out=A + 40), False), (dict(ld=20, ldp=20, out=A + 36), True)])
def test_probs_over_the_logits(lib, kw, refused):
    """Two rows of 10 logits at A."""
    if lib.pyrite_cuda_device_count() > 0:
        pytest.skip("what is not refused would be launched")
    a = dict(ld=10, out=A, ldp=10)
    a.update(kw)
    code = lib.pyrite_cuda_token_probs(A, a["ld"], 10, 2, A, None, None, None, a["out"], a["ldp"], None)
    assert code == (BUFFER if refused else -4)


@pytest.mark.parametrize("shift,refused", [(0, False), (4, True), (-4, True), (16, True), (20, False), (-20, False), (-16, True)])
def test_verify_over_the_drafts(lib, shift, refused):
    """Five tokens at A: out is the drafts themselves, or lies beside them."""
    if lib.pyrite_cuda_device_count() > 0:
        pytest.skip("what is not refused would be launched")
    code = lib.pyrite_cuda_verify_drafts(A, 10, 10, 5, None, 0, A, A, 2, A, A, A + shift, A, None)
    assert code == (BUFFER if refused else -4)
