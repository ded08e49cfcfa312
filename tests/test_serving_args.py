"""The paged KV cache's and the sampler's index rules and refusals (CPU): the
rules that the kernels share with the host, run under the undefined-behaviour
sanitizer, and calls that must fail before anything reaches a device."""
import ctypes
import os
import subprocess

import pytest

from munet_amd import _lib, build, synth

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16 = synth.F32, synth.F16, synth.BF16
A = 1 << 20  # a 16-byte aligned address that no refused call may touch


def test_paged_index_rules(tmp_path):
    exe = str(tmp_path / "check")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-D__host__=",
                        "-D__device__=", "-D__forceinline__=inline", "-I", build.CSRC,
                        os.path.join(ROOT, "tests", "cxx", "paged_index_check.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr[-2000:]


def _plan(**kw):
    a = dict(lens=A, new_lens=A, free_pages=A, tables=A, total=A, cu=A, slots=A, positions=None, used=A, B=4, n_free=8,
             width=4, page=16, n_pages=64, n_slots=10)
    a.update(kw)
    _lib.call("mh_page_plan", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(page=48), "16, 32, 64, 128 or 256"), (dict(page=8), "16, 32"), (dict(page=512), "16, 32"),
    (dict(n_pages=0), "pool"), (dict(n_pages=1 << 27), "pool"), (dict(B=-1), "negative"), (dict(width=-2), "negative"),
    (dict(n_slots=-1), "negative"), (dict(width=1 << 27), "table row"), (dict(width=(1 << 27) - 1), "table row"), (dict(lens=None), "null"), (dict(used=None), "null"),
    (dict(slots=None), "null"), (dict(tables=None), "null"), (dict(free_pages=None), "null"), (dict(B=1 << 24), "one launch")])
def test_page_plan_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _plan(**kw)


def test_page_plan_refuses_operands_that_overlap():
    """Lengths updated in place, outputs inside one another."""
    apart = dict(lens=A, new_lens=A + 64, free_pages=A + 128, tables=A + 256, total=A + 512, cu=A + 576, slots=A + 640,
                 positions=A + 704, used=A + 768)
    for kw, match in ((dict(total=A), "an input"), (dict(total=A + 12), "an input"), (dict(slots=A + 64 - 36), "an input"),
                      (dict(used=A + 128 + 28), "an input"), (dict(positions=A + 640), "two outputs"), (dict(cu=A + 512 - 16), "two outputs"),
                      (dict(tables=A + 512 - 60), "two outputs")):
        with pytest.raises(_lib.HipError, match=match):
            _plan(**{**apart, **kw})


def _store(**kw):
    a = dict(dt=BF16, k=A, v=A, ldk=1024, ldv=1024, slots=A, kc=A, vc=A, ks=A, vs=A, n=4, Hkv=8, hd=128, page=64, n_pages=16)
    a.update(kw)
    _lib.call("mh_kv_store_paged", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "dtype"), (dict(hd=24), "multiple of 16"), (dict(hd=272), "multiple of 16"), (dict(hd=0), "multiple of 16"),
    (dict(Hkv=0), "head count"), (dict(page=100), "page holds"), (dict(n=-1), "negative"), (dict(slots=None), "null"),
    (dict(k=None), "null k"), (dict(v=A + 8), "aligned"), (dict(ldk=1023), "multiple of 16"), (dict(ldv=1016), "whole"),
    (dict(kc=A + 4), "aligned"), (dict(vs=None), "null cache"), (dict(dt=F32, ldk=1026), "multiple of 16"),
    (dict(n=(1 << 27) + 1), "one launch"), (dict(Hkv=65536), "head count")])
def test_kv_store_paged_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _store(**kw)


def _attend(**kw):
    a = dict(dt=BF16, q=A, ldq=2048, kc=A, vc=A, ks=A, vs=A, tables=A, lens=A, cu=A, out=A, ldo=2048, B=2, n_rows=2, Hq=16,
             Hkv=4, hd=128, page=64, n_pages=16, width=8, max_q=1, max_len=100, causal=1, window=0, scale=0.0, ws=None, nbytes=0)
    a.update(kw)
    _lib.call("mh_attention_paged", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=4), "dtype"), (dict(Hq=15), "multiple of key/value heads"), (dict(hd=136), "multiple of 16"), (dict(page=0), "page holds"),
    (dict(q=None), "null q"), (dict(out=A + 2), "aligned"), (dict(ldq=2047), "multiple of 16"), (dict(ldo=1024), "whole"),
    (dict(B=-1), "negative"), (dict(window=-1), "negative"), (dict(max_len=-5), "negative"), (dict(lens=None), "null"),
    (dict(cu=None), "null"), (dict(tables=None), "null"), (dict(width=1 << 26), "table row"), (dict(width=(1 << 25) - 1), "table row"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(n_rows=1 << 29), "2\\^30"), (dict(max_len=100000), "workspace"),
    (dict(max_len=100000, ws=A, nbytes=100), "workspace"), (dict(max_len=100000, ws=A + 8, nbytes=1 << 40), "aligned")])
def test_attention_paged_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _attend(**kw)


def _sample(**kw):
    a = dict(dt=BF16, logits=A, ld=100, rows=2, cols=100, u=A, temperature=None, top_k=None, top_p=None, min_p=None, out=A,
             logprob=None, ws=None, nbytes=0)
    a.update(kw)
    _lib.call("mh_sample", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "dtype"), (dict(rows=-1), "bad row count"), (dict(cols=0), "empty rows"), (dict(ld=99), "overlap"),
    (dict(logits=None), "null"), (dict(u=None), "null"), (dict(out=None), "null"), (dict(logits=A + 1), "aligned"),
    (dict(rows=1 << 22), "one launch")])
def test_sample_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _sample(**kw)


def test_empty_calls_need_no_device():
    _plan(B=0)
    _store(n=0)
    _attend(B=0)
    _attend(n_rows=0)
    _sample(rows=0)


def test_workspace_sizes():
    n = ctypes.c_size_t(7)
    _lib.call("mh_attention_paged_workspace", BF16, 64, 64, 32, 8, 128, 1, 40, 0, ctypes.byref(n))
    assert n.value == 0  # one share: nothing to join
    _lib.call("mh_attention_paged_workspace", BF16, 1, 1, 8, 8, 128, 1, 100000, 0, ctypes.byref(n))
    assert n.value > 0 and n.value % (8 * (128 * 4 + 8)) == 0  # whole shares of 8 rows
    with pytest.raises(_lib.HipError, match="null output"):
        _lib.call("mh_attention_paged_workspace", BF16, 1, 1, 8, 8, 128, 1, 10, 0, None)
    with pytest.raises(_lib.HipError, match="null output"):
        _lib.call("mh_sample_workspace", BF16, 1, 8, None)


def test_tensors_must_share_a_gpu():
    torch = pytest.importorskip("torch")
    from munet_amd.backend import HipBackend
    hip = HipBackend.__new__(HipBackend)  # (no device here)
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="one GPU"):
        hip.sample(x, torch.zeros(4), torch.zeros(4, dtype=torch.int32))
