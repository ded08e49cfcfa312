"""Rotary positions and 8-bit products on the CPU: frequencies against their
formulas, and calls that must fail before anything reaches a device."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

from munet_amd import _lib, build, synth
from munet_amd.backend import rotary_frequencies

F32, F16, BF16 = synth.F32, synth.F16, synth.BF16
A = 1 << 20  # a 16-byte aligned address that no refused call may touch
FAR = 1 << 34


# ---- frequencies -------------------------------------------------------------------

def close(a, b):
    # pow within 2 units of the last place of 64 bits, a handful of products
    np.testing.assert_allclose(a, b, rtol=1e-14, atol=0)


def plain(rot, base):
    return np.array([base ** (-2.0 * j / rot) for j in range(rot // 2)])


@pytest.mark.parametrize("rot", [2, 4, 24, 64, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_frequencies(rot, base):
    f, m = rotary_frequencies(rot, base)
    assert m == 1.0 and f.dtype == np.float64 and f.shape == (rot // 2,)
    close(f, plain(rot, base))
    f, m = rotary_frequencies(rot, base, "linear", 4.0)
    assert m == 1.0
    close(f, plain(rot, base) / 4)
    if rot >= 4:
        f, m = rotary_frequencies(rot, base, "base", 8.0)
        assert m == 1.0
        close(f, plain(rot, base * 8.0 ** (rot / (rot - 2))))
        # the fastest pair stays, the slowest is stretched by the factor
        close(f[0], 1.0)
        close(f[-1], plain(rot, base)[-1] / 8)


@pytest.mark.parametrize("low,high,original", [(1.0, 32.0, 4096), (1.0, 4.0, 8192), (0.0, 1e9, 100)])
def test_frequencies_by_turns(low, high, original):
    rot, factor = 128, 16.0
    f, m = rotary_frequencies(rot, 10000.0, "turns", factor, original, low, high)
    close(m, 1 + 0.1 * math.log(factor))
    want = []
    for p in plain(rot, 10000.0):
        r = original * p / (2 * math.pi)
        want.append(p if r >= high else p / factor if r <= low else p * ((r - low) / (high - low) * (1 - 1 / factor) + 1 / factor))
    np.testing.assert_allclose(f, want, rtol=1e-12, atol=0)  # (a difference of near values in the ramp)
    assert rotary_frequencies(rot, 10000.0, "turns", 1.0, original, low, high)[1] == 1.0


@pytest.mark.parametrize("args,match", [
    ((63,), "even"), ((0,), "even"), ((-4,), "even"), ((64, 0.0), "base"), ((64, float("nan")), "base"), ((64, float("inf")), "base"),
    ((64, 1e4, "linear", 0.0), "factor"), ((64, 1e4, "linear", float("inf")), "factor"), ((2, 1e4, "base", 2.0), "4 at least"),
    ((64, 1e4, "turns", 4.0), "original"), ((64, 1e4, "turns", 4.0, 4096, 4.0, 4.0), "low < high"),
    ((64, 1e4, "turns", 4.0, 4096, -1.0, 4.0), "low < high"), ((64, 1e4, "turns", 4.0, 4096, 1.0, float("nan")), "low < high")])
def test_frequency_refusals(args, match):
    with pytest.raises(_lib.HipError, match=match):
        rotary_frequencies(*args)


def test_frequency_names():
    with pytest.raises(ValueError, match="scaling must be"):
        rotary_frequencies(64, scaling="square")
    with pytest.raises(_lib.HipError, match="unknown scaling"):
        _lib.call("mh_rotary_frequencies", (ctypes.c_double * 4)(), None, 8, 1e4, 4, 1.0, 0.0, 0.0, 0.0)
    with pytest.raises(_lib.HipError, match="null"):
        _lib.call("mh_rotary_frequencies", None, None, 8, 1e4, 0, 1.0, 0.0, 0.0, 0.0)


# ---- refusals ------------------------------------------------------------------------

def _table(**kw):
    a = dict(positions=A, freq=A, table=A, n=4, half=8, magnitude=1.0)
    a.update(kw)
    _lib.call("mh_rotary_table", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(n=-1), "negative"), (dict(half=0), "no pairs"), (dict(positions=None), "null"), (dict(freq=None), "null"),
    (dict(table=None), "null"), (dict(table=A + 8), "aligned"), (dict(freq=FAR), "overlaps"), (dict(positions=FAR), "overlaps"),
    (dict(positions=A + 240, freq=FAR), "overlaps"), (dict(n=(1 << 31) - 1, half=(1 << 31) - 1), "larger")])
def test_rotary_table_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _table(**kw)


def _rotary(**kw):
    a = dict(dt=BF16, x=A, ldx=1024, table=A, out=FAR, ldo=1024, n=4, heads=8, hd=128, half=64, inter=0, inverse=0)
    a.update(kw)
    _lib.call("mh_rotary", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "dtype"), (dict(n=-1), "negative"), (dict(heads=0), "head count"), (dict(hd=0), "head count"),
    (dict(heads=1 << 20, hd=2048), "head count"), (dict(half=0), "rotated part"), (dict(half=65), "rotated part"),
    (dict(half=-3), "rotated part"), (dict(half=0x7fffffff), "rotated part"), (dict(table=None), "null table"), (dict(table=A + 4), "aligned"),
    (dict(x=None), "null x"), (dict(out=None), "null out"), (dict(x=A + 1), "aligned to its type"), (dict(dt=F32, out=FAR + 2), "aligned to its type"),
    (dict(ldx=1023), "whole"), (dict(ldo=-5), "whole"), (dict(ldx=1 << 57), "far apart"), (dict(out=A + 16), "overlaps"), (dict(out=A, ldo=2048), "overlaps"),
    (dict(out=A - 16), "overlaps"), (dict(ldx=2048, ldo=2048, out=A + 2046), "overlaps"), (dict(ldx=2048, ldo=2048, out=A + 2 * 2048 + 2046), "overlaps"),
    (dict(table=FAR + 4096), "overlaps table"), (dict(table=FAR - 2032), "overlaps table")])
def test_rotary_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _rotary(**kw)


def _store(**kw):
    a = dict(dt=BF16, k=A, v=FAR, ldk=1024, ldv=1024, table=A, slots=A, kc=A, vc=A, ks=A, vs=A, n=4, Hkv=8, hd=128, half=64, inter=0,
             page=64, n_pages=16, q=4 * FAR, ldq=4096, q_out=8 * FAR, ldqo=4096, Hq=32)
    a.update(kw)
    _lib.call("mh_kv_store_rotary_paged", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "dtype"), (dict(hd=24), "multiple of 16"), (dict(Hkv=0), "head count"), (dict(Hkv=65535), "head count"),
    (dict(page=100), "page holds"), (dict(n=-1), "negative"), (dict(n=(1 << 27) + 1), "one launch"), (dict(slots=None), "null slots"),
    (dict(k=None), "null k"), (dict(v=FAR + 8), "aligned"), (dict(ldk=1023), "multiple of 16"), (dict(table=None), "null table"),
    (dict(table=A + 8), "aligned"), (dict(half=0), "rotated part"), (dict(half=65), "rotated part"), (dict(kc=None), "null cache"),
    (dict(Hq=0), "query head"), (dict(Hq=1 << 24), "query head"), (dict(q_out=None), "null q_out"), (dict(q=4 * FAR + 2), "aligned"),
    (dict(ldq=4095), "multiple of 16"), (dict(ldqo=2048), "whole"), (dict(q_out=4 * FAR, ldqo=8192), "overlaps"),
    (dict(q_out=4 * FAR + 64), "overlaps"), (dict(k=8 * FAR), "overlaps"), (dict(v=8 * FAR + 4096), "overlaps"), (dict(ldk=1 << 58), "far apart"),
    (dict(table=8 * FAR + 4096), "overlaps table"), (dict(slots=8 * FAR - 12), "overlaps table or slots")])
def test_kv_store_rotary_paged_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _store(**kw)


def _quant(**kw):
    a = dict(dt=BF16, x=A, ldx=100, q=FAR, ldq=100, scale=A, rows=4, cols=100)
    a.update(kw)
    _lib.call("mh_quantize_rows", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "dtype"), (dict(rows=-1), "bad row count"), (dict(cols=0), "empty rows"), (dict(x=None), "null x"), (dict(q=None), "null q"),
    (dict(scale=None), "null scale"), (dict(x=A + 1), "aligned to its type"), (dict(ldx=99), "whole"), (dict(ldq=99), "whole"),
    (dict(q=A + 50), "overlaps"), (dict(ldq=1 << 60), "far apart"), (dict(scale=FAR + 16), "scale overlaps"), (dict(scale=A + 796), "scale overlaps"),
    (dict(scale=4 * FAR + 2), "aligned to its type")])
def test_quantize_rows_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _quant(**kw)


def _dequant(**kw):
    a = dict(dt=BF16, q=A, ldq=100, scale=A, out=FAR, ldo=100, rows=4, cols=100)
    a.update(kw)
    _lib.call("mh_dequantize_rows", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "dtype"), (dict(rows=-1), "bad row count"), (dict(cols=0), "empty rows"), (dict(q=None), "null q"), (dict(out=None), "null out"),
    (dict(scale=None), "null scale"), (dict(out=FAR + 1), "aligned to its type"), (dict(ldo=99), "whole"), (dict(ldq=99), "whole"),
    (dict(out=A + 50), "overlaps"), (dict(scale=FAR + 796), "overlaps scale"), (dict(scale=FAR - 1), "aligned to its type")])
def test_dequantize_rows_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _dequant(**kw)


def _linear(**kw):
    a = dict(dt=BF16, x=A, ldx=512, sx=A, w=FAR, ldw=512, sw=A, bias=None, resid=None, ldr=0, out=4 * FAR, ldo=64, M=8, N=64, K=512, act=0)
    a.update(kw)
    _lib.call("mh_linear_i8", *a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=3), "dtype"), (dict(act=3), "activation"), (dict(act=-1), "activation"), (dict(M=-1), "negative"), (dict(N=-1), "negative"),
    (dict(K=0), "empty rows"), (dict(K=1 << 17, ldx=1 << 17, ldw=1 << 17), "32 bits"), (dict(M=1 << 22, N=1 << 13, ldo=1 << 13), "one launch"),
    (dict(x=None), "null x"), (dict(w=None), "null w"), (dict(out=None), "null out"), (dict(sx=None), "null scale"), (dict(sw=None), "null scale"),
    (dict(ldx=511), "whole"), (dict(ldw=100), "whole"), (dict(ldo=63), "whole"), (dict(out=4 * FAR + 1), "aligned to its type"),
    (dict(bias=A + 1), "aligned to its type"), (dict(resid=A + 1, ldr=64), "aligned to its type"), (dict(resid=A, ldr=63), "whole"),
    (dict(resid=4 * FAR, ldr=65), "overlaps the residual"), (dict(resid=4 * FAR + 2, ldr=64), "overlaps the residual"),
    (dict(x=4 * FAR + 100), "overlaps x or w"), (dict(w=4 * FAR - 100), "overlaps x or w"), (dict(ldx=1 << 57), "far apart"),
    (dict(sx=4 * FAR + 8), "overlaps a scale"), (dict(sw=4 * FAR - 252), "overlaps a scale"), (dict(bias=4 * FAR + 1022), "or the bias"),
    (dict(sx=A + 2), "aligned to its type"), (dict(sw=A + 1), "aligned to its type")])
def test_linear_i8_refusals(kw, match):
    with pytest.raises(_lib.HipError, match=match):
        _linear(**kw)


def test_tile_rules(tmp_path):
    exe = str(tmp_path / "check")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", build.CSRC,
                        os.path.join(root, "tests", "cxx", "gemm_i8_tiles_check.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr[-2000:]


def test_empty_calls_need_no_device():
    _table(n=0)
    _rotary(n=0)
    _store(n=0)
    _quant(rows=0)
    _dequant(rows=0)
    _linear(M=0)
    _linear(N=0)


def test_tensors_must_share_a_gpu():
    torch = pytest.importorskip("torch")
    from munet_amd.backend import HipBackend
    hip = HipBackend.__new__(HipBackend)  # (no device here)
    x, q, s = torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: hip.quantize_rows(x, q, s), lambda: hip.dequantize_rows(q, s, x), lambda: hip.linear_i8(q, s, q, s, x),
                 lambda: hip.rotary(x[None], x[None], x[None]), lambda: hip.rotary_table(s.int(), s.double(), x[None])):
        with pytest.raises(ValueError, match="one GPU"):
            call()
