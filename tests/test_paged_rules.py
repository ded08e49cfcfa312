"""How calls over the paged KV cache are cut, run on the host under the
undefined-behaviour sanitizer (CPU)."""
import os
import subprocess

from munet_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_paged_cut_rules(tmp_path):
    exe = str(tmp_path / "check")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-D__host__=",
                        "-D__device__=", "-D__forceinline__=inline", "-I", build.CSRC,
                        os.path.join(ROOT, "tests", "cxx", "paged_cut_check.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr[-2000:]
