"""Static check of the waits of the int8 products' direct-to-LDS pipelines (CPU; needs hipcc).

gemm_i8_kernel issues a slab's loads with inline assembly (buffer_load_dwordx4 ...
lds) and waits for them by a count: before the first product the loads of slabs
0 .. S - 2 are out and slab 0 must be there, and in every step the loads of one more
slab go out and the next one must be there.  vmcnt counts outstanding loads, which
complete in order, so with L loads a slab each wait may leave L (S - 2) out, none
with two stages.  The kernels are compiled to gfx950 assembly, whose barriers are
three: behind the prologue, in the first step and in the loop's body."""
import os
import re

import pytest

from test_dma_wait_counts import HIPCC, _asm

KINDS = [(r"buffer_load_dwordx4 .* lds$", "load"), (r"s_waitcnt\b.*vmcnt\(\d+\)", "wait"), (r"s_barrier\b", "barrier"),
         (r"(global|buffer|flat|scratch)_(load|store|atomic)", "memory")]


def events(body):
    out = []
    for line in body.splitlines():
        line = line.strip()
        kind = next((k for pattern, k in KINDS if re.match(pattern, line)), None)
        if kind == "wait":
            kind = int(re.search(r"vmcnt\((\d+)\)", line).group(1))
        if kind is not None:
            out.append(kind)
    return out


def check(found, loads, stages):
    """Whether the events up to the end of the loop are as they have to be."""
    at = 0
    for want in (loads * (stages - 1), loads, loads):  # behind the prologue, the first step, the loop's body
        end = found.index("barrier", at)
        part = found[at:end]
        assert part.count("load") == want, (part, want)
        assert "memory" not in part, part
        # the wait before the barrier, behind the part's loads
        assert isinstance(part[-1], int) and part[-1] <= loads * (stages - 2), (part, loads, stages)
        at = end + 1
    rest = found[at:]
    assert "barrier" not in rest and "load" not in rest
    assert rest[0] == 0  # nothing is in flight when the results are stored


def test_check_sees_planted_mistakes():
    good = ["load"] * 6 + [3, "barrier"] + ["load"] * 3 + [3, "barrier"] + ["load"] * 3 + [3, "barrier", 0, "memory"]
    check(good, 3, 3)
    for at, what in ((6, 4), (11, 4), (16, 6), (18, 1), (0, "memory"), (8, "memory"), (16, "load"), (13, 3)):
        bad = list(good)
        bad[at] = what
        with pytest.raises((AssertionError, ValueError)):
            check(bad, 3, 3)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_waits_cover_the_slabs(tmp_path):
    s = _asm("gemm_i8.hip", tmp_path)
    seen = set()
    for m in re.finditer(r"^(_Z\S*gemm_i8_kernelI((?:Li\d+E)+)E\S*):", s, re.M):
        dt, bm, bn, wgm, wgn, stages = tile = tuple(int(v) for v in re.findall(r"Li(\d+)E", m.group(2)))
        check(events(s[m.end():s.index(".Lfunc_end", m.end())]), (bm + bn) // 8 // (wgm * wgn), stages)
        seen.add(tile)
    assert len(seen) == 27, len(seen)  # nine tiles, three types
