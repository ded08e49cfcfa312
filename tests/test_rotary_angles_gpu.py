"""Tables at far positions, against angles that are reduced in exact arithmetic.

The angle position * frequency is a whole number times a 53-bit one, exact in
rational numbers, and is reduced there by 2 pi to 64 digits; what is left goes through a
64-bit cosine and sine.

Tolerance.  Of the values v = m cos a and m sin a: half a step of float32 (2^-24 |v|),
and what 64 bits may add behind an exact reduction to an eighth of a turn: the
rounding of the remainder in turns, of at most a half (2^-54 turns, 2^-51.3 rad), that
of 2 pi and the product with it (2 * 2^-53 * pi / 4), and a dozen roundings of the
series, below 2^-49 m in all; m is below 2 here: 2^-48.  The reference's own remainder
and library calls are off by 2^-51.  (An angle whose product or frequency in turns is
rounded to 64 bits is off by up to 2^-25 of a turn at 2^31 positions: three times what
this allows.)"""
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923, 10 ** 64)


def exact(pos, freq):
    """(cos, sin) [n, half] of the exact products."""
    turn, out = 2 * PI, np.empty((len(pos), len(freq), 2))
    for j, f in enumerate(freq):
        step = Fraction(float(f))
        for t, p in enumerate(pos):
            a = step * int(p)
            a = float(a - turn * round(a / turn))
            out[t, j] = np.cos(a), np.sin(a)
    return out


@pytest.mark.parametrize("base,scaling,factor", [(10000.0, None, 1.0), (500000.0, "turns", 8.0), (10000.0, "linear", 0.125),
                                                 (10000.0, "base", 32.0)])
@pytest.mark.parametrize("far", [2 ** 31, 10 ** 7, 131072])
def test_far_angles(hip, base, scaling, factor, far):
    import torch
    from munet_amd.backend import rotary_frequencies
    freq, m = rotary_frequencies(64, base, scaling, factor, 4096)
    rng = np.random.default_rng(far % 1009)
    pos = rng.integers(-far, far, 97).astype(np.int32)
    pos[:4] = [-far, far - 1, 710, 0]
    table = torch.empty((len(pos), 32, 2), device="cuda")
    hip.rotary_table(torch.from_numpy(pos).cuda(), torch.from_numpy(freq).cuda(), table, magnitude=m)
    want = exact(pos, freq) * m
    off = np.abs(table.double().cpu().numpy() - want)
    tol = 2.0 ** -24 * np.abs(want) + 2.0 ** -48
    assert (off <= tol).all(), (int((off > tol).sum()), off.max())
