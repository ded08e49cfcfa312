"""Frequencies outside the floats are refused, wherever the arguments alone are in order (CPU)."""
import numpy as np
import pytest

from munet_amd import _lib
from munet_amd.backend import rotary_frequencies


@pytest.mark.parametrize("args", [
    (64, 1e4, "linear", 1e-320), (64, 1e-300, "base", 1e-300), (64, 1e300, "base", 1e300), (4, 1e200, "base", 1e100),
    (64, 1e4, "turns", 1e-320, 4096), (64, 1e-320)])
def test_frequencies_out_of_range(args):
    with pytest.raises(_lib.HipError, match="out of range"):
        rotary_frequencies(*args)


# (a factor of 1e-310 makes a base of 10^4 10^(-310 * 64 / 62) = 10^-316, whose least power is 10^(316 * 62 / 64) = 10^306)
@pytest.mark.parametrize("args", [(64, 1e308), (2, 1e-320), (64, 1e4, "linear", 1e300), (64, 1e200, "base", 1e60), (64, 1e4, "turns", 1e300, 1e300),
                                  (64, 1e-4), (64, 1e4, "linear", 1e-290), (64, 1e4, "base", 1e-310)])
def test_frequencies_at_the_ends(args):
    freq, m = rotary_frequencies(*args)
    assert np.isfinite(freq).all() and (freq > 0).all() and np.isfinite(m)
