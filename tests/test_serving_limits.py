"""Limits of the serving calls: sizes and settings just past them are refused
before anything reaches a device (CPU)."""
import ctypes

import pytest

from munet_amd import _lib
from test_serving_args import _attend, _plan, _sample


@pytest.mark.parametrize("scale", [2.0 ** 127 * 1.0001, -3e38, 3.4e38])
def test_scales_that_pass_a_float_in_base_two(scale):
    with pytest.raises(_lib.HipError, match="2\\^127"):
        _attend(scale=scale)


@pytest.mark.parametrize("cols", [2 ** 31 - 2 ** 21 + 1, 2 ** 31 - 1])
def test_rows_of_tokens_past_32_bits(cols):
    """Indexes past a row's last token would wrap."""
    with pytest.raises(_lib.HipError, match="2\\^31 - 2\\^21"):
        _sample(cols=cols, ld=1 << 40, rows=1)
    n = ctypes.c_size_t()
    with pytest.raises(_lib.HipError, match="2\\^31 - 2\\^21"):
        _lib.call("mh_sample_workspace", 0, 1, cols, ctypes.byref(n))
    _lib.call("mh_sample_workspace", 0, 1, 2 ** 31 - 2 ** 21, ctypes.byref(n))


def test_launch_limits():
    """More workgroups than a launch has are refused by name where tiles cannot be walked instead."""
    with pytest.raises(_lib.HipError, match="one launch takes"):
        _attend(B=1 << 21, n_rows=1 << 21)
    n = ctypes.c_size_t()

    def workspace(n_rows):
        _lib.call("mh_attention_paged_workspace", 2, 1, n_rows, 16, 16, 256, 1, 100000, 0, ctypes.byref(n))
        return n.value

    assert workspace(1 << 16) > 0
    assert workspace(1 << 26) == 0  # (rows that pad the batch, more than one launch joins: no shares)


def test_plans_of_millions_of_requests():
    """Work that grows with the square of the requests ends in time."""
    with pytest.raises(_lib.HipError, match="one launch takes"):
        _plan(B=(1 << 20) + 1)
