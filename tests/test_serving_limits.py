"""Limits of the serving calls: sizes and settings just past them are refused
before anything reaches a device (CPU)."""
import pytest

from munet_amd import _lib
from test_serving_args import _attend


@pytest.mark.parametrize("scale", [2.0 ** 127 * 1.0001, -3e38, 3.4e38])
def test_scales_that_pass_a_float_in_base_two(scale):
    with pytest.raises(_lib.HipError, match="2\\^127"):
        _attend(scale=scale)
