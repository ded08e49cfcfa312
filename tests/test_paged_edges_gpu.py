"""Attention over the paged 8-bit KV cache where its forms meet their ends: joins
of odd cuts, values that are not numbers, masks that differ from wave to wave, pages
nobody wrote.  Against the formula in 64 bits, with the tolerance of
test_paged_gpu.py."""
import pytest

from test_paged_gpu import Cache, check, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd,keys", [(128, 2400), (128, 3000), (80, 2400), (80, 8100), (176, 1500)])
def test_joins_that_leave_threads_over(torch, hip, dtype, hd, keys):  # noqa: F811
    """Head sizes and shares whose product does not divide the joining workgroup."""
    check(torch, hip, Cache(torch, 1, hd, 64, [keys, 70], [1, 1], seed=hd), 2, dtype, what="join")
