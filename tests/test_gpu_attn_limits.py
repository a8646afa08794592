"""Attention over a paged cache at the ends of its arguments' ranges, on the GPU against the plain form in 64
bits."""

import pytest

from test_gpu_attn_paged import NAMES, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 5, 2 ** 31 - 1])
def test_widest_windows(gpu, name, window):
    """Windows past every length, with queries that stand before every key beside others, for both kernels."""
    Case(name, [(4, 1), (3, 200), (7, 2)], 4, 2, 64, window=window).run().check()
    Case(name, [(9, 4), (40, 7), (70, 1), (33, 300)], 4, 2, 64, window=window).run().check()
