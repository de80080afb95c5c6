"""Limits of the packed and paged operators, checked before any HIP call (no GPU needed)."""

import pytest

from test_packed_paged_cpu import _expect, decode


# Full sequences of these capacities would carry the kernels' 32-bit sums past 2^31: the steps
# of the batch and the number of shares, and a last position and the step that holds it.
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("bad", [dict(B=16, width=(1 << 25) - 1, ps=64), dict(B=9, width=(1 << 25) - 1, ps=64),
                                 dict(B=65535, width=1 << 12, ps=128), dict(B=1, width=(1 << 27) - 1, ps=16),
                                 dict(B=1, width=44739242, ps=48)], ids=str)
def test_decode_paged_refuses_more_positions_than_its_sums_hold(bad, dtype):
    _expect(-2, "sparda_decode_paged", *decode(dtype=dtype, **bad))
