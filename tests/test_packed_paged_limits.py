"""Limits of the packed and paged operators, checked before any HIP call (no GPU needed)."""

import pytest

from test_packed_paged_cpu import _expect, append, decode, packed


# Full sequences of these capacities would carry the kernels' 32-bit sums past 2^31: the steps
# of the batch and the number of shares, and a last position and the step that holds it.
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("bad", [dict(B=16, width=(1 << 25) - 1, ps=64), dict(B=9, width=(1 << 25) - 1, ps=64),
                                 dict(B=65535, width=1 << 12, ps=128), dict(B=1, width=(1 << 27) - 1, ps=16),
                                 dict(B=1, width=44739242, ps=48)], ids=str)
def test_decode_paged_refuses_more_positions_than_its_sums_hold(bad, dtype):
    _expect(-2, "sparda_decode_paged", *decode(dtype=dtype, **bad))


# A launch counts its threads in 32 bits: 2^24 workgroups of 256, one for 16 to 256 (row, head) pairs of a sequence (prefill),
# for 4 rows (append), for a share and 1 to 4 heads (decode).
@pytest.mark.parametrize("bad", [dict(dtype=0, N=1 << 25, Hq=32, Hkv=8, D=16), dict(dtype=0, N=1 << 24, Hq=32, Hkv=8, D=32),
                                 dict(n=1 << 24, N=1000), dict(n=1 << 30, N=1 << 20), dict(D=128, n=1 << 22), dict(D=16, n=1 << 22),
                                 dict(N=1 << 28, Hq=32, Hkv=8), dict(Hq=65532, Hkv=65532, N=1 << 15, out_st=65532 * 64, dtype=0)], ids=str)
def test_prefill_packed_refuses_grids_past_32_bits(bad):
    bad.setdefault("out_st", bad.get("Hq", 12) * bad.get("D", 64))
    _expect(-2, "sparda_prefill_packed", *packed(**bad))


@pytest.mark.parametrize("cu", [None, 4096])
@pytest.mark.parametrize("N", [(1 << 26) - 3, 1 << 26, (1 << 31) - 1])
def test_append_paged_refuses_grids_past_32_bits(N, cu):
    _expect(-2, "sparda_append_paged", *append(N=N, n=N if cu is None else 4, cu=cu))


@pytest.mark.parametrize("bad", [dict(B=65535, Hq=4096, Hkv=4096, width=1), dict(B=65535, Hq=2048, Hkv=1024, width=64)], ids=str)
def test_decode_paged_refuses_grids_past_32_bits(bad):
    _expect(-2, "sparda_decode_paged", *decode(out_sb=bad["Hq"] * 64, nbytes=1 << 60, **bad))
