"""Grids and sums of the rotated write, the 4-bit pages and the verification of drafts that would not
fit, refused before any HIP call (no GPU needed)."""

import pytest

import sparda
from test_serve_cpu import P, _expect, append, decode, gather, rotate, verify

ROWS = [(1 << 26) - 3, 1 << 26, (1 << 31) - 1]


# A launch counts its threads in 32 bits: 2^24 workgroups of 256, four rows each.
@pytest.mark.parametrize("cu", [None, P])
@pytest.mark.parametrize("N", ROWS)
@pytest.mark.parametrize("name,args", [("sparda_rotate_append_paged", rotate), ("sparda_append_paged_q4", append),
                                       ("sparda_gather_paged_q4", gather)], ids=["rotate", "append", "gather"])
def test_rows_past_32_bit_grids(name, args, N, cu):
    _expect(-2, name, args(N=N, n=N if cu is None else 4, cu=cu))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("bad", [dict(B=16, width=(1 << 25) - 1, ps=64), dict(B=65535, T=1, width=1 << 12, ps=128),
                                 dict(B=1, width=(1 << 27) - 1, ps=16), dict(B=65535, T=1, Hq=4096, Hkv=4096, width=1),
                                 dict(B=65535, T=64, Hq=1023, Hkv=1, width=64)], ids=str)
def test_decode_q4_grids_and_positions(bad, dtype):
    _expect(-2, "sparda_decode_paged_q4", decode(dtype=dtype, out_sb=1 << 30, nbytes=1 << 60, **bad))


@pytest.mark.parametrize("bad", [dict(B=65536, K=0), dict(B=1009, K=64), dict(B=1, K=65), dict(V=(1 << 20) - 7), dict(B=1 << 40)], ids=str)
def test_verify_rows_and_vocabularies(bad):
    _expect(-2, "sparda_verify_drafts", verify(nbytes=1 << 60, **bad))
    sizes = {**dict(B=3, K=4, V=1000), **bad}
    assert sparda.load().sparda_verify_drafts_workspace_bytes(sizes["B"], sizes["K"], sizes["V"], 1) == 0


@pytest.mark.parametrize("dtype", [0, 1])
def test_workspaces_cover_what_the_kernels_write(dtype):
    """A workspace of a byte less than asked for is refused, whatever the sizes."""
    lib = sparda.load()
    for B, T, width, ps, Hq, Hkv, D in ((1, 1, 4000, 16, 12, 4, 64), (3, 5, 700, 64, 32, 8, 128), (200, 1, 300, 16, 8, 1, 128)):
        need = lib.sparda_decode_paged_q4_workspace_bytes(B, T, width, ps, Hq, Hkv, D, dtype)
        assert need >= B * T * Hq * (D + 2) * 4
        _expect(-4, "sparda_decode_paged_q4", decode(dtype=dtype, B=B, T=T, width=width, ps=ps, Hq=Hq, Hkv=Hkv, D=D, q_sb=T * Hq * D,
                                                     q_st=Hq * D, q_sh=D, out_sb=T * Hq * D, nbytes=need - 1))
    for B, K, V in ((1, 0, 1), (64, 7, 50257), (1000, 64, 300), (2, 1, (1 << 20) - 8)):
        need = lib.sparda_verify_drafts_workspace_bytes(B, K, V, dtype)
        _expect(-4, "sparda_verify_drafts", verify(dtype=dtype, B=B, K=K, V=V, nbytes=need - 1))
