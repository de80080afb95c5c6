"""Refusals of the packed and paged operators that need no GPU: argument errors
of the C entries before any HIP call, and of the Python operators."""

import pytest
import torch

import sparda
from sparda import _lib

P = 4096  # any aligned non-null value: validation fails before it is dereferenced


def _expect(code, name, *args):
    with pytest.raises(sparda.SpardaArgumentError) as ei:
        _lib.call(name, *args)
    assert ei.value.code == code
    assert sparda.load().sparda_last_error()


def packed(q=P, k=P, v=P, dtype=1, cu=P, n=2, N=100, Hq=12, Hkv=4, D=64, out=P, out_st=768, q_st=768, q_sh=64, kv_st=256,
           kv_sh=64):
    return (q, q_st, q_sh, k, v, kv_st, kv_sh, dtype, cu, n, N, Hq, Hkv, D, 1, 0.125, out, out_st, None)


@pytest.mark.parametrize("code,bad", [
    (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(cu=None)), (-1, dict(out=None)),
    (-3, dict(dtype=2)), (-2, dict(n=0)), (-2, dict(N=0)), (-2, dict(Hq=0)), (-2, dict(Hkv=0)), (-2, dict(D=48)),
    (-2, dict(Hq=13)), (-2, dict(N=1 << 31)), (-2, dict(Hq=1 << 17)), (-5, dict(out_st=767)),
    (-2, dict(n=(1 << 30) + 1)), (-2, dict(N=1 << 30, out_st=1 << 20)), (-5, dict(q=P + 8)), (-5, dict(k=P + 2)),
    (-5, dict(v=P + 4)), (-5, dict(out=P + 8)), (-5, dict(out_st=772)), (-5, dict(q_st=772)), (-5, dict(q_sh=66)),
    (-5, dict(kv_sh=65)), (-5, dict(kv_st=260)), (-5, dict(kv_st=-256)), (-5, dict(kv_st=1 << 24))], ids=str)
def test_prefill_packed_argument_errors(code, bad):
    _expect(code, "sparda_prefill_packed", *packed(**bad))


def append(k=P, v=P, dtype=1, pages=10, ps=64, p_st=16384, s_st=256, h_st=64, table=P, t_st=8, width=8, pos=P, cu=None,
           n=4, kn=P, vn=P, N=4, new_st=256, new_sh=64, Hkv=4, D=64):
    return (k, v, dtype, pages, ps, p_st, s_st, h_st, table, t_st, width, pos, cu, n, kn, vn, N, new_st, new_sh, Hkv, D,
            None)


PAGES = [
    (-3, dict(dtype=7)), (-2, dict(pages=0)), (-2, dict(ps=8)), (-2, dict(ps=40)), (-2, dict(ps=0)), (-2, dict(width=0)),
    (-2, dict(Hkv=0)), (-2, dict(D=80)), (-2, dict(width=1 << 26)), (-2, dict(pages=1 << 31)), (-5, dict(p_st=-16384)),
    (-5, dict(s_st=260)), (-5, dict(h_st=65)), (-5, dict(p_st=4)), (-5, dict(k=P + 8)), (-5, dict(v=P + 2)),
    (-5, dict(t_st=-1)), (-5, dict(s_st=1 << 26))]


@pytest.mark.parametrize("code,bad", PAGES + [
    (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(table=None)), (-1, dict(pos=None)), (-1, dict(kn=None)),
    (-1, dict(vn=None)), (-2, dict(n=0, N=0)), (-2, dict(N=5)), (-2, dict(cu=P, n=(1 << 30) + 1)), (-2, dict(cu=P, N=0)), (-5, dict(kn=P + 8)),
    (-5, dict(new_st=252)), (-5, dict(new_sh=63))], ids=str)
def test_append_paged_argument_errors(code, bad):
    _expect(code, "sparda_append_paged", *append(**bad))


def decode(q=P, q_sb=768, q_sh=64, k=P, v=P, dtype=1, pages=10, ps=64, p_st=16384, s_st=256, h_st=64, table=P, t_st=8,
           width=8, lens=P, B=4, Hq=12, Hkv=4, D=64, out=P, out_sb=768, ws=P, nbytes=1 << 40):
    return (q, q_sb, q_sh, k, v, dtype, pages, ps, p_st, s_st, h_st, table, t_st, width, lens, B, Hq, Hkv, D, 0.125, out,
            out_sb, ws, nbytes, None)


@pytest.mark.parametrize("code,bad", PAGES + [
    (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(table=None)), (-1, dict(lens=None)),
    (-1, dict(out=None)), (-2, dict(B=0)), (-2, dict(B=1 << 17)), (-2, dict(Hq=14)), (-2, dict(Hq=0)),
    (-2, dict(B=65535, width=1 << 24)), (-5, dict(q=P + 4)), (-5, dict(q_sb=764)), (-5, dict(q_sh=60)),
    (-5, dict(out_sb=700)), (-4, dict(ws=None, width=64)), (-4, dict(nbytes=16, width=64)),
    (-4, dict(ws=P + 8, width=64))], ids=str)
def test_decode_paged_argument_errors(code, bad):
    _expect(code, "sparda_decode_paged", *decode(**bad))


def test_paged_workspace_sizes():
    ws = sparda.load().sparda_decode_paged_workspace_bytes
    assert ws(1, 1, 16, 12, 4, 64, 1) == 0            # one share a sequence: no partials
    some = ws(8, 256, 64, 12, 4, 64, 1)
    assert some > 0 and some % (12 * 66 * 4) == 0     # (m, l, o[D]) fp32 for each item and head
    assert ws(0, 256, 64, 12, 4, 64, 1) == 0 and ws(8, 256, 64, 2, 4, 64, 1) == 0


def test_operators_refuse_cpu_tensors():
    q, kv = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64)
    pages, table = torch.zeros(3, 16, 1, 64), torch.zeros(4, 1, dtype=torch.int32)
    n = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.prefill_packed(q, kv, kv, n)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.append_paged(pages, pages, table, n, kv, kv)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.decode_paged(q, pages, pages, table, n)
