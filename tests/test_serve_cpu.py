"""Refusals of the rotated write, the 4-bit pages and the verification of drafts that
need no GPU: argument errors of the C entries before any HIP call, and of the Python operators."""

import pytest
import torch

import sparda
from sparda import _lib

P = 4096  # any aligned non-null value: validation fails before it is dereferenced


def _expect(code, name, args):
    with pytest.raises(sparda.SpardaArgumentError) as ei:
        _lib.call(name, *args)
    assert ei.value.code == code
    assert sparda.load().sparda_last_error()


def rotate(k=P, v=P, dtype=1, pages=10, ps=64, p_st=16384, s_st=256, h_st=64, table=P, t_st=8, width=8, pos=P, cu=None,
           n=4, q=P, q_st=768, q_sh=64, Hq=12, kn=P, vn=P, N=4, new_st=256, new_sh=64, Hkv=4, D=64, cos=P, sin=P, cs=32,
           rows=100, qo=P, qo_st=768, qo_sh=64):
    return (k, v, dtype, pages, ps, p_st, s_st, h_st, table, t_st, width, pos, cu, n, q, q_st, q_sh, Hq, kn, vn, N, new_st,
            new_sh, Hkv, D, cos, sin, cs, rows, qo, qo_st, qo_sh, None)


def append(pages=P, n_pages=10, ps=64, p_st=18432, h_st=4608, table=P, t_st=8, width=8, pos=P, cu=None, n=4, q=P, q_st=768,
           q_sh=64, Hq=12, kn=P, vn=P, dtype=1, N=4, new_st=256, new_sh=64, Hkv=4, D=64, cos=P, sin=P, cs=32, rows=100,
           qo=P, qo_st=768, qo_sh=64):
    return (pages, n_pages, ps, p_st, h_st, table, t_st, width, pos, cu, n, q, q_st, q_sh, Hq, kn, vn, dtype, N, new_st,
            new_sh, Hkv, D, cos, sin, cs, rows, qo, qo_st, qo_sh, None)


def gather(pages=P, n_pages=10, ps=64, p_st=18432, h_st=4608, table=P, t_st=8, width=8, pos=P, cu=None, n=4, k=P, v=P,
           dtype=1, N=4, st=256, sh=64, Hkv=4, D=64):
    return (pages, n_pages, ps, p_st, h_st, table, t_st, width, pos, cu, n, k, v, dtype, N, st, sh, Hkv, D, None)


def decode(q=P, q_sb=3840, q_st=768, q_sh=64, dtype=1, pages=P, n_pages=10, ps=64, p_st=18432, h_st=4608, table=P, t_st=8,
           width=8, lens=P, B=4, T=5, Hq=12, Hkv=4, D=64, out=P, out_sb=3840, ws=P, nbytes=1 << 40):
    return (q, q_sb, q_st, q_sh, dtype, pages, n_pages, ps, p_st, h_st, table, t_st, width, lens, B, T, Hq, Hkv, D, 0.125,
            out, out_sb, ws, nbytes, None)


def verify(logits=P, dtype=1, l_sb=5000, l_st=1000, drafts=P, d_sb=4, uniform=P, u_sb=5, probs=P, p_sb=4000, p_st=1000,
           counts=P, each=None, temperature=1.0, B=3, K=4, V=1000, tokens=P, accepted=P, ws=P, nbytes=1 << 40):
    return (logits, dtype, l_sb, l_st, drafts, d_sb, uniform, u_sb, probs, p_sb, p_st, counts, each, temperature, B, K, V,
            tokens, accepted, ws, nbytes, None)


CACHE = [(-2, dict(ps=8)), (-2, dict(ps=40)), (-2, dict(ps=0)), (-2, dict(width=0)), (-2, dict(Hkv=0)), (-2, dict(D=80)),
         (-2, dict(width=1 << 26)), (-5, dict(t_st=-1)), (-3, dict(dtype=7)), (-1, dict(table=None))]
Q4 = CACHE + [(-2, dict(n_pages=0)), (-2, dict(n_pages=1 << 31)), (-5, dict(p_st=-18432)), (-5, dict(p_st=18440)),
              (-5, dict(h_st=4600)), (-5, dict(pages=P + 8)), (-1, dict(pages=None))]
ROWS = [(-1, dict(pos=None)), (-2, dict(n=0, N=0)), (-2, dict(N=5)), (-2, dict(cu=P, n=(1 << 30) + 1)), (-2, dict(cu=P, N=0)),
        (-2, dict(cu=P, N=1 << 31))]
NEW = ROWS + [(-1, dict(kn=None)), (-1, dict(vn=None)), (-5, dict(kn=P + 8)), (-5, dict(new_st=252)), (-5, dict(new_sh=63)),
              (-1, dict(cos=None)), (-1, dict(sin=None)), (-1, dict(q=None)), (-1, dict(qo=None)), (-2, dict(rows=0)),
              (-2, dict(Hq=-1)), (-2, dict(Hq=1 << 17)), (-5, dict(cos=P + 8)), (-5, dict(cs=30)), (-5, dict(cs=-32)),
              (-5, dict(q=P + 4)), (-5, dict(q_st=764)), (-5, dict(qo=P + 8)), (-5, dict(qo_st=0)), (-5, dict(qo_sh=32)),
              (-5, dict(qo_st=384)), (-5, dict(qo_st=-768))]


@pytest.mark.parametrize("code,bad", CACHE + NEW + [
    (-1, dict(k=None)), (-1, dict(v=None)), (-2, dict(pages=0)), (-2, dict(pages=1 << 31)), (-5, dict(k=P + 8)),
    (-5, dict(s_st=260)), (-5, dict(h_st=65)), (-5, dict(p_st=-16384))], ids=str)
def test_rotate_append_argument_errors(code, bad):
    _expect(code, "sparda_rotate_append_paged", rotate(**bad))


@pytest.mark.parametrize("code,bad", Q4 + NEW + [(-1, dict(cos=None, sin=None))], ids=str)
def test_append_q4_argument_errors(code, bad):
    _expect(code, "sparda_append_paged_q4", append(**bad))


@pytest.mark.parametrize("code,bad", Q4 + ROWS + [
    (-1, dict(k=None)), (-1, dict(v=None)), (-5, dict(k=P + 8)), (-5, dict(st=252)), (-5, dict(sh=32)), (-5, dict(st=128)),
    (-5, dict(st=-256))], ids=str)
def test_gather_q4_argument_errors(code, bad):
    _expect(code, "sparda_gather_paged_q4", gather(**bad))


@pytest.mark.parametrize("code,bad", Q4 + [
    (-1, dict(q=None)), (-1, dict(lens=None)), (-1, dict(out=None)), (-2, dict(B=0)), (-2, dict(B=1 << 17)),
    (-2, dict(Hq=14)), (-2, dict(Hq=0)), (-2, dict(T=0)), (-2, dict(T=65)), (-2, dict(T=64, Hq=1024)),
    (-2, dict(B=65535, width=1 << 24)), (-5, dict(q=P + 4)), (-5, dict(q_sb=3836)), (-5, dict(q_st=764)),
    (-5, dict(q_sh=60)), (-5, dict(out_sb=3839)), (-4, dict(ws=None, width=64)), (-4, dict(nbytes=16, width=64)),
    (-4, dict(ws=P + 8, width=64))], ids=str)
def test_decode_q4_argument_errors(code, bad):
    _expect(code, "sparda_decode_paged_q4", decode(**bad))


@pytest.mark.parametrize("code,bad", [
    (-1, dict(logits=None)), (-1, dict(drafts=None)), (-1, dict(uniform=None)), (-1, dict(tokens=None)),
    (-1, dict(accepted=None)), (-3, dict(dtype=2)), (-2, dict(B=0)), (-2, dict(K=-1)), (-2, dict(K=65)), (-2, dict(V=0)),
    (-2, dict(V=1 << 21)), (-2, dict(B=20000)), (-2, dict(temperature=-1.0)), (-2, dict(temperature=float("nan"))),
    (-2, dict(temperature=float("inf"))), (-5, dict(logits=P + 1)), (-5, dict(l_sb=-1)), (-5, dict(p_st=-1000)),
    (-5, dict(u_sb=-5)), (-4, dict(ws=None)), (-4, dict(nbytes=16)), (-4, dict(ws=P + 8))], ids=str)
def test_verify_argument_errors(code, bad):
    _expect(code, "sparda_verify_drafts", verify(**bad))


def test_workspace_sizes():
    ws = sparda.load().sparda_decode_paged_q4_workspace_bytes
    assert ws(1, 1, 1, 16, 12, 4, 64, 1) == 0            # one share a sequence: no partials
    some = ws(8, 1, 256, 64, 12, 4, 64, 1)
    assert some > 0 and some % (12 * 66 * 4) == 0     # (m, l, o[D]) fp32 for each item and head
    assert ws(0, 1, 256, 64, 12, 4, 64, 1) == 0 and ws(8, 0, 256, 64, 12, 4, 64, 1) == 0 and ws(8, 1, 256, 64, 2, 4, 64, 1) == 0
    ws = sparda.load().sparda_verify_drafts_workspace_bytes
    assert ws(1, 4, 32000, 1) > 0 and ws(1, 65, 32000, 1) == 0 and ws(0, 4, 32000, 1) == 0 and ws(1, 4, 1 << 21, 1) == 0


def test_page_shape():
    assert sparda.q4_page_shape(7, 64, 4, 128) == (7, 4, 4, 2304)
    assert sparda.q4_page_shape(7, 16, 4, 16) == sparda.q4_page_shape(7, 16, 4, 32) == (7, 4, 1, 576)
    for bad in ((7, 24, 4, 64), (7, 0, 4, 64), (7, 16, 4, 48)):
        with pytest.raises(ValueError):
            sparda.q4_page_shape(*bad)


def test_operators_refuse_cpu_tensors():
    q, kv = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64)
    pages, table, n = torch.zeros(3, 16, 1, 64), torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    q4, angles = torch.zeros(sparda.q4_page_shape(3, 16, 1, 64), dtype=torch.uint8), torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.rotate_append_paged(pages, pages, table, n, q, kv, kv, angles, angles)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.append_paged_q4(q4, table, n, kv, kv)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.gather_paged_q4(q4, table, n, 4)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.decode_paged_q4(q, q4, table, n)
    with pytest.raises(RuntimeError, match="GPU device"):
        sparda.verify_drafts(torch.zeros(4, 2, 10), torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 2))
