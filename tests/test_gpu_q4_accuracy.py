"""Attention over 4-bit pages against float64 in relative error (limits and their reasons: q4_accuracy): every form of the
kernel, lengths from a step to many shares, long walks of one wavefront, and keys that hold most of the weight at every kind
of border."""

import numpy as np
import pytest
import torch

import sparda
from helpers import np32
from q4_accuracy import LIMIT, aligned_queries, attend64, relative, walk_limit

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def limit(dtype):
    return LIMIT["bf16" if dtype == BF else "f32"]


def cache(lengths, ps, Hkv, D, seed):
    """Pages of N(0,1) rows in a random order, their table, and what they hold: [b] -> k, v [n,Hkv,D] float64."""
    g = torch.Generator().manual_seed(seed)
    width = max((n + ps - 1) // ps for n in lengths)
    table = torch.randperm(len(lengths) * width, generator=g).view(len(lengths), width).int().to(DEV)
    pages = torch.full(sparda.q4_page_shape(len(lengths) * width, ps, Hkv, D), 0xFF, dtype=torch.uint8, device=DEV)
    cu = torch.tensor([0, *np.cumsum(lengths)], dtype=torch.int32, device=DEV)
    pos = torch.zeros(len(lengths), dtype=torch.int32, device=DEV)
    N = int(cu[-1])
    k, v = (torch.randn(N, Hkv, D, generator=g).to(BF).to(DEV) for _ in range(2))
    sparda.append_paged_q4(pages, table, pos, k, v, cu)
    k, v = (x.double().cpu().numpy() for x in sparda.gather_paged_q4(pages, table, pos, N, cu, head_dim=D, dtype=F32))
    at = cu.tolist()
    return pages, table, [(k[at[b]:at[b + 1]], v[at[b]:at[b + 1]]) for b in range(len(lengths))]


def decode(q, pages, table, lengths):
    return sparda.decode_paged_q4(q.to(DEV), pages, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))


def worst(got, q, lengths, rows):
    """The largest relative error of a (sequence, token)."""
    B, T, Hq, D = q.shape
    got, q64 = np32(got).astype(np.float64).reshape(B, T, Hq, D), np32(q).astype(np.float64)
    off = 0.0
    for b, (k, v) in enumerate(rows):
        R = Hq // k.shape[1]
        for t in range(T):
            n = lengths[b] - T + 1 + t
            want = np.concatenate([attend64(q64[b, t, g * R:(g + 1) * R], k[:n, g], v[:n, g], D ** -0.5) for g in range(k.shape[1])])
            off = max(off, relative(got[b, t].ravel(), want.ravel()))
    return off


# columns of a KV head (query heads x tokens): one tile with its columns repeated, full, full and repeated, two full
FORMS = [(12, 4, 64, 1), (12, 2, 64, 2), (4, 1, 64, 5), (16, 2, 64, 4), (16, 4, 128, 1), (16, 2, 128, 1), (8, 2, 128, 5), (32, 2, 128, 2),
         (4, 2, 32, 1), (8, 2, 16, 3)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,T", FORMS)
@pytest.mark.parametrize("spread", [0.05, 2.0])
@pytest.mark.parametrize("lengths", [[70, 1000], [20011]], ids=str)
def test_relative_error(dtype, Hq, Hkv, D, T, spread, lengths):
    print(f"[case] q4 accuracy {dtype} {Hq}/{Hkv}x{D} T={T} {spread} {lengths}", flush=True)
    pages, table, rows = cache(lengths, 64, Hkv, D, seed=D + T)
    q = (torch.randn(len(lengths), T, Hq, D, generator=torch.Generator().manual_seed(3)) * spread).to(dtype)
    off = worst(decode(q, pages, table, lengths), q, lengths, rows)
    print(f"  off by {off:.2e}", flush=True)
    assert off <= limit(dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D,n", [(64, 32768), (128, 32768), (64, 524288)])
@pytest.mark.parametrize("spread", [0.05, 2.0])
def test_long_walks(dtype, D, n, spread):
    """256 KV heads (of the same rows: a head stride of 0) leave a sequence one item, so that a wavefront walks 256 steps, or
    4096."""
    ps, H = 64, 256
    print(f"[case] q4 long walks {dtype} {D} {n} {spread}", flush=True)
    pages, table, rows = cache([n], ps, 1, D, seed=D)
    pages = pages.expand(-1, H, -1, -1)
    q = (torch.randn(2, H, D, generator=torch.Generator().manual_seed(4)) * spread).to(dtype)
    got = decode(q, pages, table.expand(2, -1).contiguous(), [n, n])
    k, v = (torch.from_numpy(x[:, 0]).to(DEV) for x in rows[0])
    want = torch.softmax(q.to(DEV).double() @ k.T * D ** -0.5, -1) @ v
    off = relative(np32(got).reshape(2, H, D), want.cpu().numpy())
    off = np.sqrt((off * off).mean(-1)).max()                # rms over the heads of a sequence
    print(f"  off by {off:.2e}", flush=True)
    assert off <= (limit(BF) if dtype == BF else walk_limit(n // 128))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,D", [(8, 64), (4, 128), (16, 128), (16, 32)])
@pytest.mark.parametrize("n", [129, 2049, 20011])
def test_no_key_is_lost(dtype, Hq, D, n):
    """Every query holds one key: the last, the first, those at the ends of tiles, steps, pages, shares of every length. (One
    weight's rounding does not average out over keys: in bf16 it and the output's may both be the largest, 2^-8 each.)"""
    print(f"[case] q4 keys {dtype} {Hq}x{D} {n}", flush=True)
    pages, table, rows = cache([n], 48, 1, D, seed=n)
    k, v = rows[0][0][:, 0], rows[0][1][:, 0]
    at = sorted({p for s in (1, 16, 32, 48, 128, 256, 640) for m in (0, 1, 2, n // s // 2, n // s - 1, n // s) for p in (s * m - 1, s * m)
                 if 0 <= p < n} | {n - 1, n - 2})
    at += at[:-len(at) % Hq]
    for i in range(0, len(at), Hq):
        q = torch.from_numpy(aligned_queries(k, at[i:i + Hq], D ** -0.5)).to(dtype)[None]
        got = np32(decode(q, pages, table, [n])).astype(np.float64).reshape(Hq, D)
        want = attend64(np32(q[0]).astype(np.float64), k, v, D ** -0.5)
        assert relative(got.ravel(), want.ravel()) <= limit(dtype) * (2 if dtype == BF else 1), at[i:i + Hq]
