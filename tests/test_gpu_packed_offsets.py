"""Offsets of packed sequences that fall or leave [0, N]: the status word says so,
rows that no valid pair holds are left, and rows that one valid pair alone holds,
with no later offset at or before them, come out as without the bad ones."""

import numpy as np
import pytest
import torch

import sparda
from helpers import np32
from packed_oracle import attend
from test_gpu_packed import BF, DEV, F32, inputs

pytestmark = pytest.mark.gpu


def owners(cu, N):
    """Per row: the valid pair that alone holds it with no later start at or before it, -1: no valid pair, -2: neither."""
    n = len(cu) - 1
    held = [[i for i in range(n) if 0 <= cu[i] <= t < cu[i + 1] <= N] for t in range(N)]
    return [-1 if not h else h[0] if len(h) == 1 and all(cu[j] > t for j in range(h[0] + 1, n)) else -2
            for t, h in enumerate(held)]


def test_owners():
    assert owners([0, 3, 9], 6) == [0, 0, 0, -1, -1, -1]
    assert owners([0, 4, 4, 2, 6], 6) == [0, 0, -2, -2, 3, 3]
    assert owners([4, 6, 1, 2], 6) == [-1, 2, -1, -1, -2, -2]


CU = [[0, 50, 30, 100], [0, 40, 200], [-5, 60, 100], [0, 120, 90, 100], [50, 100, 10, 20], [0, 30, 30, 101], [7, 60, -2, 80, 99]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,Hq,Hkv,D,times", [(BF, 2, 1, 64, 1), (BF, 4, 2, 16, 1), (F32, 6, 2, 64, 1), (BF, 12, 4, 64, 10),
                                                  (BF, 8, 2, 128, 10), (BF, 12, 4, 32, 10), (F32, 8, 2, 32, 10)], ids=str)
@pytest.mark.parametrize("cu", CU, ids=str)
def test_prefill_beside_offsets_out_of_range(cu, dtype, Hq, Hkv, D, times, causal):
    cu, N, R = [c * times for c in cu], 100 * times, Hq // Hkv
    print(f"[case] packed offsets {cu} {dtype} {Hq}/{Hkv}x{D} causal={causal}", flush=True)
    q, k, v = inputs(N, Hq, Hkv, D, dtype, seed=4)
    out = torch.full((N, Hq * D), 7.0, dtype=dtype, device=DEV)
    sparda.status()
    sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), causal=causal,
                          out=out)
    assert sparda.status() == sparda.STATUS_SEQUENCE_RANGE
    own, got = owners(cu, N), np32(out).astype(np.float64).reshape(N, Hq, D)
    assert np.isfinite(got).all()
    assert all((got[t] == 7).all() for t in range(N) if own[t] == -1)
    q, k, v = (np32(x).astype(np.float64) for x in (q, k, v))
    for t in range(0, N, 1 + times // 2):
        if own[t] >= 0:
            a, e = cu[own[t]], t + 1 if causal else cu[own[t] + 1]
            for g in range(Hkv):
                want, bf, f32 = attend(q[t, g * R:(g + 1) * R], k[a:e, g], v[a:e, g], D ** -0.5)
                assert (np.abs(got[t, g * R:(g + 1) * R] - want) <= (bf if dtype == BF else f32)).all(), (t, own[t])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cu", CU, ids=str)
def test_append_beside_offsets_out_of_range(cu, dtype):
    # a bad pair's rows are dropped, those of them that lie inside [0, N] too
    print(f"[case] append offsets {cu} {dtype}", flush=True)
    N, n, ps, width = 100, len(cu) - 1, 16, 20
    g = torch.Generator().manual_seed(3)
    kp, vp = (torch.randn(n * width, ps, 2, 64, generator=g).to(dtype) for _ in range(2))
    kn, vn = (torch.randn(N, 2, 64, generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(n * width, generator=g).view(n, width).to(torch.int32)
    pos = torch.arange(n, dtype=torch.int32) * 5
    kd, vd = kp.to(DEV), vp.to(DEV)
    sparda.status()
    sparda.append_paged(kd, vd, table.to(DEV), pos.to(DEV), kn.to(DEV), vn.to(DEV),
                        cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    assert sparda.status() == sparda.STATUS_SEQUENCE_RANGE
    may = torch.zeros(n * width, ps, dtype=torch.bool)           # rows that a row of two pairs may have changed
    for t, i in enumerate(owners(cu, N)):
        for j in range(n):
            p = int(pos[j]) + t - cu[j]
            if i == j:
                kp[table[j, p // ps], p % ps], vp[table[j, p // ps], p % ps] = kn[t], vn[t]
            elif i == -2 and 0 <= cu[j] <= t < cu[j + 1] <= N:
                may[table[j, p // ps], p % ps] = True
    assert torch.equal(kd.cpu()[~may], kp[~may]) and torch.equal(vd.cpu()[~may], vp[~may])
