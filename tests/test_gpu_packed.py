"""Attention over packed prompts (sparda.prefill_packed) against float64: both
types, head dims and head groups, lengths from nothing to several windows, rows
outside every sequence, strides and alignment, what a row may not attend, and
replay from a graph as the offsets change. Bounds: packed_oracle."""

import numpy as np
import pytest
import torch

import sparda
from helpers import np32
from packed_oracle import attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def offsets(lengths, start=0):
    return np.concatenate(([start], start + np.cumsum(lengths))).astype(np.int32)


def inputs(N, Hq, Hkv, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda h: torch.randn(N, h, D, generator=g)
    return (r(Hq) * std).to(dtype), r(Hkv).to(dtype), r(Hkv).to(dtype)


def check(got, q, k, v, cu, causal=True, scale=None, rows=None):
    """got [N, Hq*D] against float64 on the packed inputs (CPU tensors), row by row within the bounds."""
    N, Hq, D = q.shape
    R = Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    dtype = q.dtype
    q, k, v = (np32(x).astype(np.float64) for x in (q, k, v))
    got = np32(got).astype(np.float64).reshape(N, Hq, D)
    worst = 0.0
    for i in range(len(cu) - 1):
        a, b = int(cu[i]), int(cu[i + 1])
        ts = range(a, b) if rows is None else [t for t in rows if a <= t < b]
        for t in ts:
            e = t + 1 if causal else b
            for g in range(k.shape[1]):
                want, bf, f32 = attend(q[t, g * R:(g + 1) * R], k[a:e, g], v[a:e, g], scale)
                tol = bf if dtype == BF else f32
                err = np.abs(got[t, g * R:(g + 1) * R] - want)
                assert (err <= tol).all(), f"sequence {i} row {t - a} group {g}: {(err / tol).max():.2f} of the bound"
                worst = max(worst, float((err / tol).max()))
    return worst


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (4, 4, 64), (6, 3, 128), (8, 1, 128), (5, 1, 64), (34, 2, 64),
                                      (3, 1, 32), (4, 2, 16)])
@pytest.mark.parametrize("lengths", [[1], [37], [5, 0, 64, 1, 130], [0, 33, 65, 0]], ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_prompts_against_float64(dtype, Hq, Hkv, D, lengths, causal):
    print(f"[case] packed {dtype} {Hq}/{Hkv}x{D} {lengths} causal={causal}", flush=True)
    cu = offsets(lengths)
    q, k, v = inputs(int(cu[-1]), Hq, Hkv, D, dtype, seed=sum(lengths) + Hq + D)
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV), causal=causal)
    check(got, q, k, v, cu, causal)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("lengths", [[700, 3, 1025, 256], [2111], [300] * 9], ids=str)
def test_packed_prompts_of_several_windows(dtype, Hq, Hkv, D, lengths):
    print(f"[case] packed long {dtype} {Hq}/{Hkv}x{D} {lengths}", flush=True)
    cu = offsets(lengths)
    N = int(cu[-1])
    q, k, v = inputs(N, Hq, Hkv, D, dtype, seed=N, std=2.0)
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV))
    edges = {int(c) + d for c in cu for d in range(-3, 4)}
    rows = sorted(t for t in edges | set(range(0, N, 61)) if 0 <= t < N)
    check(got, q, k, v, cu, rows=rows)


@pytest.mark.parametrize("scale", [0.0, -0.25, 3.0])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_packed_prompts_other_scales(dtype, scale):
    print(f"[case] packed scale {scale} {dtype}", flush=True)
    cu = offsets([70, 129])
    q, k, v = inputs(199, 6, 2, 64, dtype, seed=3)
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV), scale=scale)
    check(got, q, k, v, cu, scale=scale)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_packed_prompts_scores_that_rise_and_fall(dtype, D):
    # a key far above and keys far below the first ones: the statistics have to follow
    print(f"[case] packed rising scores {dtype} D={D}", flush=True)
    cu = offsets([400, 150])
    q, k, v = inputs(550, 4, 2, D, dtype, seed=11)
    k[::7] *= 12
    k[200] *= 60
    k[:40] *= 0.01
    k[400:420] *= 40
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV))
    check(got, q, k, v, cu)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_rows_outside_every_sequence_are_left(dtype):
    print(f"[case] packed rows left {dtype}", flush=True)
    cu = offsets([40, 0, 90], start=7)
    N = 160
    q, k, v = inputs(N, 12, 4, 64, dtype, seed=5)
    for x in (q, k, v):
        x[:7] = float("nan")
        x[137:] = float("nan")
    out = torch.full((N, 768), 7.0, dtype=dtype, device=DEV)
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV), out=out)
    assert got is out
    assert (out[:7] == 7).all() and (out[137:] == 7).all()
    check(out, q, k, v, cu)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("D", [64, 128])
def test_what_a_row_may_not_attend_stays_out(dtype, bad, D):
    # a key and a value at one row of the middle sequence: the rows before it and the other sequences never see them
    print(f"[case] packed {bad} {dtype} D={D}", flush=True)
    cu = offsets([50, 120, 60])
    q, k, v = inputs(230, 6, 2, D, dtype, seed=8)
    cud = torch.from_numpy(cu).to(DEV)
    for at in (50, 95, 169):
        k2, v2 = k.clone(), v.clone()
        v2[at, :, 3] = bad
        got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v2.to(DEV), cud)
        clean = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), cud)
        g, c = got.view(230, 6, D).float(), clean.view(230, 6, D).float()
        keep = [i for i in range(D) if i != 3]
        torch.testing.assert_close(g[..., keep], c[..., keep], rtol=2 ** -6, atol=2 ** -6)
        seen = torch.zeros(230, dtype=torch.bool)
        seen[at:170] = True
        assert not torch.isfinite(g[seen][..., 3]).any()
        torch.testing.assert_close(g[~seen], c[~seen], rtol=2 ** -6, atol=2 ** -6)
        k2[at] = bad
        got = sparda.prefill_packed(q.to(DEV), k2.to(DEV), v.to(DEV), cud)
        torch.testing.assert_close(got.float()[~seen], clean.float()[~seen], rtol=2 ** -6, atol=2 ** -6)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_keys_of_minus_infinity_weigh_nothing(dtype, D):
    # scores of -inf at the first keys (a positive query against -inf), finite ones later
    print(f"[case] packed -inf scores {dtype} D={D}", flush=True)
    cu = offsets([200])
    q, k, v = inputs(200, 2, 1, D, dtype, seed=9)
    q[..., 0] = q[..., 0].abs() + 0.5
    k2 = k.clone()
    k2[:90, :, 0] = -float("inf")
    got = sparda.prefill_packed(q.to(DEV), k2.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV))
    assert torch.isnan(got[:90].float()).all()       # no key with a weight: 0 / 0
    qn, kn, vn = (np32(x).astype(np.float64) for x in (q, k, v))
    for t in range(90, 200, 9):
        want, bf, f32 = attend(qn[t], kn[90:t + 1, 0], vn[90:t + 1, 0], D ** -0.5)
        err = np.abs(np32(got[t]).reshape(2, D) - want)
        assert (err <= (bf if dtype == BF else f32)).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_packed_strides_and_alignment(dtype):
    print(f"[case] packed strides {dtype}", flush=True)
    cu = offsets([100, 31])
    N, Hq, Hkv, D = 131, 6, 2, 64
    q, k, v = inputs(N, Hq, Hkv, D, dtype, seed=6)
    cud = torch.from_numpy(cu).to(DEV)
    # one buffer of q, k and v rows, as a fused projection writes them
    buf = torch.zeros(N, (Hq + 2 * Hkv) * D, dtype=dtype, device=DEV)
    qd, kd, vd = (x.view(N, -1, D) for x in buf.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    qd.copy_(q), kd.copy_(k), vd.copy_(v)
    check(sparda.prefill_packed(qd, kd, vd, cud), q, k, v, cu)
    # heads before rows, k and v of different strides, rows off 16 bytes
    qh = q.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    kh = k.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    check(sparda.prefill_packed(qh, kh, v.to(DEV), cud), q, k, v, cu)
    off = torch.zeros(N * Hkv * D + 1, dtype=dtype, device=DEV)[1:].view(N, Hkv, D)
    off.copy_(k)
    check(sparda.prefill_packed(q.to(DEV), off, v.to(DEV), cud), q, k, v, cu)
    wide = torch.zeros(N, Hq * D + 3, dtype=dtype, device=DEV)
    check(sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), cud, out=wide[:, :Hq * D]), q, k, v, cu)
    assert (wide[:, Hq * D:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_packed_rows_far_apart_and_an_output_off_16_bytes(dtype):
    print(f"[case] packed far rows {dtype}", flush=True)
    cu = offsets([3, 0, 4], start=1)
    N, D = 9, 64
    q, k, v = inputs(N, 6, 2, D, dtype, seed=21)
    far = torch.zeros(N, 1 << 24, dtype=dtype, device=DEV)     # rows 2^24 elements apart
    kd, vd = (far[:, i * 128:(i + 1) * 128].view(N, 2, D) for i in range(2))
    kd.copy_(k), vd.copy_(v)
    out = torch.full((N, 6 * D + 3), 7.0, dtype=dtype, device=DEV)[:, 1:6 * D + 1]
    got = sparda.prefill_packed(q.to(DEV), kd, vd, torch.from_numpy(cu).to(DEV), out=out)
    assert got is out and (out[:1] == 7).all() and (out[8:] == 7).all()
    check(out, q, k, v, cu)
    one = sparda.prefill_packed(q[:1].to(DEV), kd[1:2], vd[1:2], torch.tensor([0, 1], dtype=torch.int32, device=DEV))
    check(one, q[:1], k[1:2], v[1:2], [0, 1])                  # one row: its stride has no meaning


def test_many_sequences():
    print("[case] packed 300 sequences", flush=True)
    r = np.random.default_rng(2)
    lengths = r.integers(0, 12, 300)
    cu = offsets(lengths)
    N = int(cu[-1])
    for dtype in (BF, F32):
        q, k, v = inputs(N, 6, 2, 64, dtype, seed=1)
        check(sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV)), q, k, v, cu)


@pytest.mark.parametrize("cu", [[0, 50, 30, 100], [0, 40, 200], [-5, 60, 100], [0, 120, 90, 100]], ids=str)
@pytest.mark.parametrize("D", [64, 32])
def test_offsets_out_of_range_raise_the_status_and_stay_inside(cu, D):
    # the bad sequences' rows are left; nothing outside the buffers is touched
    print(f"[case] packed offsets {cu} D={D}", flush=True)
    sparda.status()
    q, k, v = inputs(100, 2, 1, D, BF, seed=4)
    out = torch.full((100, 2 * D), 7.0, dtype=BF, device=DEV)
    sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), out=out)
    assert sparda.status() == sparda.STATUS_SEQUENCE_RANGE
    bad = np.zeros(100, bool)
    good = []
    for a, b in zip(cu, cu[1:]):
        if 0 <= a <= b <= 100:
            good.append((a, b))
    o = np32(out)
    covered = np.zeros(100, bool)
    for a, b in good:
        covered[a:b] = True
    assert (o[~covered] == 7).all()
    assert np.isfinite(o).all()
    assert not bad.any()


def test_packed_no_rows_and_no_sequences():
    q, k, v = (x.to(DEV) for x in inputs(8, 2, 1, 64, BF, seed=1))
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full((8, 128), 7.0, dtype=BF, device=DEV)
    assert (sparda.prefill_packed(q, k, v, zero, out=out) == 7).all()
    assert sparda.prefill_packed(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device=DEV)).shape == (0, 128)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_packed_captured_and_replayed_with_other_offsets(dtype):
    print(f"[case] packed graph {dtype}", flush=True)
    N = 300
    q, k, v = inputs(N, 6, 2, 64, dtype, seed=12)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)
    cud = torch.tensor([0, 100, 300], dtype=torch.int32, device=DEV)
    out = torch.zeros(N, 384, dtype=dtype, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        sparda.prefill_packed(qd, kd, vd, cud, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sparda.prefill_packed(qd, kd, vd, cud, out=out)
    for cu in ([0, 100, 300], [0, 299, 300], [0, 0, 300], [0, 1, 300]):
        cud.copy_(torch.tensor(cu, dtype=torch.int32))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = sparda.prefill_packed(qd, kd, vd, cud)
        assert torch.equal(out, eager)
        check(out, q, k, v, np.array(cu), rows=range(0, N, 23))


# sizes on either side of the limits at which the work is cut differently
CUTS = [(BF, 12, 4, 64, [500]), (BF, 12, 4, 64, [2000]), (BF, 12, 4, 64, [1600]), (BF, 12, 4, 64, [2800, 2850]), (BF, 32, 8, 128, [1200]), (BF, 12, 4, 64, [4200]), (BF, 12, 4, 64, [700] * 8),
        (BF, 12, 4, 64, [9000, 13001]), (BF, 16, 16, 64, [1500, 600]), (BF, 32, 8, 128, [400]), (BF, 12, 4, 32, [900, 77]), (BF, 6, 2, 16, [300, 40]), (F32, 6, 2, 32, [300, 40]), (BF, 8, 2, 128, [4300]),
        (BF, 32, 8, 128, [150] * 10), (BF, 32, 8, 128, [3000, 2000]), (F32, 12, 4, 64, [3000]), (F32, 8, 1, 128, [1000, 700]),
        (BF, 12, 4, 64, [300, 41]), (BF, 8, 2, 128, [260, 33]), (BF, 8, 4, 32, [380, 100]), (F32, 6, 2, 32, [2000]),
        (F32, 6, 2, 32, [3000, 200]), (BF, 8, 2, 16, [2500, 33]), (F32, 8, 2, 16, [2500, 33]), (F32, 8, 2, 128, [3500])]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,Hq,Hkv,D,lengths", CUTS, ids=str)
def test_packed_prompts_at_every_cut_of_the_work(dtype, Hq, Hkv, D, lengths, causal):
    """Ordinary values; keys that rise far above the first ones; one value that is
    not finite: sampled rows against float64, and every row for where it shows."""
    print(f"[case] packed cut {dtype} {Hq}/{Hkv}x{D} {lengths} causal={causal}", flush=True)
    cu = offsets(lengths)
    N = int(cu[-1])
    cud = torch.from_numpy(cu).to(DEV)
    q, k, v = inputs(N, Hq, Hkv, D, dtype, seed=N, std=2.0)
    rows = sorted({int(c) + d for c in cu for d in (-2, -1, 0, 1, 31, 32, 63, 64) if 0 <= c + d < N}
                  | {int(x) for x in np.random.default_rng(N).integers(0, N, 12)})
    qd, vd = q.to(DEV), v.to(DEV)
    clean = sparda.prefill_packed(qd, k.to(DEV), vd, cud, causal=causal)
    check(clean, q, k, v, cu, causal, rows=rows)
    high = k.clone()
    high[N // 3::5] *= 15
    check(sparda.prefill_packed(qd, high.to(DEV), vd, cud, causal=causal), q, high, v, cu, causal, rows=rows)
    last = len(lengths) - 1
    a, b = int(cu[last]), int(cu[last + 1])
    for at in (a, a + (b - a) // 2 + 1, b - 1):
        v2 = v.clone()
        v2[at, Hkv - 1, 5] = float("inf")
        got = sparda.prefill_packed(qd, k.to(DEV), v2.to(DEV), cud, causal=causal).view(N, Hq, D)
        hit = torch.zeros(N, Hq, D, dtype=torch.bool)
        hit[(at if causal else a):b, Hq - Hq // Hkv:, 5] = True
        assert torch.equal(~torch.isfinite(got).cpu(), hit)
        torch.testing.assert_close(got.cpu()[~hit].float(), clean.cpu().view(N, Hq, D)[~hit].float(), rtol=0, atol=0)


def test_packed_more_sequences_than_lanes_and_long_ones():
    print("[case] packed 130 sequences of up to 700", flush=True)
    r = np.random.default_rng(7)
    lengths = np.where(r.random(130) < 0.1, r.integers(300, 700, 130), r.integers(0, 40, 130))
    cu = offsets(lengths)
    N = int(cu[-1])
    q, k, v = inputs(N, 12, 4, 64, BF, seed=3)
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV))
    check(got, q, k, v, cu, rows=range(0, N, 17))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (8, 1, 128), (6, 2, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_short_sequences_in_a_large_batch(dtype, Hq, Hkv, D, causal):
    """Many short sequences of odd lengths between rows of no sequence that hold
    NaN, and, in one of them, a value that is not finite and keys whose scores are -inf."""
    print(f"[case] packed large batch {dtype} {Hq}/{Hkv}x{D} causal={causal}", flush=True)
    cu = offsets([5, 0, 64, 1, 130, 33, 120, 31] * 6, start=3)
    N = int(cu[-1]) + 9
    q, k, v = inputs(N, Hq, Hkv, D, dtype, seed=D)
    q[..., 0] = q[..., 0].abs() + 0.5
    for x in (q, k, v):
        x[:3] = float("nan")
        x[N - 9:] = float("nan")
    cud = torch.from_numpy(cu).to(DEV)
    out = torch.full((N, Hq * D), 7.0, dtype=dtype, device=DEV)
    sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), cud, causal=causal, out=out)
    assert (out[:3] == 7).all() and (out[N - 9:] == 7).all()
    rows = sorted({int(c) + d for c in cu for d in (-2, -1, 0, 1, 15, 16, 31, 32) if 3 <= c + d < N - 9})
    check(out, q, k, v, cu, causal, rows=rows)
    a, b = int(cu[20]), int(cu[21])                  # a sequence of 130
    k2, v2 = k.clone(), v.clone()
    k2[a:a + 40, 0, 0] = -float("inf")               # of the first KV head
    v2[a + 77, Hkv - 1, 5] = float("nan")
    R, got = Hq // Hkv, sparda.prefill_packed(q.to(DEV), k2.to(DEV), v2.to(DEV), cud, causal=causal).view(N, Hq, D).cpu().float()
    nan = torch.zeros(N, Hq, D, dtype=torch.bool)
    nan[(a + 77 if causal else a):b, Hq - R:, 5] = True
    if causal:
        nan[a:a + 40, :R] = True                     # every key weighs nothing: 0 / 0
    inside = slice(3, N - 9)
    assert torch.equal(torch.isnan(got)[inside], nan[inside])
    same = torch.ones(N, Hq, D, dtype=torch.bool)
    same[a:b] = False
    torch.testing.assert_close(got[inside][same[inside]], out.view(N, Hq, D).cpu().float()[inside][same[inside]], rtol=0, atol=0)
    qn, kn, vn = (np32(x).astype(np.float64) for x in (q, k, v))
    for t in range(a + 41, b, 7):
        e = t + 1 if causal else b
        want, bf, f32 = attend(qn[t, :R], kn[a + 40:e, 0], vn[a + 40:e, 0], D ** -0.5)
        ok = ~nan[t, :R].numpy()
        assert (np.abs(got[t, :R].numpy() - want)[ok] <= (bf if dtype == BF else f32)[ok]).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n", [63, 64, 65, 128, 1000, 4097])
def test_packed_search_over_many_offsets(dtype, n):
    print(f"[case] packed {n} sequences {dtype}", flush=True)
    r = np.random.default_rng(n)
    lengths = np.where(r.random(n) < 0.3, 0, r.integers(1, 5, n))
    lengths[-1] = 3
    cu = offsets(lengths, start=2)
    N = int(cu[-1]) + 1
    q, k, v = inputs(N, 3, 1, 64, dtype, seed=n)
    out = torch.full((N, 192), 7.0, dtype=dtype, device=DEV)
    sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV), out=out)
    assert (out[:2] == 7).all() and (out[N - 1] == 7).all()
    check(out, q, k, v, cu, rows=range(0, N, 1 + N // 500))


@pytest.mark.parametrize("dtype,N,Hq,Hkv,D", [(BF, 600_000, 32, 8, 128), (F32, 300_000, 32, 8, 64)], ids=str)
def test_packed_rows_past_32_bit_offsets(dtype, N, Hq, Hkv, D):
    # q and out beyond 2^31 bytes (bf16: 2^31 elements), sequences of 100 rows
    print(f"[case] packed 64-bit offsets {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(17)
    q, k, v = (torch.randn(N, h, D, generator=g, device=DEV, dtype=dtype) for h in (Hq, Hkv, Hkv))
    cu = torch.arange(0, N + 1, 100, dtype=torch.int32, device=DEV)
    out = sparda.prefill_packed(q, k, v, cu)
    for a in (0, N // 2, N - 100):
        part = [x[a:a + 100].cpu() for x in (q, k, v)]
        check(out[a:a + 100], *part, [0, 100], rows=(0, 1, 50, 99))
