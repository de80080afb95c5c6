"""The rotated write into 16-bit and 32-bit pages (sparda.rotate_append_paged): bit for bit the formula
in fp32, rounded once, and an indexed copy; every other row of the pages and of `out` stays."""

import numpy as np
import pytest
import torch

import sparda
from model.rope import rope_tables
from q4_oracle import turn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def dev(x):
    return x.to(DEV) if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=torch.int32, device=DEV)


def randn(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def server(news, olds, ps, seed, spare=2):
    """A page table in random order for sequences of olds + news rows."""
    need = [max(0, (n + max(o, 0) + ps - 1) // ps) for n, o in zip(news, olds)]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(need), max(1, max(need))), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    return table, sum(need) + spare


def expect(kp, vp, table, olds, cu, q, kn, vn, cos, sin, out):
    """The plain loop over rows, on the CPU."""
    ps, (kp, vp, out) = kp.shape[1], (x.clone() for x in (kp, vp, out))
    for b, old in enumerate(olds):
        if old < 0:
            continue
        for j, t in enumerate(range(cu[b], cu[b + 1])):
            p = old + j
            out[t] = turn(q[t:t + 1], cos, sin, [p])[0].to(q.dtype)
            page = int(table[b, p // ps])
            kp[page, p % ps] = turn(kn[t:t + 1], cos, sin, [p])[0].to(q.dtype)
            vp[page, p % ps] = vn[t]
    return kp, vp, out


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (32, 8, 128), (3, 1, 32), (5, 5, 16), (40, 8, 128), (1, 1, 64), (70, 7, 16)])
@pytest.mark.parametrize("news,olds,ps", [([1], [0], 16), ([1, 1, 1, 1], [5, 0, -1, 47], 16),
                                          ([0, 19, 1, 64, 3], [7, 15, 63, 0, -1], 64), ([300, 2], [1, 200], 48)], ids=str)
def test_rotated_write_is_the_formula(dtype, Hq, Hkv, D, news, olds, ps):
    print(f"[case] rotate {dtype} {Hq}/{Hkv}x{D} {news} {olds} ps={ps}", flush=True)
    cu = np.concatenate(([0], np.cumsum(news))).tolist()
    N = cu[-1] + (3 if max(news) > 1 else 0)      # rows behind the last sequence
    table, P = server(news, olds, ps, seed=D + ps)
    kp, vp = (randn(P, ps, Hkv, D, dtype=dtype, seed=s) for s in (1, 2))
    q, kn, vn = randn(N, Hq, D, dtype=dtype, seed=3), randn(N, Hkv, D, dtype=dtype, seed=4), randn(N, Hkv, D, dtype=dtype, seed=5)
    cos, sin = rope_tables(D, 600)
    out = randn(N, Hq, D, dtype=dtype, seed=6)
    want = expect(kp, vp, table, olds, cu, q, kn, vn, cos, sin, out)
    kd, vd, od = dev(kp), dev(vp), dev(out)
    sparda.status()
    one = max(news) == min(news) == 1
    got = sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), dev(q), dev(kn), dev(vn), dev(cos), dev(sin),
                                     cu_seqlens=None if one else dev(cu), out=od)
    assert got is od and sparda.status() == 0
    for a, b in zip((kd, vd, od), want):
        assert torch.equal(a.cpu(), b)
    # without out (the native path), in place, and without queries
    kd, vd, qd = dev(kp), dev(vp), dev(q)
    got = sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), qd, dev(kn), dev(vn), dev(cos), dev(sin),
                                     None if one else dev(cu))
    rows = [t for b, o in enumerate(olds) if o >= 0 for t in range(cu[b], cu[b + 1])]
    assert torch.equal(got.cpu()[rows], want[2][rows]) and torch.equal(kd.cpu(), want[0]) and torch.equal(qd.cpu(), q)
    sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), qd, dev(kn), dev(vn), dev(cos), dev(sin),
                               None if one else dev(cu), out=qd)
    rest = [t for t in range(N) if t not in set(rows)]
    assert torch.equal(qd.cpu()[rows], want[2][rows]) and torch.equal(qd.cpu()[rest], q[rest])
    kd, vd = dev(kp), dev(vp)
    assert sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), None, dev(kn), dev(vn), dev(cos), dev(sin),
                                      None if one else dev(cu)) is None
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_rotated_write_of_strided_rows_and_tables(dtype):
    print(f"[case] rotate strided {dtype}", flush=True)
    N, Hq, Hkv, D, ps = 21, 6, 2, 64, 32
    olds, cu = [3, 40], [0, 9, 21]
    table, P = server([9, 12], olds, ps, seed=9)
    wide = dev(randn(N, Hq + 2 * Hkv, D, dtype=dtype, seed=1))              # one projection's output
    q, kn, vn = wide[:, :Hq], wide[:, Hq:Hq + Hkv], wide[:, Hq + Hkv:]
    cos, sin = rope_tables(D, 100)
    kp, vp = (randn(P, ps, Hkv, D, dtype=dtype, seed=s) for s in (2, 3))
    both = dev(torch.stack((cos, sin), 1))                                  # [L,2,D/2]: rows of one table apart
    room = torch.zeros(Hq, N, D + 8, dtype=dtype, device=DEV)               # heads outside of tokens, rows apart
    out = room[..., :D].transpose(0, 1)
    want = expect(kp, vp, table, olds, cu, q.cpu(), kn.cpu(), vn.cpu(), cos, sin, torch.zeros(N, Hq, D, dtype=dtype))
    big = torch.zeros(P, ps, 2, Hkv, D, dtype=dtype, device=DEV)            # keys and values side by side
    kd, vd = big[:, :, 0], big[:, :, 1]
    kd.copy_(kp), vd.copy_(vp)
    sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), q, kn, vn, both[:, 0], both[:, 1], dev(cu), out=out)
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1]) and torch.equal(out.cpu(), want[2])
    assert (room[..., D:] == 0).all()
    # rows off 16 bytes go through copies
    flat = torch.zeros(N * Hq * D + 1, dtype=dtype, device=DEV)
    odd = flat[1:].view(N, Hq, D)
    odd.copy_(q)
    sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), odd, kn, vn, both[:, 0], both[:, 1], dev(cu), out=odd)
    assert torch.equal(odd.cpu(), want[2]) and flat[0] == 0


def test_positions_and_pages_out_of_range():
    print("[case] rotate out of range", flush=True)
    Hq, Hkv, D, ps = 2, 1, 64, 16
    cos, sin = rope_tables(D, 40)
    q, kn, vn = (randn(4, h, D, dtype=BF, seed=h) for h in (Hq, Hkv, Hkv))
    kp = randn(5, ps, Hkv, D, dtype=BF, seed=7)
    table = torch.tensor([[0, 1, 2], [3, -1, 4], [1 << 30, 0, 0], [4, 4, 4]], dtype=torch.int32)
    olds = [39, 20, 3, 47]                        # fine; no page; no such page; behind the angles
    sparda.status()
    for bad in (dict(olds=[40, 0, 0, 0], bit=sparda.STATUS_POSITION_RANGE), dict(olds=[2 ** 31 - 1, 0, 0, 0], bit=12),
                dict(olds=[39, 20, 0, 0], bit=sparda.STATUS_PAGE_RANGE), dict(olds=[0, 0, 0, 300], bit=12)):
        kd, vd = dev(kp), dev(kp)
        sparda.rotate_append_paged(kd, vd, dev(torch.tensor([[0, 1, 2], [3, -1, 4], [4, 0, 0], [2, 4, 4]], dtype=torch.int32)),
                                   dev(bad["olds"]), dev(q), dev(kn), dev(vn), dev(cos), dev(sin))
        assert sparda.status() == bad["bit"], bad
    kd, vd = dev(kp), dev(kp)
    got = sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), dev(q), dev(kn), dev(vn), dev(cos), dev(sin)).cpu()
    assert sparda.status() == sparda.STATUS_PAGE_RANGE | sparda.STATUS_POSITION_RANGE
    want = torch.cat([turn(q[t:t + 1], cos, sin, [olds[t]]).to(BF) for t in range(3)])
    assert torch.equal(got[:3], want) and got[3].isnan().all()
    kp[2, 39 % ps] = turn(kn[:1], cos, sin, [39])[0].to(BF)                 # the only row that has a place
    assert torch.equal(kd.cpu(), kp)


def test_first_halves_that_are_not_finite_stay_in_their_pairs():
    print("[case] rotate inf and NaN", flush=True)
    D = 32
    cos, sin = rope_tables(D, 8)
    q = randn(2, 1, D, dtype=BF, seed=1)
    q[0, 0, 3], q[1, 0, 20] = float("inf"), float("nan")
    kp = torch.zeros(2, 16, 1, D, dtype=BF)
    got = sparda.rotate_append_paged(dev(kp), dev(kp), dev(torch.tensor([[0], [1]], dtype=torch.int32)), dev([5, 2]), dev(q),
                                     dev(q), dev(q), dev(cos), dev(sin)).cpu()
    for t, p, d in ((0, 5, 3), (1, 2, 4)):
        want = turn(q[t:t + 1], cos, sin, [p])[0].to(BF)
        assert torch.equal(got[t].isnan(), want.isnan()) and torch.equal(got[t].nan_to_num(), want.nan_to_num())
        assert not got[t, 0, [i for i in range(D) if i % 16 != d]].isnan().any()


@pytest.mark.parametrize("n", [65, 4097])
def test_rotated_write_of_many_sequences(n):
    print(f"[case] rotate {n} sequences", flush=True)
    r = np.random.default_rng(n)
    news = np.where(r.random(n) < 0.3, 0, r.integers(1, 4, n))
    cu = np.concatenate(([0], np.cumsum(news))).astype(np.int32).tolist()
    olds = r.integers(-1, 28, n).tolist()
    table = torch.from_numpy(r.permutation(2 * n).reshape(n, 2).astype(np.int32))
    N, D = cu[-1], 16
    q, kn, vn = (randn(N, 2, D, dtype=BF, seed=s) for s in (1, 2, 3))
    kp, out = torch.full((2 * n, 16, 2, D), 7.0, dtype=BF), torch.full((N, 2, D), 3.0, dtype=BF)
    cos, sin = rope_tables(D, 32)
    want = expect(kp, kp, table, olds, cu, q, kn, vn, cos, sin, out)
    kd, vd, od = dev(kp), dev(kp), dev(out)
    sparda.rotate_append_paged(kd, vd, dev(table), dev(olds), dev(q), dev(kn), dev(vn), dev(cos), dev(sin), dev(cu), out=od)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((kd, vd, od), want)) and sparda.status() == 0


def test_offsets_out_of_range_raise_the_status():
    print("[case] rotate offsets", flush=True)
    cos, sin = rope_tables(16, 64)
    q = randn(6, 1, 16, dtype=F32, seed=1)
    kp, table = torch.zeros(4, 16, 1, 16), torch.tensor([[0], [1], [2]], dtype=torch.int32)
    for cu in ([0, 3, 2, 6], [-1, 2, 4, 6], [0, 2, 4, 7]):
        kd, vd = dev(kp), dev(kp)
        sparda.rotate_append_paged(kd, vd, dev(table), dev([0, 0, 0]), dev(q), dev(q), dev(q), dev(cos), dev(sin), dev(cu))
        assert sparda.status() == sparda.STATUS_SEQUENCE_RANGE
        assert (kd.cpu()[3] == 0).all()


def test_refusals_of_tensors_that_do_not_fit():
    print("[case] rotate refusals", flush=True)
    q, kn = randn(3, 4, 64, dtype=BF, seed=1).to(DEV), randn(3, 2, 64, dtype=BF, seed=2).to(DEV)
    kp, table, pos = torch.zeros(3, 16, 2, 64, dtype=BF, device=DEV), dev([[0], [1], [2]]), dev([0, 1, 2])
    cos, sin = (dev(x) for x in rope_tables(64, 32))
    good = dict(k_pages=kp, v_pages=kp.clone(), page_table=table, positions=pos, q=q, k_new=kn, v_new=kn.clone(), cos=cos, sin=sin)
    sparda.rotate_append_paged(**good)
    for bad, err in ((dict(cos=cos.double()), TypeError), (dict(cos=cos[:, :16]), ValueError), (dict(sin=sin[:5]), ValueError),
                     (dict(q=q.float()), TypeError), (dict(q=q[:2]), ValueError), (dict(k_new=kn.float(), v_new=kn.float()), TypeError),
                     (dict(v_new=kn[:2]), ValueError), (dict(positions=pos.long()), TypeError), (dict(positions=pos[:2]), ValueError),
                     (dict(cu_seqlens=dev([0, 3])), ValueError), (dict(out=torch.empty_like(q[:2])), ValueError),
                     (dict(q=None, out=torch.empty_like(q)), ValueError), (dict(cos=cos[:0], sin=sin[:0]), ValueError),
                     (dict(out=torch.zeros(1, 4, 64, dtype=BF, device=DEV).expand(3, 4, 64)), ValueError),
                     (dict(q=q.cpu()), RuntimeError), (dict(k_new=kn.clone().requires_grad_()), RuntimeError)):
        with pytest.raises(err):
            sparda.rotate_append_paged(**{**good, **bad})
