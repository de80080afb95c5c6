"""The cache in pages (sparda.append_paged, sparda.decode_paged): the write is
bit for bit an indexed copy, the attention is compared with float64 (bounds:
packed_oracle), and the three serving operators run together as a server would."""

import numpy as np
import pytest
import torch

import sparda
from helpers import np32
from packed_oracle import attend

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def cache(lengths, ps, Hkv, D, dtype, seed, spare=3, width=None, fill=float("nan")):
    """Pages in random order with NaN in every row that no sequence holds, the
    table (entries past a sequence: far out of range), and the sequences' keys and values."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + ps - 1) // ps for n in lengths]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g)
    kp, vp = (torch.full((P, ps, Hkv, D), fill, dtype=dtype) for _ in range(2))
    table = torch.full((len(lengths), width or max(1, max(need))), 1 << 30, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for b, n in enumerate(lengths):
        k, v = (torch.randn(n, Hkv, D, generator=g).to(dtype) for _ in range(2))
        ks.append(k), vs.append(v)
        for i in range(need[b]):
            page, rows = int(order[at]), min(ps, n - i * ps)
            table[b, i] = page
            kp[page, :rows], vp[page, :rows] = k[i * ps:i * ps + rows], v[i * ps:i * ps + rows]
            at += 1
    return kp, vp, table, ks, vs


def check(got, q, ks, vs, scale=None):
    B, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    got = np32(got).astype(np.float64).reshape(B, Hq, D)
    for b, (k, v) in enumerate(zip(ks, vs)):
        if k.shape[0] == 0:
            assert (got[b] == 0).all()
            continue
        R = Hq // k.shape[1]
        for g in range(k.shape[1]):
            want, bf, f32 = attend(np32(q[b, g * R:(g + 1) * R]).astype(np.float64), np32(k[:, g]).astype(np.float64),
                                   np32(v[:, g]).astype(np.float64), scale)
            tol = bf if q.dtype == BF else f32
            err = np.abs(got[b, g * R:(g + 1) * R] - want)
            assert (err <= tol).all(), f"sequence {b} group {g}: {(err / tol).max():.2f} of the bound"


def queries(B, Hq, D, dtype, seed):
    return torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (4, 4, 64), (8, 1, 128), (6, 3, 128), (5, 1, 64), (34, 2, 64),
                                      (3, 1, 32), (4, 2, 16)])
@pytest.mark.parametrize("lengths,ps", [([1], 16), ([1000], 16), ([0, 5, 16, 17, 33, 300], 16), ([64, 1, 0, 129], 64),
                                        ([47, 49, 48, 200], 48), ([700, 2], 128)], ids=str)
def test_paged_decode_against_float64(dtype, Hq, Hkv, D, lengths, ps):
    print(f"[case] paged {dtype} {Hq}/{Hkv}x{D} {lengths} ps={ps}", flush=True)
    kp, vp, table, ks, vs = cache(lengths, ps, Hkv, D, dtype, seed=sum(lengths) + D)
    q = queries(len(lengths), Hq, D, dtype, seed=7)
    sparda.status()
    got = sparda.decode_paged(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV),
                              torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check(got, q, ks, vs)
    assert sparda.status() == 0


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize("lengths", [[20011], [3, 9000, 0, 5000, 1]], ids=str)
def test_paged_decode_over_many_shares(dtype, Hq, Hkv, D, lengths):
    print(f"[case] paged long {dtype} {Hq}/{Hkv}x{D} {lengths}", flush=True)
    kp, vp, table, ks, vs = cache(lengths, 64, Hkv, D, dtype, seed=5, width=512)
    q = queries(len(lengths), Hq, D, dtype, seed=8) * 2
    got = sparda.decode_paged(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV),
                              torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check(got, q, ks, vs)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(6, 2, 16), (3, 3, 32), (34, 1, 128)])
def test_paged_decode_shares_of_other_heads(dtype, Hq, Hkv, D):
    print(f"[case] paged shares {dtype} {Hq}/{Hkv}x{D}", flush=True)
    lengths = [4100, 0, 1, 2999]
    kp, vp, table, ks, vs = cache(lengths, 32, Hkv, D, dtype, seed=D)
    q = queries(len(lengths), Hq, D, dtype, seed=10) * 2
    got = sparda.decode_paged(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV),
                              torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check(got, q, ks, vs)


@pytest.mark.parametrize("n", [64, 65, 1000, 4097])
def test_paged_append_of_many_sequences(n):
    print(f"[case] paged append {n} sequences", flush=True)
    r = np.random.default_rng(n)
    lengths = np.where(r.random(n) < 0.3, 0, r.integers(1, 5, n))
    cu = np.concatenate(([0], np.cumsum(lengths))).astype(np.int32)
    N, ps = int(cu[-1]), 16
    pos = r.integers(-1, 28, n).astype(np.int32)
    table = r.permutation(2 * n).reshape(n, 2).astype(np.int32)
    kn, vn = (torch.randn(N + 3, 2, 16, generator=torch.Generator().manual_seed(i)).to(BF) for i in (1, 2))
    kp, vp = (torch.full((2 * n, ps, 2, 16), 7.0, dtype=BF) for _ in range(2))
    kd, vd = kp.to(DEV), vp.to(DEV)
    dev = lambda x: torch.from_numpy(x).to(DEV)
    sparda.append_paged(kd, vd, dev(table), dev(pos), kn.to(DEV), vn.to(DEV), cu_seqlens=dev(cu))
    for b in range(n):
        for j in range(lengths[b]):
            p = int(pos[b]) + j
            if pos[b] >= 0:
                kp[table[b, p // ps], p % ps], vp[table[b, p // ps], p % ps] = kn[cu[b] + j], vn[cu[b] + j]
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp) and sparda.status() == 0


def test_paged_decode_of_many_sequences():
    print("[case] paged 200 sequences", flush=True)
    r = np.random.default_rng(3)
    lengths = [int(x) for x in r.integers(0, 400, 200)]
    kp, vp, table, ks, vs = cache(lengths, 32, 2, 64, BF, seed=6, width=40)
    q = queries(200, 6, 64, BF, seed=9)
    got = sparda.decode_paged(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV),
                              torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check(got, q, ks, vs)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.5, 4.0])
def test_paged_decode_other_scales(dtype, scale):
    print(f"[case] paged scale {scale} {dtype}", flush=True)
    lengths = [333, 40]
    kp, vp, table, ks, vs = cache(lengths, 16, 2, 64, dtype, seed=2)
    q = queries(2, 6, 64, dtype, seed=3)
    got = sparda.decode_paged(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV),
                              torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=scale)
    check(got, q, ks, vs, scale=scale)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_paged_decode_strides(dtype):
    # keys and values interleaved page by page, a table inside a wider one, a strided q and out
    print(f"[case] paged strides {dtype}", flush=True)
    lengths, ps, Hkv, D = [100, 37, 64], 32, 2, 64
    kp, vp, table, ks, vs = cache(lengths, ps, Hkv, D, dtype, seed=4)
    both = torch.stack((kp, vp), dim=1).to(DEV)
    heads = torch.stack((kp, vp), dim=1).transpose(2, 3).contiguous().to(DEV).transpose(2, 3)
    wide = torch.full((3, 9), -1, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = table
    wt = wide.to(DEV)[:, 2:2 + table.shape[1]]
    q = queries(3, 6, D, dtype, seed=5)
    qt = q.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    qo = torch.zeros(3 * 6 * D + 1, dtype=dtype, device=DEV)[1:].view(3, 6, D)
    qo.copy_(q)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out = torch.zeros(3, 6 * D + 5, dtype=dtype, device=DEV)
    for pages in (both, heads):
        for qd in (qt, qo):
            check(sparda.decode_paged(qd, pages[:, 0], pages[:, 1], wt, n), q, ks, vs)
    sparda.decode_paged(qt, both[:, 0], both[:, 1], wt, n, out=out[:, :6 * D])
    check(out[:, :6 * D], q, ks, vs)
    assert (out[:, 6 * D:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_bad_pages_and_lengths_stay_alone(dtype):
    print(f"[case] paged bad {dtype}", flush=True)
    lengths, ps = [100, 300, 40, 2000, 64], 32
    kp, vp, table, ks, vs = cache(lengths, ps, 2, 64, dtype, seed=4)
    q = queries(5, 6, 64, dtype, seed=6)
    kd, vd, qd = kp.to(DEV), vp.to(DEV), q.to(DEV)
    n = torch.tensor(lengths, dtype=torch.int32)
    cap = table.shape[1] * ps
    for what in ("page", "negative page", "length", "negative length", "late page"):
        t2, n2, hit = table.clone(), n.clone(), 1
        if what == "page":
            t2[1, 4] = kp.shape[0]
        elif what == "negative page":
            t2[1, 0] = -1
        elif what == "late page":
            t2[3, 50], hit = -7, 3
        elif what == "length":
            n2[1] = cap + 1
        else:
            n2[1] = -3
        if what == "length":
            t2[1, :] = 0                              # (every page it reaches is one of the cache's)
        sparda.status()
        got = sparda.decode_paged(qd, kd, vd, t2.to(DEV), n2.to(DEV))
        assert sparda.status() == sparda.STATUS_PAGE_RANGE, what
        assert torch.isnan(got[hit].float()).all(), what
        rest = [b for b in range(5) if b != hit]
        check(got[rest], q[rest], [ks[b] for b in rest], [vs[b] for b in rest])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hkv,D,ps", [(4, 64, 64), (1, 128, 16), (3, 32, 48), (2, 16, 32)])
def test_append_is_an_indexed_copy(dtype, Hkv, D, ps):
    print(f"[case] append {dtype} {Hkv}x{D} ps={ps}", flush=True)
    g = torch.Generator().manual_seed(1)
    B, P, width = 70, 400, 5
    table = torch.randperm(P, generator=g)[:B * width].view(B, width).to(torch.int32)
    kp, vp = (torch.randn(P, ps, Hkv, D, generator=g).to(dtype) for _ in range(2))
    pos = torch.randint(0, 2 * ps, (B,), generator=g).to(torch.int32)
    pos[3] = pos[69] = -1
    for packed in (False, True):
        counts = torch.randint(0, 2 * ps, (B,), generator=g) if packed else torch.ones(B, dtype=torch.int64)
        counts[5:9] = 0 if packed else 1
        lead = 2 if packed else 0                      # rows before the first sequence, and three behind the last
        N = int(counts.sum()) + (lead + 3 if packed else 0)
        kn, vn = (torch.randn(N, Hkv, D, generator=g).to(dtype) for _ in range(2))
        cu = torch.cat((torch.tensor([lead]), lead + counts.cumsum(0))).to(torch.int32)
        wk, wv = kp.clone(), vp.clone()
        for b in range(B):
            for j in range(int(counts[b])):
                p = int(pos[b]) + j
                if pos[b] >= 0:
                    page, t = int(table[b, p // ps]), int(cu[b]) + j
                    wk[page, p % ps], wv[page, p % ps] = kn[t], vn[t]
        kd, vd = kp.to(DEV), vp.to(DEV)
        sparda.status()
        assert sparda.append_paged(kd, vd, table.to(DEV), pos.to(DEV), kn.to(DEV), vn.to(DEV),
                                   cu_seqlens=cu.to(DEV) if packed else None) is None
        assert torch.equal(kd.cpu(), wk) and torch.equal(vd.cpu(), wv)
        assert sparda.status() == 0


def test_append_strided_rows_and_pages():
    print("[case] append strides", flush=True)
    P, ps, Hkv, D, B = 6, 32, 2, 64, 3
    both = torch.zeros(P, 2, ps, Hkv, D, dtype=BF, device=DEV)
    rows = torch.randn(B, (6 + 2 * Hkv) * D, device=DEV).to(BF)       # q, k, v rows of a fused projection
    k, v = rows[:, 6 * D:8 * D].view(B, Hkv, D), rows[:, 8 * D:].view(B, Hkv, D)
    table = torch.tensor([[5, 0], [1, 3], [2, 4]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([31, 32, 0], dtype=torch.int32, device=DEV)
    sparda.append_paged(both[:, 0], both[:, 1], table, pos, k, v)
    want = torch.zeros_like(both)
    for b, (page, row) in enumerate([(5, 31), (3, 0), (2, 0)]):
        want[page, 0, row], want[page, 1, row] = k[b], v[b]
    assert torch.equal(both, want)
    # rows off 16 bytes, and k and v of different strides
    off = torch.zeros(B * Hkv * D + 1, dtype=BF, device=DEV)[1:].view(B, Hkv, D)
    off.copy_(k)
    both.zero_()
    sparda.append_paged(both[:, 0], both[:, 1], table, pos, off, v)
    assert torch.equal(both, want)


def test_append_rows_without_a_page_are_dropped():
    print("[case] append bad", flush=True)
    P, ps = 4, 16
    kp, vp = torch.zeros(P, ps, 1, 64, dtype=BF, device=DEV), torch.zeros(P, ps, 1, 64, dtype=BF, device=DEV)
    table = torch.tensor([[0, -1], [4, 1], [2, 3]], dtype=torch.int32, device=DEV)
    kn = torch.ones(3, 1, 64, dtype=BF, device=DEV)
    for pos, ok in (([16, 16, 0], [(1, 0), (2, 0)]), ([0, 0, 0], [(0, 0), (2, 0)]), ([1, 17, 32], [(0, 1), (1, 1)]),
                    ([1, 17, 2 ** 31 - 1], [(0, 1), (1, 1)])):
        kp.zero_(), vp.zero_()
        sparda.status()
        sparda.append_paged(kp, vp, table, torch.tensor(pos, dtype=torch.int32, device=DEV), kn, kn)
        assert sparda.status() == sparda.STATUS_PAGE_RANGE
        want = torch.zeros(P, ps)
        for page, row in ok:
            want[page, row] = 1
        assert torch.equal(kp[:, :, 0, 0].float().cpu(), want) and torch.equal(vp[:, :, 0, 0].float().cpu(), want)


@pytest.mark.parametrize("cu", [[0, 3, 9], [0, 5, 2], [-1, 2, 4]], ids=str)
def test_append_offsets_out_of_range_raise_the_status(cu):
    print(f"[case] append offsets {cu}", flush=True)
    kp, vp = torch.zeros(4, 16, 1, 64, dtype=BF, device=DEV), torch.zeros(4, 16, 1, 64, dtype=BF, device=DEV)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    kn = torch.ones(6, 1, 64, dtype=BF, device=DEV)
    sparda.status()
    sparda.append_paged(kp, vp, table, torch.zeros(2, dtype=torch.int32, device=DEV), kn, kn,
                        cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    assert sparda.status() & sparda.STATUS_SEQUENCE_RANGE


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_paged_decode_captured_and_replayed(dtype):
    # two graphs, each with its own workspace, replayed in turn as lengths and tables change
    print(f"[case] paged graph {dtype}", flush=True)
    Hq, Hkv, D, ps = 6, 2, 64, 32
    kp, vp, table, ks, vs = cache([1500, 900, 64], ps, Hkv, D, dtype, seed=4)
    q = queries(3, Hq, D, dtype, seed=6)
    qd, kd, vd, td = q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV)
    n = torch.tensor([1500, 900, 64], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sparda.decode_paged(qd, kd, vd, td, n)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(sparda.decode_paged(qd, kd, vd, td, n))
    for step, lens in enumerate(([1500, 900, 64], [10, 0, 64], [1400, 1, 33], [1500, 900, 64])):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        graphs[step % 2].replay()
        eager = sparda.decode_paged(qd, kd, vd, td, n)
        torch.cuda.synchronize()
        assert torch.equal(outs[step % 2], eager)
        check(eager, q, [k[:m] for k, m in zip(ks, lens)], [v[:m] for v, m in zip(vs, lens)])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (8, 2, 128)])
def test_a_server_prefills_and_decodes(dtype, Hq, Hkv, D):
    """Packed prompts through prefill_packed and into the pages, then decode
    steps that append a token of every running sequence and attend; sequences
    end, and one joins the batch. Every output against float64 over the
    sequence's own rows."""
    print(f"[case] server {dtype} {Hq}/{Hkv}x{D}", flush=True)
    g = torch.Generator().manual_seed(20)
    ps, P, width, B = 16, 64, 12, 4
    kp, vp = (torch.full((P, ps, Hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    free = [int(i) for i in torch.randperm(P, generator=g)]
    table = torch.full((B, width), -1, dtype=torch.int32)
    lens = [0] * B
    hist = [(torch.zeros(0, Hkv, D, dtype=dtype), torch.zeros(0, Hkv, D, dtype=dtype)) for _ in range(B)]

    def grow(b, n):
        while sum(int(x) >= 0 for x in table[b]) * ps < lens[b] + n:
            table[b, sum(int(x) >= 0 for x in table[b])] = free.pop()

    def rows(n, h):
        return torch.randn(n, h, D, generator=g).to(dtype)

    def prompts(counts):
        for b, n in enumerate(counts):
            grow(b, n)
        N = sum(counts)
        q, k, v = rows(N, Hq), rows(N, Hkv), rows(N, Hkv)
        cu = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        cud, pos = torch.from_numpy(cu).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
        out = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), cud)
        sparda.append_paged(kp, vp, table.to(DEV), pos, k.to(DEV), v.to(DEV), cu_seqlens=cud)
        for b, n in enumerate(counts):
            a = int(cu[b])
            if n:
                hist[b] = (k[a:a + n], v[a:a + n])
                lens[b] = n
                last = q[a + n - 1:a + n]
                check(out[a + n - 1:a + n], last, [k[a:a + n]], [v[a:a + n]])

    def step(running):
        for b in running:
            grow(b, 1)
        q, k, v = rows(B, Hq), rows(B, Hkv), rows(B, Hkv)
        pos = torch.tensor([lens[b] if b in running else -1 for b in range(B)], dtype=torch.int32, device=DEV)
        td = table.to(DEV)
        sparda.append_paged(kp, vp, td, pos, k.to(DEV), v.to(DEV))
        out = sparda.decode_paged(q.to(DEV), kp, vp, td, pos + 1)      # 0 for a slot that is idle
        for b in range(B):
            if b in running:
                hist[b] = tuple(torch.cat((h, x[b:b + 1])) for h, x in zip(hist[b], (k, v)))
                lens[b] += 1
                check(out[b:b + 1], q[b:b + 1], [hist[b][0]], [hist[b][1]])
            else:
                assert (out[b] == 0).all()

    sparda.status()
    prompts([15, 70, 1, 0])
    for _ in range(4):
        step([0, 1, 2])
    for i in range(width):                             # sequence 1 ends; its pages go back
        if table[1, i] >= 0:
            free.insert(0, int(table[1, i]))
            table[1, i] = -1
    lens[1] = 0
    step([0, 2])
    prompts_kept = lens[0], lens[2]
    lens_before = list(lens)
    lens[0], lens[2] = lens_before[0], lens_before[2]
    counts = [0, 0, 0, 40]
    prompts(counts)
    assert (lens[0], lens[2]) == prompts_kept
    for _ in range(3):
        step([0, 2, 3])
    assert sparda.status() == 0


_FIRST_CALLS_CAPTURED = r"""
import sys
sys.path[:0] = sys.argv[1:3]
import torch
import sparda
t = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
q, k, v, cu = t(40, 6, 64), t(40, 2, 64), t(40, 2, 64), i(0, 25, 40)
kp, vp, table, zero, n = t(8, 16, 2, 64), t(8, 16, 2, 64), i(3, 1, 5, 2).view(2, 2), i(0, 0), i(25, 15)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = sparda.prefill_packed(q, k, v, cu)
    sparda.append_paged(kp, vp, table, zero, k, v, cu_seqlens=cu)
    b = sparda.decode_paged(q[:2], kp, vp, table, n)
for _ in range(3):
    a.zero_(), b.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, sparda.prefill_packed(q, k, v, cu))
    assert torch.equal(b, sparda.decode_paged(q[:2], kp, vp, table, n))
assert sparda.status() == 0
print("CAPTURED", flush=True)
"""


def test_first_calls_of_a_process_can_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "local-research-small-language-model_amd")
    print("[case] first calls in a capture, fresh process", flush=True)
    r = subprocess.run([sys.executable, "-c", _FIRST_CALLS_CAPTURED, root, pkg], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "CAPTURED" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_operators_on_a_side_stream_and_without_the_native_host_path():
    print("[case] paged and packed on a side stream, through Python", flush=True)
    from sparda import ops
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(90, h, 64, generator=g).to(BF).to(DEV) for h in (6, 2, 2))
    cu = torch.tensor([0, 33, 90], dtype=torch.int32, device=DEV)
    table = torch.tensor([[1, 7, 3, -1], [0, 2, 4, 6]], dtype=torch.int32, device=DEV)
    zero, n = torch.zeros(2, dtype=torch.int32, device=DEV), torch.tensor([33, 57], dtype=torch.int32, device=DEV)

    def all_three():
        kp, vp = torch.zeros(8, 16, 2, 64, dtype=BF, device=DEV), torch.zeros(8, 16, 2, 64, dtype=BF, device=DEV)
        a = sparda.prefill_packed(q, k, v, cu)
        sparda.append_paged(kp, vp, table, zero, k, v, cu_seqlens=cu)
        return a, kp, vp, sparda.decode_paged(q[:2], kp, vp, table, n)

    want = all_three()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_three()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))

    class Off:
        def __getattr__(self, name):
            return lambda *args: None

    host, ops._host = ops._host, Off()
    try:
        got = all_three()
    finally:
        ops._host = host
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_refusals_of_tensors_that_do_not_fit():
    q, kv = torch.zeros(4, 2, 64, dtype=BF, device=DEV), torch.zeros(4, 1, 64, dtype=BF, device=DEV)
    pages, table = torch.zeros(3, 16, 1, 64, dtype=BF, device=DEV), torch.zeros(4, 1, dtype=torch.int32, device=DEV)
    n = torch.zeros(4, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    for exc, call in [
            (TypeError, lambda: sparda.prefill_packed(q, kv.float(), kv, cu)),
            (TypeError, lambda: sparda.prefill_packed(q, kv, kv, cu.long())),
            (TypeError, lambda: sparda.prefill_packed(q.half(), kv.half(), kv.half(), cu)),
            (ValueError, lambda: sparda.prefill_packed(q, kv[:3], kv[:3], cu)),
            (ValueError, lambda: sparda.prefill_packed(q, kv, kv, cu.view(1, 2))),
            (ValueError, lambda: sparda.prefill_packed(q, kv, kv, cu, out=torch.zeros(4, 64, dtype=BF, device=DEV))),
            (ValueError, lambda: sparda.prefill_packed(torch.zeros(4, 3, 64, dtype=BF, device=DEV),
                                                       torch.zeros(4, 2, 64, dtype=BF, device=DEV),
                                                       torch.zeros(4, 2, 64, dtype=BF, device=DEV), cu)),
            (TypeError, lambda: sparda.append_paged(pages, pages, table, n, kv.float(), kv.float())),
            (TypeError, lambda: sparda.append_paged(pages, pages, table.long(), n, kv, kv)),
            (ValueError, lambda: sparda.append_paged(pages, pages, table, n[:3], kv, kv)),
            (ValueError, lambda: sparda.append_paged(pages, pages, table, n, kv[:3], kv[:3])),
            (ValueError, lambda: sparda.append_paged(pages, pages, table, n, kv, kv, cu_seqlens=cu)),
            (ValueError, lambda: sparda.append_paged(pages, pages.transpose(1, 2), table, n, kv, kv)),
            (ValueError, lambda: sparda.append_paged(pages[:, :8], pages[:, :8], table, n, kv, kv)),
            (TypeError, lambda: sparda.decode_paged(q.float(), pages, pages, table, n)),
            (TypeError, lambda: sparda.decode_paged(q, pages, pages, table, n.long())),
            (ValueError, lambda: sparda.decode_paged(q[:3], pages, pages, table, n)),
            (ValueError, lambda: sparda.decode_paged(q, pages, pages, table[:, :0], n)),
            (ValueError, lambda: sparda.decode_paged(q, pages, pages, table, n[:2]))]:
        with pytest.raises(exc):
            call()
    grad = q.clone().requires_grad_(True)
    for call in (lambda: sparda.prefill_packed(grad, kv, kv, cu), lambda: sparda.decode_paged(grad, pages, pages, table, n)):
        with pytest.raises(RuntimeError, match="inference-only"):
            call()
    with torch.no_grad():
        assert sparda.decode_paged(grad, pages, pages, table, n).shape == (4, 128)


def test_pages_past_32_bit_offsets():
    # 70,000 pages of 64 rows of 8 heads of 128: 4.6e9 elements, the sequences in the last pages
    print("[case] paged 64-bit offsets", flush=True)
    P, ps, Hkv, D = 70000, 64, 8, 128
    kp, vp = (torch.empty(P, ps, Hkv, D, dtype=BF, device=DEV) for _ in range(2))
    lengths = [130, 1, 64]
    table = torch.tensor([[P - 1, P - 5, P - 2], [P - 3, 0, 0], [P - 4, 0, 0]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(31)
    ks, vs = ([torch.randn(n, Hkv, D, generator=g).to(BF) for n in lengths] for _ in range(2))
    cu = torch.tensor([0, 130, 131, 195], dtype=torch.int32, device=DEV)
    sparda.append_paged(kp, vp, table, torch.zeros(3, dtype=torch.int32, device=DEV), torch.cat(ks).to(DEV),
                        torch.cat(vs).to(DEV), cu_seqlens=cu)
    q = queries(3, 32, D, BF, seed=32)
    got = sparda.decode_paged(q.to(DEV), kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check(got, q, ks, vs)
    assert sparda.status() == 0


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_sequences_that_share_pages(dtype):
    print(f"[case] paged shared pages {dtype}", flush=True)
    lengths = [700, 480, 700, 1]
    kp, vp, table, ks, vs = cache([700], 16, 2, 64, dtype, seed=12)
    q = queries(4, 6, 64, dtype, seed=13)
    got = sparda.decode_paged(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV).expand(4, -1),
                              torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check(got, q, [ks[0][:n] for n in lengths], [vs[0][:n] for n in lengths])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("width", [None, 512])
def test_paged_values_that_are_not_finite(dtype, width):
    """Scores of -inf at a sequence's first keys, at all of another's; an infinite
    value at one position of a third: in one share a sequence, and in several."""
    print(f"[case] paged not finite {dtype} {width}", flush=True)
    lengths, D = [300, 90, 300, 300], 64
    kp, vp, table, ks, vs = cache(lengths, 32, 1, D, dtype, seed=14, width=width)
    q = queries(4, 2, D, dtype, seed=15)
    q[..., 0] = q[..., 0].abs() + 0.5
    for b, upto in ((0, 200), (1, 90)):
        for p in range(upto):
            kp[table[b, p // 32], p % 32, 0, 0] = -float("inf")
    vp[table[2, 100 // 32], 100 % 32, 0, 5] = float("inf")
    got = sparda.decode_paged(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV),
                              torch.tensor(lengths, dtype=torch.int32, device=DEV)).cpu()
    assert torch.isnan(got[1].float()).all()             # no key with a weight: 0 / 0
    assert (got[2].view(2, D)[:, 5] == float("inf")).all()
    check(got[3:], q[3:], ks[3:], vs[3:])
    check(got[:1], q[:1], [ks[0][200:]], [vs[0][200:]])
    got[2].view(2, D)[:, 5] = 0                          # (the cache's own copy of that value is finite)
    vs[2][:, :, 5] = 0
    check(got[2:3], q[2:3], ks[2:3], vs[2:3])
    assert sparda.status() == 0


def test_paged_calls_on_two_streams_at_once():
    print("[case] paged two streams", flush=True)
    sets = []
    for seed, lengths in ((1, [9000, 40, 0, 3000]), (2, [5000, 7000, 12, 1])):
        kp, vp, table, _, _ = cache(lengths, 64, 4, 64, BF, seed=seed)
        q = queries(4, 12, 64, BF, seed=seed)
        sets.append([x.to(DEV) for x in (q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32))])
    want = [sparda.decode_paged(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(sparda.decode_paged(*sets[i]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,Hq,Hkv,D", [(4, 40, 2, 64), (4, 128, 1, 64), (70, 12, 4, 64), (130, 6, 2, 128), (70, 5, 1, 32)])
def test_paged_decode_in_a_wide_table(dtype, B, Hq, Hkv, D):
    """A table far wider than the sequences: many heads a KV head, neighbouring
    heads together, more sequences than lanes."""
    print(f"[case] paged wide table {dtype} {B} {Hq}/{Hkv}x{D}", flush=True)
    r = np.random.default_rng(B + Hq)
    lengths = [int(x) for x in r.integers(0, 1500 if B < 10 else 300, B)]
    lengths[1], lengths[-1] = 0, 1200
    kp, vp, table, ks, vs = cache(lengths, 32, Hkv, D, dtype, seed=B, width=512)
    q = queries(B, Hq, D, dtype, seed=16) * 2
    args = [x.to(DEV) for x in (q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32))]
    got = sparda.decode_paged(*args)
    check(got, q, ks, vs)
    assert torch.equal(got, sparda.decode_paged(*args)) and sparda.status() == 0
