"""Pages of 4-bit codes: the write is the format's definition byte by byte, what is read back are
its values, and the attention over them is compared with float64 (bounds: q4_oracle)."""

import numpy as np
import pytest
import torch

import sparda
from helpers import np32
from model.rope import rope_tables
from q4_oracle import attend, codes, held, put, turn, values
from test_gpu_rotate import dev, randn, server

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def written(P, ps, Hkv, D, table, olds, cu, kn, vn, fill=0):
    """Pages on the CPU as a plain loop over the rows writes them. kn, vn fp32 numpy [N,Hkv,D], rotated."""
    pages = np.full(sparda.q4_page_shape(P, ps, Hkv, D), fill, np.uint8)
    for b, old in enumerate(olds):
        if old < 0:
            continue
        for j, t in enumerate(range(cu[b], cu[b + 1])):
            p = old + j
            for h in range(Hkv):
                put(pages[int(table[b, p // ps])], h, p % ps, kn[t, h], vn[t, h])
    return torch.from_numpy(pages)


# codes of dims that a head of 16 does not have are not looked at
def same_pages(got, want, D):
    if D != 16:
        return torch.equal(got, want)
    real = torch.ones(576, dtype=torch.bool)
    i = torch.arange(576)
    real[:256] = i[:256] % 16 < 8                 # quarters 0 and 1 of a key
    real[256:512] = (i[256:512] - 256) // 4 % 16 < 8   # words 0 .. 7 of a value
    return torch.equal(got[..., real], want[..., real])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (8, 2, 128), (3, 1, 32), (5, 5, 16), (9, 9, 64)])
@pytest.mark.parametrize("news,olds,ps", [([1], [0], 16), ([1, 1, 1, 1], [5, 0, -1, 47], 16),
                                          ([0, 19, 1, 34, 3], [7, 15, 63, 0, -1], 64)], ids=str)
def test_append_writes_the_format(dtype, Hq, Hkv, D, news, olds, ps):
    print(f"[case] append q4 {dtype} {Hq}/{Hkv}x{D} {news} {olds} ps={ps}", flush=True)
    cu = np.concatenate(([0], np.cumsum(news))).tolist()
    one = max(news) == min(news) == 1
    N = cu[-1] + (0 if one else 2)
    table, P = server(news, olds, ps, seed=D + ps)
    q, kn, vn = randn(N, Hq, D, dtype=dtype, seed=3), randn(N, Hkv, D, dtype=dtype, seed=4) * 3, randn(N, Hkv, D, dtype=dtype, seed=5)
    cos, sin = rope_tables(D, 600)
    pos = torch.zeros(N, dtype=torch.long)
    for b, old in enumerate(olds):
        for j, t in enumerate(range(cu[b], cu[b + 1])):
            pos[t] = max(old, 0) + j
    offs = None if one else dev(cu)
    rows = [t for b, o in enumerate(olds) if o >= 0 for t in range(cu[b], cu[b + 1])]
    for fill in (0, 0x5A):
        # without and with the rotation
        pages = torch.full(sparda.q4_page_shape(P, ps, Hkv, D), fill, dtype=torch.uint8, device=DEV)
        assert sparda.append_paged_q4(pages, dev(table), dev(olds), dev(kn), dev(vn), offs) is None
        assert same_pages(pages.cpu(), written(P, ps, Hkv, D, table, olds, cu, np32(kn), np32(vn), fill), D)
        pages.fill_(fill)
        got = sparda.append_paged_q4(pages, dev(table), dev(olds), dev(kn), dev(vn), offs, dev(q), dev(cos), dev(sin))
        turned = turn(kn, cos, sin, pos).numpy()
        assert same_pages(pages.cpu(), written(P, ps, Hkv, D, table, olds, cu, turned, np32(vn), fill), D)
        assert torch.equal(got.cpu()[rows], turn(q, cos, sin, pos).to(dtype)[rows])
    # keys alone rotated; out kept where no sequence is; in place
    again, out = torch.full_like(pages, fill), dev(q)
    assert sparda.append_paged_q4(again, dev(table), dev(olds), dev(kn), dev(vn), offs, None, dev(cos), dev(sin)) is None
    assert torch.equal(again, pages)
    assert sparda.append_paged_q4(again, dev(table), dev(olds), dev(kn), dev(vn), offs, out, dev(cos), dev(sin), out=out) is out
    rest = [t for t in range(N) if t not in set(rows)]
    assert torch.equal(out[rows], got[rows]) and torch.equal(out.cpu()[rest], q[rest])
    # read back
    for dt in (BF, F32):
        k, v = sparda.gather_paged_q4(pages, dev(table), dev(olds), N, offs, head_dim=D, dtype=dt)
        for x, y in ((k, turned), (v, np32(vn))):
            want = torch.from_numpy(held(y).astype(np.float32)).to(dt)
            assert x.dtype == dt and torch.equal(x.cpu()[rows], want[rows])
    assert sparda.status() == 0


def test_values_of_every_size():
    """Zeros, the smallest and largest numbers, ties of the levels, and values that are not finite, a group each."""
    print("[case] q4 sizes", flush=True)
    D, n = 128, 16
    x = randn(n, 1, D, dtype=F32, seed=1)
    scales = [0.0, 2.0 ** -149, 2.0 ** -30, 2.0 ** -24, 1e-6, 1e-3, 1.0, 100.0, 7.5, 15.0, 6e4, 9e5, 2e6, 1e30, 3e38, 1.0]
    x *= torch.tensor(scales)[:, None, None]
    x[8] = (torch.arange(128) % 16 - 7.5).view(1, D)              # on the levels and
    x[9] = (torch.arange(128) % 31 - 15.0).view(1, D)             # between them
    x[10, 0, 32:64], x[11, 0, 64:96] = 0.0, -0.0
    x[15, 0, 5], x[15, 0, 40], x[15, 0, 70] = float("inf"), float("nan"), float("-inf")
    x = x.to(BF)
    table, pos = dev([[0]]), dev([0])
    pages = torch.zeros(sparda.q4_page_shape(1, 16, 1, D), dtype=torch.uint8, device=DEV)
    sparda.append_paged_q4(pages, table, pos, dev(x), dev(x.flip(0)), dev([0, n]))
    k, v = sparda.gather_paged_q4(pages, table, pos, n, dev([0, n]), dtype=F32)
    want = torch.from_numpy(held(np32(x)).astype(np.float32))
    assert torch.equal(k.cpu().isnan(), want.isnan()) and torch.equal(k.cpu().nan_to_num(), want.nan_to_num())
    assert torch.equal(v.cpu().nan_to_num(), want.flip(0).nan_to_num())
    assert want[15, 0, :96].isnan().all() and not want[15, 0, 96:].isnan().any() and (want[0] == 0).all()
    # the format's own claim: a value is off by h at most, within its range
    c, h = codes(np32(x)[:, 0])
    fine = np.isfinite(h) & (h > 0) & (h < 65504)
    err = np.abs(values(c, h) - np32(x)[:, 0].astype(np.float64)).reshape(n, 4, 32).max(-1)
    assert (err[fine] <= h.astype(np.float64)[fine] * (1 + 15 * 2.0 ** -11) + 15 * 2.0 ** -25).all()


def cache(lengths, ps, Hkv, D, seed, width=None, spare=3):
    """Pages written by the plain loop, NaN numbers in every row that no sequence holds; held keys, values, h."""
    g = np.random.default_rng(seed)
    need = [(n + ps - 1) // ps for n in lengths]
    P = sum(need) + spare
    order = g.permutation(P)
    shape = sparda.q4_page_shape(P, ps, Hkv, D)
    G = shape[3] // 576
    pages = np.full(shape, 0xFF, np.uint8)
    table = torch.full((len(lengths), width or max(1, max(need))), 1 << 30, dtype=torch.int32)
    out, at = [], 0
    flat = pages.reshape(P, Hkv, -1, 576 * G)
    for b, n in enumerate(lengths):
        k, v = (bf(g.standard_normal((n, Hkv, D))) for _ in range(2))
        (ck, hk), (cv, hv) = codes(k), codes(v)
        for i in range(need[b]):
            table[b, i] = int(order[at])
            rows = slice(i * ps, min(n, (i + 1) * ps))
            fill(flat[order[at]], ck[rows], hk[rows], cv[rows], hv[rows])
            at += 1
        out.append((values(ck, hk), values(cv, hv), hk, hv))
    return torch.from_numpy(pages), table, out


def bf(x):
    return torch.from_numpy(x).to(BF).float().numpy()


def fill(page, ck, hk, cv, hv):
    """Rows [n,Hkv,...] into a page [Hkv,tiles,576 G] from its first row on (vectorised ``put``)."""
    n, Hkv, D = ck.shape
    G = hk.shape[-1]
    r = np.arange(n)
    tile, i = r // 16, r % 16
    for d in range(D):
        g, e = d // 32, d % 32
        m = e % 8 // 2 + 4 * (e % 2)
        at = 16 * G * i + 4 * G * (e // 8) + 4 * g + m // 2
        for h in range(Hkv):
            page[h, tile, at] = page[h, tile, at] & (0xF0 if m % 2 == 0 else 0x0F) | ck[:, h, d] << 4 * (m % 2)
        at = 256 * G + 4 * G * (16 * (i // 4) + e // 2) + 4 * g + np.array([0, 2, 1, 3])[i % 4]
        for h in range(Hkv):
            page[h, tile, at] = page[h, tile, at] & (0xF0 if e % 2 == 0 else 0x0F) | cv[:, h, d] << 4 * (e % 2)
    for w, x in ((0, hk), (32 * G, hv)):
        b = np.ascontiguousarray(x).view(np.uint8).reshape(n, Hkv, 2 * G)
        for j in range(2 * G):
            for h in range(Hkv):
                page[h, tile, 512 * G + w + 2 * G * i + j] = b[:, h, j]


def check(got, q, lengths, rows, scale=None):
    if q.dim() == 3:
        q, got = q[:, None], got[:, None]
    B, T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    got = np32(got).astype(np.float64).reshape(B, T, Hq, D)
    worst = 0.0
    for b, (k, v, hk, hv) in enumerate(rows):
        R = Hq // k.shape[1]
        for t in range(T):
            n = lengths[b] - T + 1 + t
            if n <= 0:
                assert (got[b, t] == 0).all()
                continue
            for g in range(k.shape[1]):
                want, tb, tf = attend(np32(q[b, t, g * R:(g + 1) * R]).astype(np.float64), k[:n, g], v[:n, g], hk[:n, g], hv[:n, g],
                                      scale)
                tol = tb if q.dtype == BF else tf
                err = np.abs(got[b, t, g * R:(g + 1) * R] - want)
                worst = max(worst, (err / tol).max())
                assert (err <= tol).all(), f"sequence {b} token {t} group {g}: {(err / tol).max():.2f} of the bound"
    return worst


HEADS = [(12, 4, 64), (4, 4, 64), (8, 1, 128), (6, 3, 128), (34, 2, 64), (3, 1, 32), (4, 2, 16)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("lengths,ps", [([1], 16), ([1000], 16), ([0, 5, 16, 17, 33, 300], 16), ([64, 1, 0, 129], 64),
                                        ([47, 49, 48, 200], 48)], ids=str)
def test_decode_against_float64(dtype, Hq, Hkv, D, lengths, ps):
    print(f"[case] q4 {dtype} {Hq}/{Hkv}x{D} {lengths} ps={ps}", flush=True)
    pages, table, rows = cache(lengths, ps, Hkv, D, seed=sum(lengths) + D)
    q = randn(len(lengths), Hq, D, dtype=dtype, seed=7)
    sparda.status()
    got = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths))
    print("  of the bound:", check(got, q, lengths, rows))
    assert sparda.status() == 0


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (16, 2, 128), (6, 2, 16), (3, 3, 32)])
@pytest.mark.parametrize("T", [2, 5, 64])
@pytest.mark.parametrize("lengths", [[70, 3, 0, 400, 64], [4100, 1]], ids=str)
def test_decode_of_several_tokens(dtype, Hq, Hkv, D, T, lengths):
    print(f"[case] q4 {T} tokens {dtype} {Hq}/{Hkv}x{D} {lengths}", flush=True)
    pages, table, rows = cache(lengths, 32, Hkv, D, seed=D + T)
    q = randn(len(lengths), T, Hq, D, dtype=dtype, seed=8)
    got = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths))
    assert got.shape == (len(lengths), T, Hq * D)
    print("  of the bound:", check(got, q, lengths, rows))
    if T == 2:    # one token is the form without that dimension
        a = sparda.decode_paged_q4(dev(q[:, 1:].contiguous()), dev(pages), dev(table), dev(lengths))
        assert torch.equal(a[:, 0], sparda.decode_paged_q4(dev(q[:, 1].contiguous()), dev(pages), dev(table), dev(lengths)))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (16, 2, 128), (34, 1, 128), (4, 2, 16)])
@pytest.mark.parametrize("lengths", [[20011], [3, 9000, 0, 5000, 1]], ids=str)
def test_decode_over_many_shares(dtype, Hq, Hkv, D, lengths):
    print(f"[case] q4 long {dtype} {Hq}/{Hkv}x{D} {lengths}", flush=True)
    pages, table, rows = cache(lengths, 64, Hkv, D, seed=5, width=512)
    q = randn(len(lengths), Hq, D, dtype=dtype, seed=8) * 2
    got = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths))
    print("  of the bound:", check(got, q, lengths, rows))
    again = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths))
    assert torch.equal(got, again)                # no sum depends on timing


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,T", [(12, 4, 64, 1), (8, 2, 128, 1), (8, 1, 128, 5), (4, 1, 128, 5), (6, 2, 64, 7), (34, 2, 64, 2), (4, 2, 16, 3), (8, 8, 32, 1)])
def test_decode_with_tables_of_large_capacity(dtype, Hq, Hkv, D, T):
    """More codes than the last-level cache holds, were the tables full: other loads, the same results."""
    G = max(1, D // 32)
    width = (257 << 20) // (2 * 16 * Hkv * G * 36) + 1
    lengths = [700, 2001]
    print(f"[case] q4 capacity {dtype} {Hq}/{Hkv}x{D} T={T} width {width}", flush=True)
    pages, table, rows = cache(lengths, 16, Hkv, D, seed=6, width=width)
    q = randn(2, T, Hq, D, dtype=dtype, seed=7) * 2
    got = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths))
    print("  of the bound:", check(got, q, lengths, rows))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 128), (5, 1, 128), (8, 1, 64), (9, 1, 64), (2, 2, 128), (16, 1, 32), (16, 1, 128), (17, 1, 128),
                                      (40, 2, 128), (21, 1, 128), (17, 1, 64), (48, 2, 64), (25, 1, 64), (18, 1, 32), (24, 1, 16)])
def test_decode_at_the_number_of_columns_that_changes_the_form(dtype, Hq, Hkv, D):
    lengths = [333, 31, 32, 0, 2500]
    print(f"[case] q4 columns {dtype} {Hq}/{Hkv}x{D}", flush=True)
    pages, table, rows = cache(lengths, 16, Hkv, D, seed=11)
    q = randn(len(lengths), Hq, D, dtype=dtype, seed=12) * 3
    got = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths))
    print("  of the bound:", check(got, q, lengths, rows))
    # a column does not see what the others hold
    q[:, :-1] = float("nan")
    alone = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths)).view(len(lengths), Hq, D)
    assert torch.equal(alone[:, -1], got.view(len(lengths), Hq, D)[:, -1])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.5, 4.0])
def test_decode_other_scales(dtype, scale):
    print(f"[case] q4 scale {scale} {dtype}", flush=True)
    lengths = [333, 40]
    pages, table, rows = cache(lengths, 16, 2, 64, seed=2)
    q = randn(2, 6, 64, dtype=dtype, seed=3)
    check(sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths), scale=scale), q, lengths, rows, scale)


@pytest.mark.parametrize("T", [1, 3])
def test_rows_behind_a_token_and_lost_pages(T):
    """A row that is not finite changes the tokens that see it alone; so does a page that is not there."""
    print(f"[case] q4 values not finite, {T} tokens", flush=True)
    lengths, Hq, Hkv, D = [100, 37, 1, 640], 6, 2, 64
    pages, table, rows = cache(lengths, 16, Hkv, D, seed=12)
    q = dev(randn(4, T, Hq, D, dtype=BF, seed=3))
    good = sparda.decode_paged_q4(q, dev(pages), dev(table), dev(lengths))
    p = dev(pages)
    x = torch.full((4, Hkv, D), float("nan"), dtype=BF, device=DEV)
    sparda.append_paged_q4(p, dev(table), dev([99, 36, -1, -1]), x, x)        # the last tokens' own rows
    got = sparda.decode_paged_q4(q, p, dev(table), dev(lengths))
    assert got[:2, -1].isnan().all() and torch.equal(got[2:], good[2:]) and torch.equal(got[:2, :-1], good[:2, :-1])
    assert sparda.status() == 0
    lost, at = table.clone(), dev([100, 37, 1 << 20, 640])
    lost[0, 3], lost[3, 20] = -1, pages.shape[0]
    got = sparda.decode_paged_q4(q, dev(pages), dev(lost), at)
    assert got[[0, 2, 3]].isnan().all() and torch.equal(got[1], good[1])
    assert sparda.status() == sparda.STATUS_PAGE_RANGE
    got = sparda.decode_paged_q4(q, dev(pages), dev(table), dev([100, 37, -5, 640]))
    assert got[2].isnan().all() and torch.equal(got[[0, 1, 3]], good[[0, 1, 3]])
    assert sparda.status() == sparda.STATUS_PAGE_RANGE
    k, v = sparda.gather_paged_q4(dev(pages), dev(lost), dev([50, 0, -1, 330]), 4)
    assert k[0].isnan().all() and v[0].isnan().all() and not k[1].isnan().any() and k[3].isnan().all()
    assert sparda.status() == sparda.STATUS_PAGE_RANGE


def test_strided_queries_pages_and_outputs():
    print("[case] q4 strides", flush=True)
    lengths, Hq, Hkv, D, T = [300, 77], 6, 2, 128, 3
    pages, table, rows = cache(lengths, 32, Hkv, D, seed=4)
    q = randn(2, T, Hq, D, dtype=BF, seed=5)
    want = sparda.decode_paged_q4(dev(q), dev(pages), dev(table), dev(lengths))
    layers = torch.zeros(pages.shape[0], 3, *pages.shape[1:], dtype=torch.uint8, device=DEV)   # pages of three layers
    layers[:, 1] = dev(pages)
    wide = torch.zeros(2, Hq, T, D + 8, dtype=BF, device=DEV)
    wide[..., :D] = dev(q).transpose(1, 2)
    wt = torch.full((2, table.shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    wt[:, :-3] = dev(table)
    out = torch.zeros(2, T * Hq * D + 16, dtype=BF, device=DEV)
    got = sparda.decode_paged_q4(wide[..., :D].transpose(1, 2), layers[:, 1], wt[:, :-3], dev(lengths),
                                 out=out[:, :T * Hq * D].view(2, T, Hq * D))
    assert torch.equal(got, want) and (out[:, T * Hq * D:] == 0).all()
    odd = torch.zeros(q.numel() + 1, dtype=BF, device=DEV)[1:].view(q.shape)      # rows off 16 bytes
    odd.copy_(q)
    assert torch.equal(sparda.decode_paged_q4(odd, dev(pages), dev(table), dev(lengths)), want)
    k, v = randn(2, Hkv, D, dtype=BF, seed=6).to(DEV), randn(2, Hkv, D, dtype=BF, seed=7).to(DEV)
    plain = dev(pages)
    sparda.append_paged_q4(plain, dev(table), dev([299, 70]), k, v)
    sparda.append_paged_q4(layers[:, 1], wt[:, :-3], dev([299, 70]), k, v)
    assert torch.equal(layers[:, 1], plain) and (layers[:, 0] == 0).all() and (layers[:, 2] == 0).all()
    a = sparda.gather_paged_q4(layers[:, 1], wt[:, :-3], dev([299, 70]), 2)
    b = sparda.gather_paged_q4(plain, dev(table), dev([299, 70]), 2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_pages_past_32_bit_offsets():
    print("[case] q4 pages past 2^32 bytes", flush=True)
    shape = sparda.q4_page_shape(4_000_000, 16, 1, 64)            # 4.6 GB
    pages = torch.empty(shape, dtype=torch.uint8, device=DEV)
    table = dev([[3_999_999, 5], [3_800_001, 3_999_998]])
    k, v, q = (randn(40, 1, 64, dtype=BF, seed=s).to(DEV) for s in (1, 2, 3))
    sparda.append_paged_q4(pages, table, dev([0, 0]), k, v, dev([0, 20, 40]))
    a, b = sparda.gather_paged_q4(pages, table, dev([0, 0]), 40, dev([0, 20, 40]), dtype=F32)
    assert torch.equal(a.cpu().double(), torch.from_numpy(held(np32(k)))) and torch.equal(b.cpu().double(), torch.from_numpy(held(np32(v))))
    got = sparda.decode_paged_q4(q[:2], pages, table, dev([20, 20]))
    rows = [(held(np32(k))[i:i + 20], held(np32(v))[i:i + 20], codes(np32(k))[1][i:i + 20], codes(np32(v))[1][i:i + 20]) for i in (0, 20)]
    check(got, q[:2].cpu(), [20, 20], rows)
    assert sparda.status() == 0


def test_a_page_of_more_than_two_gibibytes():
    """Offsets inside one page pass 32 bits: rows before and behind that place are written, read and attended to."""
    print("[case] q4 page of 2.1 GB", flush=True)
    D, ps = 128, 16 * 932_300                                     # 932068 tiles of 2304 bytes are 2^31
    pages = torch.zeros(sparda.q4_page_shape(1, ps, 1, D), dtype=torch.uint8, device=DEV)
    table, n = dev([[0]]), 40
    at = [5, 16 * 932_060, ps - n]
    k, v = randn(n, 1, D, dtype=BF, seed=1), randn(n, 1, D, dtype=BF, seed=2)
    for p in at:
        sparda.append_paged_q4(pages, table, dev([p]), dev(k), dev(v), dev([0, n]))
    kh, vh = held(np32(k)), held(np32(v))
    for p in at:
        got = sparda.gather_paged_q4(pages, table, dev([p]), n, dev([0, n]), dtype=F32)
        assert np.array_equal(got[0].cpu().numpy(), kh.astype(np.float32)) and np.array_equal(got[1].cpu().numpy(), vh.astype(np.float32))
    # (the other rows are zeros: a score of 0 each and no value)
    q = (dev(k[:2]) * 3).view(1, 2, D)
    for length in (ps, ps - n // 2, 16 * 932_060 + n):
        out = sparda.decode_paged_q4(q, pages, table, dev([length]))[0].view(2, D).cpu().double().numpy()
        rows = [r for p in at for r in range(n) if p + r < length]
        s = np32(q.cpu()).astype(np.float64)[0] @ kh[rows, 0].T / D ** 0.5
        w = np.exp(s - s.max(-1, keepdims=True))
        rest = (length - len(rows)) * np.exp(-s.max(-1, keepdims=True))
        want = w @ vh[rows, 0] / (w.sum(-1, keepdims=True) + rest)
        # (outputs are of the size of 1: the weights' and the result's rounding to bf16, 2^-8 each of a sum's terms)
        assert np.abs(out - want).max() <= 2 * 2.0 ** -8 * np.abs(vh).max() and np.abs(want).max() > 0.5


def test_refusals_of_tensors_that_do_not_fit():
    print("[case] q4 refusals", flush=True)
    q, kn = randn(3, 4, 64, dtype=BF, seed=1).to(DEV), randn(3, 2, 64, dtype=BF, seed=2).to(DEV)
    pages = torch.zeros(sparda.q4_page_shape(3, 16, 2, 64), dtype=torch.uint8, device=DEV)
    table, pos = dev([[0], [1], [2]]), dev([0, 1, 2])
    cos, sin = (dev(x) for x in rope_tables(64, 32))
    good = dict(pages=pages, page_table=table, positions=pos, k_new=kn, v_new=kn.clone())
    sparda.append_paged_q4(**good)
    for bad, err in ((dict(pages=pages.int()), TypeError), (dict(pages=pages[..., :576]), ValueError), (dict(pages=pages[0]), ValueError),
                     (dict(k_new=kn[..., :32].contiguous(), v_new=kn[..., :32].contiguous()), ValueError),
                     (dict(k_new=kn.float()), TypeError), (dict(k_new=kn.half(), v_new=kn.half()), TypeError), (dict(q=q), ValueError),
                     (dict(cos=cos), ValueError), (dict(cos=cos, sin=sin, q=q.float()), TypeError),
                     (dict(cos=cos, sin=sin, out=torch.empty_like(q)), ValueError), (dict(positions=pos.long()), TypeError),
                     (dict(cu_seqlens=dev([0, 3])), ValueError), (dict(page_table=table.long()), TypeError),
                     (dict(k_new=kn[:2], v_new=kn[:2]), ValueError), (dict(k_new=kn.clone().requires_grad_()), RuntimeError)):
        with pytest.raises(err):
            sparda.append_paged_q4(**{**good, **bad})
    good = dict(q=q, pages=pages, page_table=table, lengths=pos)
    sparda.decode_paged_q4(**good)
    for bad, err in ((dict(q=q.half()), TypeError), (dict(q=q[..., :32].contiguous()), ValueError), (dict(q=q[:2]), ValueError),
                     (dict(q=q[:, None, None]), ValueError), (dict(q=q[:, :3]), ValueError), (dict(lengths=pos.long()), TypeError),
                     (dict(lengths=pos[:2]), ValueError), (dict(q=q[:, None].expand(3, 65, 4, 64)), ValueError),
                     (dict(out=torch.empty(3, 256, device=DEV)), ValueError), (dict(pages=torch.zeros(3, 2, 3, 1152, dtype=torch.uint8, device=DEV)[:, :, ::2]), ValueError),
                     (dict(q=q.clone().requires_grad_()), RuntimeError), (dict(pages=pages.cpu()), RuntimeError)):
        with pytest.raises(err):
            sparda.decode_paged_q4(**{**good, **bad})
    for bad, err in ((dict(rows=2), ValueError), (dict(rows=-1), ValueError), (dict(rows=3, head_dim=128), ValueError),
                     (dict(rows=3, dtype=torch.float16), TypeError), (dict(rows=3, cu_seqlens=dev([0, 3])), ValueError)):
        with pytest.raises(err):
            sparda.gather_paged_q4(pages, table, pos, **bad)
