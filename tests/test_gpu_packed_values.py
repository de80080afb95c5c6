"""Packed prompts whose values are large where their scores rise far above the
first keys': a weight against a reference taken early times a value may pass the
type's range although the output, a mean of values, does not."""

import numpy as np
import pytest
import torch

import sparda
from packed_oracle import attend
from test_gpu_packed import BF, DEV, F32, check, offsets

pytestmark = pytest.mark.gpu

SCALE = float(np.float32(np.log(2.0)))   # a score in log2 units is the dot product

# one size for every form of the launch
FORMS = [(BF, 12, 4, 64, [500]), (BF, 12, 4, 64, [2000]), (BF, 12, 4, 64, [4200]), (BF, 12, 4, 64, [700] * 8),
         (BF, 12, 4, 64, [9000, 13001]), (BF, 12, 4, 32, [900, 77]), (BF, 32, 8, 128, [400]), (BF, 8, 2, 128, [4300]),
         (BF, 32, 8, 128, [3000, 2000]), (BF, 6, 2, 64, [200, 61]), (BF, 8, 2, 16, [700, 61]), (F32, 6, 2, 64, [300, 61])]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lift,vexp", [(60, 70), (27, 100), (40, 112)])
@pytest.mark.parametrize("dtype,Hq,Hkv,D,lengths", FORMS, ids=str)
def test_large_values_at_keys_far_above_the_first(dtype, Hq, Hkv, D, lengths, lift, vexp, causal):
    print(f"[case] packed values {dtype} {Hq}/{Hkv}x{D} {lengths} lift={lift} 2^{vexp} causal={causal}", flush=True)
    cu = offsets(lengths)
    N = int(cu[-1])
    g = torch.Generator().manual_seed(N + lift)
    q, k, v = (torch.randn(N, h, D, generator=g) for h in (Hq, Hkv, Hkv))
    q[..., 0], k[..., 0], q[..., 1:], k[..., 1:] = 1.0, 0.0, q[..., 1:] * 0.25, k[..., 1:] * 0.25
    for a, b in zip(cu, cu[1:]):
        k[a + 40:b:37, :, 0] = lift      # (37: every key group and every place in a block has some)
    q, k, v = q.to(dtype), k.to(dtype), (v * 2.0 ** vexp).to(dtype)
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV), causal=causal, scale=SCALE)
    assert torch.isfinite(got.float()).all()
    rows = sorted({int(c) + d for c in cu for d in (-2, -1, 0, 1, 39, 40, 41, 77, 78, 120) if 0 <= c + d < N}
                  | {int(x) for x in np.random.default_rng(N).integers(0, N, 12)})
    check(got, q, k, v, cu, causal, scale=SCALE, rows=rows)


@pytest.mark.parametrize("Hq,Hkv,D,lengths", [f[1:] for f in FORMS if f[0] == BF], ids=str)
def test_products_that_pass_the_range_only_when_key_groups_are_added(Hq, Hkv, D, lengths):
    """Weights of 2^27 times values of 1.5 2^100: every product is finite, the sum
    of two is not, their mean is 1.5 2^100."""
    print(f"[case] packed value sums {Hq}/{Hkv}x{D} {lengths}", flush=True)
    cu = offsets(lengths)
    N = int(cu[-1])
    q, k, v = (torch.zeros(N, h, D, dtype=BF) for h in (Hq, Hkv, Hkv))
    q[..., 0] = 1.0
    a, b = int(cu[-2]), int(cu[-1])
    for block in (32, 64):               # a place in the second and in the third block of keys
        k.zero_(), v.zero_()
        ats = [a + i * block + 5 for i in (1, 2) if a + i * block + 5 < b]
        for at in ats:
            k[at, :, 0], v[at] = 27.0, 1.5 * 2.0 ** 100
        got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV), scale=SCALE)
        check(got, q, k, v, cu, scale=SCALE, rows=sorted({a, *ats, a + 60, (a + b) // 2, b - 1}))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D,lengths", [f[1:] for f in FORMS if f[0] == BF], ids=str)
def test_large_values_beside_an_infinite_one(Hq, Hkv, D, lengths, causal):
    print(f"[case] packed values beside inf {Hq}/{Hkv}x{D} {lengths} causal={causal}", flush=True)
    cu = offsets(lengths)
    N, R = int(cu[-1]), Hq // Hkv
    a, b = int(cu[-2]), int(cu[-1])
    g = torch.Generator().manual_seed(N)
    q, k, v = (torch.randn(N, h, D, generator=g) for h in (Hq, Hkv, Hkv))
    q[..., 0], k[..., 0], q[..., 1:], k[..., 1:] = 1.0, 0.0, q[..., 1:] * 0.25, k[..., 1:] * 0.25
    k[a + 40:b:19, :, 0] = 60.0
    q, k, v = q.to(BF), k.to(BF), (v * 2.0 ** 70).to(BF)
    at = a + 40                                  # the inf has a weight in every row that may attend it
    v[at, Hkv - 1, 5] = float("inf")
    got = sparda.prefill_packed(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(cu).to(DEV), causal=causal, scale=SCALE)
    got = got.view(N, Hq, D).cpu()
    hit = torch.zeros(N, Hq, D, dtype=torch.bool)
    hit[(at if causal else a):b, Hq - R:, 5] = True
    assert torch.equal(~torch.isfinite(got), hit)
    keep = [d for d in range(D) if d != 5]
    qn, kn, vn, gn = (x.float().numpy().astype(np.float64) for x in (q, k, v, got))
    for t in sorted({a, a + 39, at, a + 45, a + 60, (a + b) // 2, b - 1}):
        e = t + 1 if causal else b
        for h in range(Hkv):
            want, bf, _ = attend(qn[t, h * R:(h + 1) * R], kn[a:e, h], vn[a:e, h][:, keep], SCALE)
            assert (np.abs(gn[t, h * R:(h + 1) * R][:, keep] - want) <= bf).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("Hq,Hkv,D,lengths", [f[1:] for f in FORMS if f[0] == BF], ids=str)
def test_a_value_that_is_not_finite_changes_no_other_bit(Hq, Hkv, D, lengths, bad, causal):
    # under weights of 2^20 against the first keys, and ordinary values
    print(f"[case] packed {bad} alone {Hq}/{Hkv}x{D} {lengths} causal={causal}", flush=True)
    cu = offsets(lengths)
    N, R = int(cu[-1]), Hq // Hkv
    a, b = int(cu[-2]), int(cu[-1])
    g = torch.Generator().manual_seed(N + 1)
    q, k, v = (torch.randn(N, h, D, generator=g) for h in (Hq, Hkv, Hkv))
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[a + 40:b:19, :, 0] = 20.0
    q, k, v = q.to(BF).to(DEV), k.to(BF).to(DEV), v.to(BF).to(DEV)
    cud = torch.from_numpy(cu).to(DEV)
    clean = sparda.prefill_packed(q, k, v, cud, causal=causal, scale=SCALE).view(N, Hq, D)
    assert torch.isfinite(clean).all()
    for at in (a + 2, a + 40):
        v2 = v.clone()
        v2[at, Hkv - 1, 5] = bad
        got = sparda.prefill_packed(q, k, v2, cud, causal=causal, scale=SCALE).view(N, Hq, D)
        hit = torch.zeros(N, Hq, D, dtype=torch.bool, device=DEV)
        hit[(at if causal else a):b, Hq - R:, 5] = True
        assert torch.equal(~torch.isfinite(got), hit)
        assert torch.equal(got[~hit], clean[~hit])
