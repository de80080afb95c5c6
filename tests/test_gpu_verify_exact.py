"""Verification next to its borders: what is accepted and which token is drawn are float64's, whatever the size of the
batch that the sequence is in."""

import numpy as np
import pytest
import torch

import sparda

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
B, V = 24, 50257                       # 2.4 M logits with a draft each


def case(dtype, temperature, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, 2, V, generator=g) * 3 * (temperature if temperature < 1e-30 else 1)).to(dtype)
    p = torch.softmax(x.double() / float(np.float32(temperature)), -1)
    return g, x, p


def alone(x, drafts, u, probs, temperature):
    """The same, a sequence a call."""
    r = [sparda.verify_drafts(x[b:b + 1], drafts[b:b + 1], u[b:b + 1], probs[b:b + 1] if probs is not None else None,
                              temperature=temperature) for b in range(B)]
    return torch.cat([t for t, _ in r]), torch.cat([n for _, n in r])


@pytest.mark.parametrize("dtype,temperature", [(BF, 1.0), (BF, 0.5), (F32, 1.0), (F32, 0.5), (F32, 1e-39)])   # (the last: 1 / T is no fp32 number)
@pytest.mark.parametrize("given", [True, False], ids=["probs", "tokens"])
def test_acceptance_next_to_its_border(dtype, temperature, given):
    """u q and p closer than fp32 tells apart: u is the fp32 number below or above p / q. (p in float64 is right to 1e-14;
    where u q is closer than 1e-11 of p, u moves on.)"""
    print(f"[case] verify border {dtype} {temperature} {given}", flush=True)
    g, x, p = case(dtype, temperature, seed=17)
    drafts = p[:, 0].topk(40).indices.gather(1, torch.randint(0, 40, (B, 1), generator=g)).int()
    pd = p[:, 0].gather(1, drafts.long())[:, 0].numpy()
    probs = torch.full((B, 1, V), 1e-6) if given else None
    q = np.ones(B)
    if given:
        q = (pd * (1.05 + 0.9 * torch.rand(B, generator=g).numpy())).astype(np.float32).astype(np.float64)
        probs[torch.arange(B), 0, drafts[:, 0].long()] = torch.from_numpy(q).float()
    u0 = (pd / q).astype(np.float32)
    want = np.arange(B) % 2 == 0
    for b in range(B):
        while not (u0[b] * q[b] < pd[b] * (1 - 1e-11) if want[b] else u0[b] * q[b] > pd[b] * (1 + 1e-11)):
            u0[b] = np.nextafter(u0[b], np.float32(0 if want[b] else 2))
    assert (np.abs(u0 * q - pd) < 4e-7 * pd).all() and (u0 < 1).all()
    u = torch.stack((torch.from_numpy(u0), torch.rand(B, generator=g)), 1)
    args = (x.to(DEV), drafts.to(DEV), u.to(DEV), probs.to(DEV) if given else None)
    tokens, n = sparda.verify_drafts(*args, temperature=temperature)
    assert n.cpu().tolist() == want.astype(int).tolist()
    t1, n1 = alone(*args, temperature)
    assert torch.equal(n, n1) and torch.equal(tokens, t1)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("near", [1e-6, 1e-4, 1e-2])
def test_residual_of_a_draft_that_is_nearly_the_target(dtype, near):
    """q = p (1 + near N(0,1)): max(p - q, 0) is a sum of differences that p's total in fp32 would hide. u is the middle of
    one token's part of the sum (of 1e-4 of it at least; float64 has it to 1e-14 / near)."""
    print(f"[case] verify residual {dtype} {near}", flush=True)
    g, x, p = case(dtype, 1.0, seed=5)
    probs = (p[:, :1] * (1 + near * torch.randn(B, 1, V, generator=g).double())).clamp(min=0).float()
    r = (p[:, 0] - probs[:, 0].double()).clamp(min=0)
    total, upto = r.sum(-1), r.cumsum(-1)
    want = torch.stack([(r[b] > 1e-4 * total[b]).nonzero()[:, 0][torch.randint(0, 30, (1,), generator=g)][0] for b in range(B)])
    over = (probs[:, 0].double() / p[:, 0] - 1).masked_fill(p[:, 0] < 1e-5, 0)
    drafts = over.argmax(-1, keepdim=True).int()          # far enough above p that u = 1 - 2^-24 rejects it
    assert (over.max(-1).values > 4e-7).all()
    mid = ((upto.gather(1, want[:, None]) - 0.5 * r.gather(1, want[:, None])) / total[:, None])[:, 0]
    u = torch.stack((torch.full((B,), 1 - 2.0 ** -24), mid.float()), 1)
    args = (x.to(DEV), drafts.to(DEV), u.to(DEV), probs.to(DEV))
    tokens, n = sparda.verify_drafts(*args)
    assert (n == 0).all() and tokens[:, 0].cpu().tolist() == want.tolist()
    t1, n1 = alone(*args, 1.0)
    assert torch.equal(n, n1) and torch.equal(tokens, t1)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("given", [True, False], ids=["probs", "tokens"])
def test_several_drafts_next_to_their_borders(dtype, given):
    """Up to three drafts in a row that fp32 leaves open, each number of accepted ones, and rows without a distribution behind
    them: float64's acceptances, and the tokens that a call of the sequence alone gives (whose sums are float64's)."""
    print(f"[case] verify several borders {dtype} {given}", flush=True)
    b_, K = 12, 3
    g = torch.Generator().manual_seed(23)
    x = (torch.randn(b_, K + 1, V, generator=g) * 3).to(dtype)
    want = [b % (K + 1) for b in range(b_)]
    for b in range(8, 12):
        x[b, want[b], 11] = float("nan")
    p = torch.softmax(x.double(), -1).nan_to_num(0.5)
    drafts = p[:, :K].topk(40, -1).indices.gather(-1, torch.randint(0, 40, (b_, K, 1), generator=g))[..., 0]
    pd = p[:, :K].gather(-1, drafts[..., None])[..., 0].numpy()
    probs = (p[:, :K] * (1 + 0.2 * torch.rand(b_, K, V, generator=g).double())).float() if given else None
    q = np.ones((b_, K))
    if given:
        q = (pd * 1.3).astype(np.float32).astype(np.float64)
        probs.scatter_(-1, drafts[..., None], torch.from_numpy(q).float()[..., None])
    u = (pd / q).astype(np.float32)
    for b in range(b_):
        for i in range(K):
            yes = i < want[b]
            while not (u[b, i] * q[b, i] < pd[b, i] * (1 - 1e-11) if yes else u[b, i] * q[b, i] > pd[b, i] * (1 + 1e-11)):
                u[b, i] = np.nextafter(u[b, i], np.float32(0 if yes else 2))
    u = torch.cat((torch.from_numpy(u), torch.rand(b_, 1, generator=g)), 1)
    args = [x.to(DEV), drafts.int().to(DEV), u.to(DEV), probs.to(DEV) if given else None]
    tokens, n = sparda.verify_drafts(*args)
    assert n.cpu().tolist() == want
    assert (tokens.cpu()[8:].gather(1, torch.tensor(want[8:])[:, None]) == -1).all()
    one = [sparda.verify_drafts(*(a[b:b + 1] if a is not None else None for a in args)) for b in range(b_)]
    assert torch.equal(n, torch.cat([m for _, m in one])) and torch.equal(tokens, torch.cat([t for t, _ in one]))
