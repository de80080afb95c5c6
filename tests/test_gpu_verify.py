"""Verification of drafted tokens (sparda.verify_drafts) against a loop in float64: tokens and
counts are equal. The row that a token is drawn from is summed in fp64 on both sides; a test of
a draft is off by 1e-6 of p at most, and the random numbers here come no nearer to it."""

import numpy as np
import pytest
import torch

import sparda

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def oracle(logits, drafts, uniform, probs=None, counts=None, temperature=1.0):
    """The definition, sequence by sequence; all on the CPU."""
    x = logits.double().numpy()
    B, K1, V = x.shape
    tokens, accepted = np.full((B, K1), -1, np.int32), np.zeros(B, np.int32)
    u = uniform.double().numpy()
    for b in range(B):
        T = float(temperature[b]) if isinstance(temperature, torch.Tensor) else temperature
        count = min(max(int(counts[b]), 0), K1 - 1) if counts is not None else K1 - 1
        n, token = 0, None
        while token is None:
            row = x[b, n]
            if not np.isfinite(row.max()):                    # nothing, or NaN or +inf among it
                token = -1
                break
            best = int(np.argmax(row))
            p = np.exp((row - row.max()) / T) if T > 0 else None
            if p is not None:
                p /= p.sum()
            r = p
            if n < count:
                d = int(drafts[b, n])
                q = probs[b, n].double().numpy() if probs is not None else None
                if T > 0:
                    inside = 0 <= d < V
                    if inside:
                        lhs, rhs = u[b, n] * (q[d] if q is not None else 1.0), p[d]
                        assert abs(lhs - rhs) > 1e-6 * rhs or lhs == rhs, "a test too near its border to compare"
                    if inside and lhs < rhs:
                        tokens[b, n] = d
                        n += 1
                        continue
                    if q is not None:
                        r = np.maximum(p - q, 0.0)
                    elif inside:
                        r = p.copy()
                        r[d] = 0.0
                    if r.sum() == 0:
                        r = p
                elif d == best:
                    tokens[b, n] = d
                    n += 1
                    continue
            if T > 0:
                c = np.cumsum(r)
                at = np.nonzero(c > u[b, K1 - 1] * c[-1])[0]
                token = int(at[0]) if at.size else int(np.nonzero(r)[0][-1])
            else:
                token = best
        tokens[b, n], accepted[b] = token, n
    return torch.from_numpy(tokens), torch.from_numpy(accepted)


def inputs(B, K, V, dtype, sampled, seed, temperature=0.8, near=0.6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K + 1, V, generator=g) * 3
    logits = x.to(dtype)
    q = torch.softmax((x[:, :K] + torch.randn(B, K, V, generator=g) * near) / temperature, -1)
    drafts = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, K).int() if K else torch.zeros(B, 0, dtype=torch.int32)
    return logits, drafts, torch.rand(B, K + 1, generator=g), q if sampled else None


def same(args, kw=None):
    kw = kw or {}
    want = oracle(*args, **{{"draft_probs": "probs", "n_drafts": "counts"}.get(k, k): v for k, v in kw.items()})
    on = lambda t: t.to(DEV) if isinstance(t, torch.Tensor) else t
    got = sparda.verify_drafts(*(on(a) for a in args), **{k: on(v) for k, v in kw.items()})
    assert torch.equal(got[1].cpu(), want[1]), (got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0]), (got[0].cpu(), want[0])
    return want


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("sampled", [False, True], ids=["given", "sampled"])
@pytest.mark.parametrize("B,K,V", [(1, 4, 32000), (5, 1, 1), (7, 3, 2), (3, 2, 7), (4, 8, 1000), (2, 5, 50257), (33, 0, 2049),
                                   (3, 64, 300), (1, 0, 131072), (2, 1, 2047), (40, 3, 2048)])
def test_tokens_and_counts(B, K, V, dtype, sampled):
    print(f"[case] verify {B}x{K} of {V} {dtype} sampled={sampled}", flush=True)
    logits, drafts, uniform, q = inputs(B, K, V, dtype, sampled, seed=B + K + V)
    same((logits, drafts, uniform), dict(draft_probs=q, temperature=0.8))
    counts = torch.randint(-1, K + 3, (B,), generator=torch.Generator().manual_seed(1)).int()
    each = torch.tensor([0.8, 0.0, 1.3, 0.25])[torch.arange(B) % 4]
    same((logits, drafts, uniform), dict(draft_probs=q, n_drafts=counts, temperature=each))
    same((logits, drafts, uniform), dict(draft_probs=q, temperature=0.0))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("sampled", [False, True], ids=["given", "sampled"])
@pytest.mark.parametrize("B,K,V", [(11, 4, 50257), (70, 1, 15001), (5, 0, 524289), (2, 1, 1048568)])
def test_calls_of_more_than_two_million_logits(B, K, V, dtype, sampled):
    """The statistics are in fp32 there, the drawn row's sums still in fp64."""
    print(f"[case] verify {B}x{K} of {V} {dtype} sampled={sampled}", flush=True)
    logits, drafts, uniform, q = inputs(B, K, V, dtype, sampled, seed=B + K)
    each = torch.tensor([0.8, 1.3, 0.0, 0.25])[torch.arange(B) % 4]
    same((logits, drafts, uniform), dict(draft_probs=q, temperature=each))


@pytest.mark.parametrize("sampled", [False, True], ids=["given", "sampled"])
def test_masks_in_calls_of_more_than_two_million_logits(sampled):
    print(f"[case] verify masks, many logits, sampled={sampled}", flush=True)
    inf, B, K, V = float("inf"), 12, 3, 50003
    logits, drafts, uniform, q = inputs(B, K, V, F32, sampled, seed=6)
    logits[0, :, 100:] = -inf
    logits[1, 0] = -inf
    logits[2, 0, 7] = float("nan")
    logits[3, 1, V - 1] = inf
    logits[4, 0] = torch.finfo(F32).min
    drafts[6, 0], drafts[7, 0] = V, -1
    logits[8, :, drafts[8, 0]] = 80.0                             # all of p on one token, and drafts beside it
    drafts[9, 0] = (int(logits[9, 0].argmin()))
    uniform[9, 0] = 0.5
    tokens, n = same((logits, drafts, uniform), dict(draft_probs=q))
    assert tokens[1, 0] == -1 and tokens[2, 0] == -1 and n[6] == 0 and n[7] == 0
    same((logits, drafts, uniform), dict(draft_probs=q, temperature=1e-30))


def test_every_count_of_accepted_drafts():
    """Drafts that are accepted up to a place and not there, each place of a row of 70 sequences."""
    print("[case] verify every place", flush=True)
    K, V = 6, 4001
    logits, drafts, uniform, _ = inputs(K + 1, K, V, BF, False, seed=3)
    logits[:, :, :] -= 20
    for b in range(K + 1):
        for i in range(K):
            logits[b, i, drafts[b, i]] = 20.0 if i != b else -60.0
    for q in (None, torch.softmax(torch.randn(K + 1, K, V, generator=torch.Generator().manual_seed(2)), -1)):
        _, n = same((logits, drafts, uniform), dict(draft_probs=q))
        assert n.tolist() == list(range(K + 1))


def test_the_drawn_token_is_where_the_sum_passes():
    """Rows of few, equal and ordered weights: every token is drawn by the numbers that belong to it, the
    ends of the range and the last token with a weight among them."""
    print("[case] verify draws", flush=True)
    V, n = 5003, 64
    heavy = torch.randperm(V, generator=torch.Generator().manual_seed(1))[:n].sort().values
    logits = torch.full((4 * n, 1, V), -float("inf"))
    logits[:, 0, heavy] = 0.0                                     # 64 tokens of 1/64 each: sums without rounding
    u = (torch.arange(4 * n) % n + torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -18]).repeat_interleave(n)) / n
    tokens, _ = same((logits, torch.zeros(4 * n, 0, dtype=torch.int32), u[:, None]))
    assert torch.equal(tokens[:, 0], heavy[torch.arange(4 * n) % n].int())
    top = torch.tensor([1.0, 1 - 2.0 ** -24, 0.0, 2.0 ** -126, float("nan")])
    tokens = sparda.verify_drafts(logits[:5].to(DEV), torch.zeros(5, 0, dtype=torch.int32, device=DEV), top[:, None].to(DEV))[0]
    assert tokens[:, 0].tolist() == [heavy[-1], heavy[-1], heavy[0], heavy[0], heavy[-1]]


def test_equal_logits_and_borders():
    print("[case] verify ties", flush=True)
    V = 4
    logits = torch.zeros(8, 2, V)
    drafts = torch.tensor([[0], [1], [2], [3], [0], [1], [2], [3]]).int()
    uniform = torch.tensor([[0.25, 0.5], [0.2499, 0.5], [0.0, 0.75], [0.25, 0.0], [0.5, 0.99], [0.75, 1 / 3], [0.2, 0.2], [0.9, 0.7]])
    same((logits, drafts, uniform))                               # u q < p: 0.25 is not below 0.25
    same((logits, drafts, uniform), dict(temperature=0.0))        # the lowest index wins
    q = torch.full((8, 1, V), 0.25)
    tokens, n = same((logits, drafts, uniform), dict(draft_probs=q))   # p = q: accepted by every u below 1
    assert n.tolist() == [1] * 8
    q = torch.zeros(8, 1, V)
    q[:, 0, 0] = 1.0
    same((logits, drafts, uniform), dict(draft_probs=q))


def test_masked_rows_and_rows_without_a_distribution():
    print("[case] verify masks", flush=True)
    inf, V, K = float("inf"), 3000, 3
    logits, drafts, uniform, q = inputs(9, K, V, F32, True, seed=5)
    logits[0, 0, 100:] = -inf                                     # a filter
    drafts[0, 0] = 2500                                           # a draft that it leaves out
    logits[1, 1] = -inf                                           # nothing left
    logits[2, 0, 7] = float("nan")
    logits[3, 2, 2999] = inf
    logits[4, 3] = -inf
    logits[5, 0] = torch.finfo(F32).min                           # masked with the type's lowest value: all equal
    drafts[6, 0], drafts[7, 1], drafts[8, 2] = V, -1, 2 ** 31 - 1
    logits[7, 0, drafts[7, 0]] = 60.0
    for kw in (dict(draft_probs=q), dict(), dict(temperature=0.0), dict(draft_probs=q, temperature=1e-3),
               dict(temperature=torch.tensor([1e-30, 1e30, 1.0] * 3))):
        tokens, n = same((logits, drafts, uniform), kw)
        assert tokens[2, 0] == -1 and n[2] == 0 and n[6] == 0


def test_a_rejection_that_leaves_nothing_draws_from_p():
    print("[case] verify p below q everywhere", flush=True)
    V = 1000
    logits = torch.randn(3, 2, V, generator=torch.Generator().manual_seed(1))
    q = torch.ones(3, 1, V)                                       # (no distribution, but max(p - q, 0) is zero)
    drafts, uniform = torch.tensor([[5], [6], [7]]).int(), torch.tensor([[0.99, 0.3], [0.98, 0.0], [0.97, 0.9]])
    same((logits, drafts, uniform), dict(draft_probs=q))
    logits = torch.full((1, 2, V), -float("inf"))
    logits[0, :, 9] = 1.0                                         # all of p on the draft, u = 1: rejected, nothing else
    tokens = sparda.verify_drafts(logits.to(DEV), torch.tensor([[9]], dtype=torch.int32, device=DEV), torch.ones(1, 2, device=DEV))
    assert tokens[0].tolist() == [[9, -1]] and tokens[1].tolist() == [0]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_strides_and_odd_rows(dtype):
    print(f"[case] verify strides {dtype}", flush=True)
    B, K, V = 5, 3, 1237
    logits, drafts, uniform, q = inputs(B, K, V, dtype, True, seed=9)
    want = oracle(logits, drafts, uniform, q)
    wide = torch.full((K + 1, B, V + 5), 1e9, dtype=dtype, device=DEV)       # rows before sequences, other values beside them
    wide[:, :, 3:V + 3] = logits.to(DEV).transpose(0, 1)
    qw = torch.full((B, K + 2, V + 1), 5.0, device=DEV)
    qw[:, 1:K + 1, 1:] = q.to(DEV)
    dw = torch.zeros(B, 9, dtype=torch.int32, device=DEV)
    dw[:, 2:2 + K] = drafts.to(DEV)
    uw = torch.zeros(B, 7, device=DEV)
    uw[:, 1:K + 2] = uniform.to(DEV)
    got = sparda.verify_drafts(wide[:, :, 3:V + 3].transpose(0, 1), dw[:, 2:2 + K], uw[:, 1:K + 2], draft_probs=qw[:, 1:K + 1, 1:])
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    # every dimension strided: copies
    got = sparda.verify_drafts(logits.to(DEV).transpose(1, 2).contiguous().transpose(1, 2), drafts.to(DEV).t().contiguous().t(),
                               uniform.to(DEV).t().contiguous().t(), draft_probs=q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_drawn_tokens_follow_the_distribution():
    """Accepted and redrawn tokens together are distributed as p: 20000 draws, every cell within six
    standard deviations (a false alarm in 32 cells has a probability of 6e-8)."""
    print("[case] verify distribution", flush=True)
    g = torch.Generator().manual_seed(11)
    V, B = 32, 20000
    x, y = torch.randn(V, generator=g) * 1.5, torch.randn(V, generator=g) * 1.5
    p, q = torch.softmax(x, 0), torch.softmax(y, 0)
    drafts = torch.multinomial(q, B, replacement=True, generator=g).int()[:, None]
    tokens, n = sparda.verify_drafts(x.to(DEV).expand(B, 2, V).contiguous(), drafts.to(DEV), torch.rand(B, 2, generator=g).to(DEV),
                                     draft_probs=q.to(DEV).expand(B, 1, V).contiguous())
    seen = torch.bincount(tokens[:, 0].cpu().long(), minlength=V).double()
    assert ((seen - B * p).abs() <= 6 * (B * p * (1 - p)).sqrt() + 1).all()
    rate = float(torch.minimum(p, q).sum())
    assert abs(n.double().mean().item() - rate) <= 6 * (rate * (1 - rate) / B) ** 0.5


def test_captured_and_replayed():
    print("[case] verify captured", flush=True)
    B, K, V = 6, 4, 5000
    sets = [inputs(B, K, V, BF, True, seed=s) for s in range(4)]
    bufs = [t.to(DEV) for t in sets[0]]
    each = torch.tensor([0.8, 0.0, 1.0] * 2, device=DEV)
    call = lambda: sparda.verify_drafts(bufs[0], bufs[1], bufs[2], draft_probs=bufs[3], temperature=each)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for s in (1, 2, 3, 1):
        for b, t in zip(bufs, sets[s]):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = oracle(*sets[s], temperature=each.cpu())
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("B,V", [(4, 700), (60, 50257)])
def test_an_infinite_temperature_and_numbers_below_zero(B, V):
    """All tokens with a logit are alike at a temperature of +inf, one with -inf keeps its weight of zero; a number
    below zero draws as zero does."""
    print(f"[case] verify infinite temperature {B} of {V}", flush=True)
    logits, drafts, uniform, q = inputs(B, 1, V, F32, True, seed=12)
    logits[:, :, ::3] = -float("inf")
    drafts[1, 0] = 3
    call = lambda T, u: [t.cpu() for t in sparda.verify_drafts(logits.to(DEV), drafts.to(DEV), u.to(DEV), draft_probs=q.to(DEV),
                                                               temperature=torch.full((B,), T, device=DEV))]
    want = oracle(logits, drafts, uniform, q, temperature=3.4e38)
    got = call(float("inf"), uniform)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (got[0][:, 0] >= 0).all()
    uniform[:, 1] = 0.0
    want = call(0.9, uniform)
    uniform[:, 1] = -0.5
    assert all(torch.equal(a, b) for a, b in zip(call(0.9, uniform), want))


def test_refusals():
    print("[case] verify refusals", flush=True)
    logits, drafts, uniform, q = (t.to(DEV) for t in inputs(3, 2, 100, BF, True, seed=1))
    good = dict(logits=logits, drafts=drafts, uniform=uniform, draft_probs=q)
    sparda.verify_drafts(**good)
    for bad, err in ((dict(logits=logits.half()), TypeError), (dict(logits=logits[0]), ValueError), (dict(logits=logits[:, :2]), ValueError),
                     (dict(drafts=drafts.long()), TypeError), (dict(drafts=drafts[:2]), ValueError), (dict(uniform=uniform.double()), TypeError),
                     (dict(uniform=uniform[:, :2]), ValueError), (dict(draft_probs=q.to(BF)), TypeError), (dict(draft_probs=q[..., :99]), ValueError),
                     (dict(n_drafts=drafts[:, 0].long()), TypeError), (dict(n_drafts=drafts[:2, 0]), ValueError), (dict(temperature=-1.0), ValueError),
                     (dict(temperature=float("nan")), ValueError), (dict(temperature=torch.ones(2, device=DEV)), ValueError),
                     (dict(temperature=torch.ones(3)), RuntimeError), (dict(uniform=uniform.cpu()), RuntimeError),
                     (dict(logits=logits.clone().requires_grad_()), RuntimeError)):
        with pytest.raises(err):
            sparda.verify_drafts(**{**good, **bad})
