"""Generation with a draft model where attention is sparse and past the context length: every row that a draft
is judged by is the row that the target gives for the tokens before it alone."""

import pytest
import torch

import sparda
from model.config import ModelConfig
from model.model import SparDAResearchModel

pytestmark = pytest.mark.gpu
DEV = "cuda"
CONTEXT, BLOCK, TOP_K = 64, 16, 2
# fp32 forwards of other lengths: sums of at most 512 products in another order, 512 2^-24 = 3e-5 of them at
# most, through three layers of gains near one; logits of about 1.6
ROW_TOL = 1e-3


def models(backend="hip_sparse"):
    # weights of a gain above one, so that which blocks a row sees moves its logits
    base = dict(vocab_size=500, n_embd=256, n_head=8, n_kv_head=2, head_dim=32, ffn_dim=512, forecast_heads=2, forecast_dim=32,
                context_length=CONTEXT, block_size=BLOCK, top_k_blocks=TOP_K, attention_backend=backend, initializer_range=0.1)
    torch.manual_seed(11)
    return SparDAResearchModel(ModelConfig(n_layer=3, **base)).to(DEV), SparDAResearchModel(ModelConfig(n_layer=1, **base)).to(DEV)


class Steps:
    """What every step of drafted generation scored: the logits, the drafts, how many were taken."""

    def __init__(self, monkeypatch):
        self.all, verify = [], sparda.verify_drafts

        def spy(logits, drafts, *a, **kw):
            tokens, n = verify(logits, drafts, *a, **kw)
            self.all.append((logits.clone(), drafts.clone(), int(n)))
            return tokens, n
        monkeypatch.setattr(sparda, "verify_drafts", spy)


@torch.no_grad()
@pytest.mark.parametrize("backend", ["hip_sparse", "static", "dense", "offload"])
def test_scored_rows_are_those_of_separate_forwards(monkeypatch, backend):
    print(f"[case] drafted rows {backend}", flush=True)
    target, draft = models(backend)
    steps = Steps(monkeypatch)
    prompt = torch.randint(0, 500, (1, 20), device=DEV)
    out = target.generate(prompt, max_new_tokens=56, temperature=1.0, top_k=0, draft_model=draft, num_drafts=5)
    n, most = 20, {}
    for x, drafts, taken in steps.all:
        K = drafts.shape[1]
        most[n] = K
        for i in range(K + 1):
            ids = torch.cat((out[:, :n], drafts[:, :i].long()), 1)[:, -CONTEXT:]
            want = target(ids)["logits"][0, -1]
            assert (x[0, i] - want).abs().max() <= ROW_TOL, (n, i, K)
        n += taken + 1
    assert n == out.shape[1] == 76
    limit = BLOCK * TOP_K if backend == "hip_sparse" else CONTEXT
    assert all(K == 0 if n >= limit else K == min(5, limit - n) for n, K in most.items())   # (and drafts are made up to there)


@torch.no_grad()
@pytest.mark.parametrize("backend", ["hip_sparse", "static", "offload"])
@pytest.mark.parametrize("prompt_len", [4, 30, 40, 70])
def test_greedy_drafted_generation_equals_plain(backend, prompt_len):
    print(f"[case] drafted greedy {backend} {prompt_len}", flush=True)
    target, draft = models(backend)
    prompt = torch.randint(0, 500, (1, prompt_len), device=DEV)
    plain = target.generate(prompt, max_new_tokens=40, temperature=0.0)
    for d in (draft, target):
        out = target.generate(prompt, max_new_tokens=40, temperature=0.0, draft_model=d, num_drafts=4)
        assert out.shape == plain.shape
        other = (out != plain).nonzero()
        if len(other):                # only where rounding decides between two logits
            at = int(other[0, 1])
            x = target(plain[:, :at][:, -CONTEXT:])["logits"][0, -1].topk(2).values
            assert x[0] - x[1] <= 2 * ROW_TOL, at


def spoil(model, at, value):
    """The model's logits are spoiled at the rows that see as many tokens as `at` holds."""
    forward = model.forward

    def spoiled(ids, **kw):
        out = forward(ids, **kw)
        x = out["logits"].clone()
        for n in at:
            if n <= ids.shape[1]:
                x[:, n - 1] = value(x[:, n - 1])
        return {**out, "logits": x}
    model.forward = spoiled


SPOIL = {"nan": lambda x: x.index_fill(1, torch.tensor([7, 300], device=x.device), float("nan")),
         "inf": lambda x: x.index_fill(1, torch.tensor([7], device=x.device), float("inf")),
         "none": lambda x: torch.full_like(x, -float("inf"))}


@torch.no_grad()
@pytest.mark.parametrize("how", list(SPOIL))
@pytest.mark.parametrize("of", ["target", "draft", "both"])
def test_rows_without_a_distribution(how, of):
    """Greedy: the tokens of plain generation. Sampled: an error where the target has no distribution, and the
    target's tokens where the draft model has none. Never a token of -1."""
    print(f"[case] drafted spoiled rows {how} {of}", flush=True)
    target, draft = models("dense")
    prompt = torch.randint(0, 500, (1, 9), device=DEV)
    for m, name in ((target, "target"), (draft, "draft")):
        if of in (name, "both"):
            spoil(m, {9, 12, 13, 20}, SPOIL[how])
    plain = target.generate(prompt, max_new_tokens=20, temperature=0.0)
    out = target.generate(prompt, max_new_tokens=20, temperature=0.0, draft_model=draft, num_drafts=3)
    assert torch.equal(out, plain)
    run = lambda: target.generate(prompt, max_new_tokens=20, temperature=1.0, top_k=0, draft_model=draft, num_drafts=3)
    if of == "draft":
        out = run()
        assert out.shape == (1, 29) and 0 <= int(out.min()) and int(out.max()) < 500
    else:
        with pytest.raises(RuntimeError, match="no distribution"):
            run()
