"""The rotated write, the 4-bit pages and the verification of drafts together: as a server runs them step by step,
captured into graphs, on side streams, and through the native host path and the Python one alike."""

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import sparda
from model.config import ModelConfig
from model.model import SparDAResearchModel
from model.rope import rope_tables
from q4_oracle import bf16, codes, turn, values
from sparda import _lib, ops
from test_gpu_host_path import Spy, _flat
from test_gpu_q4 import check
from test_gpu_rotate import dev, randn
from test_gpu_verify import oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _calls(dtype):
    Hq, Hkv, D, B, T = 6, 2, 64, 3, 4
    cos, sin = (dev(x) for x in rope_tables(D, 64))
    table, pos, cu = dev([[0, 1], [2, 3], [4, 5]]), dev([3, 0, 17]), dev([0, 5, 5, 9])
    q, k, v = (randn(9, h, D, dtype=dtype, seed=h + i).to(DEV) for i, h in enumerate((Hq, Hkv, Hkv)))
    wide = randn(9, Hq + 2 * Hkv, D, dtype=dtype, seed=4).to(DEV)
    kp, vp = (torch.zeros(6, 16, Hkv, D, dtype=dtype, device=DEV) for _ in range(2))
    pages = torch.zeros(sparda.q4_page_shape(6, 16, Hkv, D), dtype=torch.uint8, device=DEV)
    sparda.append_paged_q4(pages, table, dev([0, 0, 0]), randn(60, Hkv, D, dtype=dtype, seed=8).to(DEV),
                           randn(60, Hkv, D, dtype=dtype, seed=9).to(DEV), dev([0, 20, 40, 60]))
    qs = randn(B, T, Hq, D, dtype=dtype, seed=5).to(DEV)
    g = torch.Generator().manual_seed(6)
    logits = (torch.randn(B, T, 999, generator=g) * 3).to(dtype).to(DEV)
    probs = torch.softmax(torch.randn(B, T - 1, 999, generator=g) * 3, -1).to(DEV)
    drafts = torch.multinomial(probs.view(-1, 999).cpu(), 1, generator=g).view(B, T - 1).int().to(DEV)
    u = torch.rand(B, T, generator=g).to(DEV)
    return {
        "rotate_append_paged": lambda: (sparda.rotate_append_paged(kp, vp, table, pos, q, k, v, cos, sin, cu), kp.clone(), vp.clone(),
                                        sparda.rotate_append_paged(kp, vp, table, pos, wide[:3, :Hq], wide[:3, Hq:Hq + Hkv],
                                                                   wide[:3, Hq + Hkv:], cos, sin), kp.clone(), vp.clone()),
        "append_paged_q4": lambda: (sparda.append_paged_q4(pages, table, pos, k, v, cu), pages.clone(),
                                    sparda.append_paged_q4(pages, table, pos, k, v, cu, q, cos, sin), pages.clone(),
                                    sparda.append_paged_q4(pages, table, pos, k[:3], v[:3], q=q[:3], cos=cos, sin=sin), pages.clone()),
        "gather_paged_q4": lambda: (sparda.gather_paged_q4(pages, table, dev([0, 2, 4]), 3),
                                    sparda.gather_paged_q4(pages, table, dev([0, 1, 0]), 9, cu, dtype=torch.float32),
                                    sparda.gather_paged_q4(pages, table, dev([0, 1, 0]), 9, cu, head_dim=64)),
        "decode_paged_q4": lambda: (sparda.decode_paged_q4(qs, pages, table, dev([20, 19, 4])),
                                    sparda.decode_paged_q4(qs[:, 0], pages, table, dev([20, 0, 4]), 0.3),
                                    sparda.decode_paged_q4(qs.transpose(1, 2).contiguous().transpose(1, 2), pages, table, dev([20, 19, 4]), 1)),
        "verify_drafts": lambda: (sparda.verify_drafts(logits, drafts, u), sparda.verify_drafts(logits, drafts, u, probs, dev([3, 0, 1])),
                                  sparda.verify_drafts(logits, drafts, u, probs, None, 0),
                                  sparda.verify_drafts(logits, drafts, u, probs, None, torch.tensor([1.0, 0.0, 0.5], device=DEV)),
                                  sparda.verify_drafts(logits[:, :1], drafts[:, :0], u[:, :1], temperature=0.7)),
    }


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", ["rotate_append_paged", "append_paged_q4", "gather_paged_q4", "decode_paged_q4", "verify_drafts"])
def test_native_path_equals_the_python_path(monkeypatch, name, dtype):
    print(f"[case] serving host path {name} {dtype}", flush=True)
    spy = Spy()
    monkeypatch.setattr(ops, "_host", spy)
    got = _flat(_calls(dtype)[name]())
    monkeypatch.setattr(ops, "_host", _lib._NoHost())
    want = _flat(_calls(dtype)[name]())
    assert len(got) == len(want) and all(a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b) for a, b in zip(got, want))
    assert name in spy.taken, "the native path answered none of the calls"


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (8, 1, 128)])
def test_a_server_decodes_drafted_tokens(dtype, Hq, Hkv, D):
    """Prompts into 4-bit pages; then steps of T = 3 tokens a sequence (the last one and two drafts): rotated and
    appended, attended to, verified; what was rejected is overwritten by the next step. Every output against
    the sequence's own history."""
    print(f"[case] drafted server {dtype} {Hq}/{Hkv}x{D}", flush=True)
    g = torch.Generator().manual_seed(20)
    B, T, ps, width, V = 3, 3, 16, 9, 700
    cos, sin = rope_tables(D, ps * width)
    cd, sd = dev(cos), dev(sin)
    table = torch.randperm(B * width + 4, generator=g)[:B * width].view(B, width).int()
    pages = torch.full(sparda.q4_page_shape(B * width + 4, ps, Hkv, D), 0xFF, dtype=torch.uint8, device=DEV)
    td, lens, hist = dev(table), [40, 1, 17], [None] * B

    def rows(n, h):
        return torch.randn(n, h, D, generator=g).to(dtype)

    def held(b, k, v, at):
        """Rows k, v of sequence b from position `at` on, as its pages hold them; what lay there is gone."""
        pos = list(range(at, at + k.shape[0]))
        (ck, hk), (cv, hv) = codes(turn(k, cos, sin, pos).numpy()), codes(v.float().numpy())
        new = (values(ck, hk), values(cv, hv), hk, hv)
        hist[b] = new if at == 0 else tuple(np.concatenate((o[:at], n)) for o, n in zip(hist[b], new))

    N = sum(lens)
    cu = np.concatenate(([0], np.cumsum(lens))).tolist()
    q, k, v = rows(N, Hq), rows(N, Hkv), rows(N, Hkv)
    turned = sparda.append_paged_q4(pages, td, dev([0] * B), dev(k), dev(v), dev(cu), dev(q), cd, sd)
    pos = [p for n in lens for p in range(n)]
    assert torch.equal(turned.cpu(), turn(q, cos, sin, pos).to(dtype))
    for b in range(B):
        held(b, k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]], 0)
    # the prompt's own rows come back for a chunk that attends to them with prefill_packed
    kb, vb = sparda.gather_paged_q4(pages, td, dev([0] * B), N, dev(cu), dtype=F32)
    assert np.array_equal(kb.cpu().double().numpy(), np.concatenate([h[0] for h in hist]))
    assert np.array_equal(vb.cpu().double().numpy(), np.concatenate([h[1] for h in hist]))
    out = sparda.prefill_packed(turned.float(), kb, vb, dev(cu))
    one = sparda.decode_paged_q4(turned[[c - 1 for c in cu[1:]]], pages, td, dev(lens))
    last = out[[c - 1 for c in cu[1:]]]
    assert (one.float() - last).abs().max() <= (2e-2 if dtype == BF else 1e-4)

    taken = 0
    for step in range(8):
        q, k, v = rows(B * T, Hq), rows(B * T, Hkv), rows(B * T, Hkv)
        qt = sparda.append_paged_q4(pages, td, dev(lens), dev(k), dev(v), dev([0, T, 2 * T, 3 * T]), dev(q), cd, sd)
        for b in range(B):
            held(b, k[b * T:(b + 1) * T], v[b * T:(b + 1) * T], lens[b])
        out = sparda.decode_paged_q4(qt.view(B, T, Hq, D), pages, td, dev([n + T for n in lens]))
        check(out, qt.view(B, T, Hq, D).cpu(), [n + T for n in lens], hist)
        # the target's logits and a draft's distribution near them
        x = torch.randn(B, T, V, generator=g) * 3
        probs = torch.softmax(x[:, :T - 1] + torch.randn(B, T - 1, V, generator=g) * 0.4, -1)
        drafts = torch.multinomial(probs.view(-1, V), 1, generator=g).view(B, T - 1).int()
        u = torch.rand(B, T, generator=g)
        tokens, n = sparda.verify_drafts(dev(x), dev(drafts), dev(u), draft_probs=dev(probs))
        want = oracle(x, drafts, u, probs)
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(n.cpu(), want[1])
        for b in range(B):
            lens[b] += 1 + int(want[1][b])        # the last token and its accepted drafts stay
            hist[b] = tuple(h[:lens[b]] for h in hist[b])
        taken += int(want[1].sum())
    assert 0 < taken < 8 * B * (T - 1) and sparda.status() == 0


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_a_decode_step_captured_and_replayed(dtype):
    """Rotation, write, attention over several shares and verification in two graphs, replayed in turn as positions,
    tables, rows and random numbers change, with eager work and synchronizations between."""
    print(f"[case] serving graph {dtype}", flush=True)
    Hq, Hkv, D, ps, B, T, V = 6, 2, 64, 16, 3, 2, 3000
    width = 100
    cos, sin = (dev(x) for x in rope_tables(D, ps * width))
    g = torch.Generator().manual_seed(3)
    order = torch.randperm(B * width, generator=g).view(B, width).int()
    start = torch.randint(0, 256, sparda.q4_page_shape(B * width, ps, Hkv, D), generator=g, dtype=torch.uint8)
    start[..., 1024:] = torch.full((1,), 0.2).half().view(torch.uint8).repeat(64)    # finite numbers
    pages, kp, vp = dev(start), torch.zeros(B * width, ps, Hkv, D, dtype=dtype, device=DEV), torch.zeros(B * width, ps, Hkv, D, dtype=dtype, device=DEV)
    q, k, v = (torch.zeros(B * T, h, D, dtype=dtype, device=DEV) for h in (Hq, Hkv, Hkv))
    table, pos, cu = dev(order), dev([0] * B), dev([0, T, 2 * T, 3 * T])
    logits, u = torch.zeros(B, T, V, device=DEV), torch.zeros(B, T, device=DEV)
    drafts, probs = torch.zeros(B, T - 1, dtype=torch.int32, device=DEV), torch.zeros(B, T - 1, V, device=DEV)

    def step():
        a = sparda.rotate_append_paged(kp, vp, table, pos, q, k, v, cos, sin, cu)
        b = sparda.append_paged_q4(pages, table, pos, k, v, cu, q, cos, sin)
        c = sparda.gather_paged_q4(pages, table, pos, B * T, cu)
        d = sparda.decode_paged_q4(b.view(B, T, Hq, D), pages, table, pos + T)
        return [a, b, *c, d, *sparda.verify_drafts(logits, drafts, u, draft_probs=probs)]

    def feed(i):
        h = torch.Generator().manual_seed(100 + i)
        for x, y in ((q, Hq), (k, Hkv), (v, Hkv)):
            x.copy_(torch.randn(B * T, y, D, generator=h).to(dtype))
        pos.copy_(torch.tensor([[5, 1200, 0], [1590, 3, 700], [-1, 40, 1598], [5, 1201, 33]][i]))
        table.copy_(order.roll(i, 1))
        z = torch.randn(B, T, V, generator=h) * 3
        logits.copy_(z), u.copy_(torch.rand(B, T, generator=h))
        probs.copy_(torch.softmax(z[:, :T - 1] + torch.randn(B, T - 1, V, generator=h) * 0.4, -1))
        drafts.copy_(torch.multinomial(probs.view(-1, V).cpu(), 1, generator=h).view(B, T - 1))

    feed(0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    live = torch.tensor([0, 1, 2, 3, 4, 5])
    for i in (0, 1, 2, 3, 1, 0):
        feed(i)
        pages.copy_(start), kp.zero_(), vp.zero_()
        graphs[i % 2].replay()
        got = [x.clone() for x in outs[i % 2]] + [pages.clone(), kp.clone(), vp.clone()]
        torch.cuda.synchronize()
        pages.copy_(start), kp.zero_(), vp.zero_()
        want = step() + [pages, kp, vp]
        torch.cuda.synchronize()
        rows = live[T:] if i == 2 else live       # (the first sequence takes no part: its rows hold anything)
        for j, (a, b) in enumerate(zip(got, want)):
            if j < 4:
                a, b = a[rows], b[rows]
            elif j == 4 and i == 2:
                a, b = a[1:], b[1:]
            assert torch.equal(a, b), (i, j)
    sparda.status()


_FIRST_CALLS_CAPTURED = r"""
import sys
sys.path[:0] = sys.argv[1:3]
import torch
import sparda
t = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
q, k, v, cu = t(40, 6, 64), t(40, 2, 64), t(40, 2, 64), i(0, 25, 40)
cos, sin = torch.rand(64, 32, device="cuda"), torch.rand(64, 32, device="cuda")
kp, vp, table, zero, n = t(8, 16, 2, 64), t(8, 16, 2, 64), i(3, 1, 5, 2).view(2, 2), i(0, 0), i(25, 15)
pages = torch.zeros(sparda.q4_page_shape(8, 16, 2, 64), dtype=torch.uint8, device="cuda")
logits, drafts, u = t(2, 3, 5000), i(1, 2, 3, 4).view(2, 2), torch.rand(2, 3, device="cuda")
torch.cuda.synchronize()

def step():
    a = sparda.rotate_append_paged(kp, vp, table, zero, q, k, v, cos, sin, cu)
    b = sparda.append_paged_q4(pages, table, zero, k, v, cu, q, cos, sin)
    return [a, b, sparda.decode_paged_q4(b[:2], pages, table, n), *sparda.verify_drafts(logits, drafts, u)]

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
for _ in range(3):
    for x in got:
        x.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, step()))
assert sparda.status() == 0
print("CAPTURED", flush=True)
"""


def test_first_calls_of_a_process_can_be_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "local-research-small-language-model_amd")
    print("[case] first serving calls in a capture, fresh process", flush=True)
    r = subprocess.run([sys.executable, "-c", _FIRST_CALLS_CAPTURED, root, pkg], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "CAPTURED" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_two_streams_at_once():
    """Steps of different sizes in flight on two streams, each with workspaces of its own: every result as alone."""
    print("[case] serving on two streams", flush=True)
    def make(seed, B, n, V):
        Hq, Hkv, D, ps = 12, 4, 64, 16
        width = n // ps + 1
        cos, sin = (dev(x) for x in rope_tables(D, n + 16))
        table = torch.randperm(B * width, generator=torch.Generator().manual_seed(seed)).view(B, width).int().to(DEV)
        pages = torch.zeros(sparda.q4_page_shape(B * width, ps, Hkv, D), dtype=torch.uint8, device=DEV)
        q, k, v = (randn(B * n, h, D, dtype=BF, seed=seed + h).to(DEV) for h in (Hq, Hkv, Hkv))
        cu = dev(list(range(0, B * n + 1, n)))
        x, u = torch.randn(B, 5, V, device=DEV) * 3, torch.rand(B, 5, device=DEV)
        probs = torch.softmax(torch.randn(B, 4, V, device=DEV) * 3, -1)
        drafts = torch.multinomial(probs.view(-1, V), 1).view(B, 4).int()

        def run():
            qt = sparda.append_paged_q4(pages, table, dev([0] * B), k, v, cu, q, cos, sin)
            out = sparda.decode_paged_q4(qt[n - 1::n].contiguous(), pages, table, dev([n] * B))
            return [qt, out, *sparda.verify_drafts(x, drafts, u, draft_probs=probs)]
        return run

    a, b = make(1, 3, 3000, 20000), make(2, 17, 150, 3001)
    want = a(), b()
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for stream in (s, t):
        stream.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        with torch.cuda.stream(s):
            got.append((0, a()))
        with torch.cuda.stream(t):
            got.append((1, b()))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for i, r in got for x, y in zip(r, want[i]))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_writes_larger_than_the_caches(D, dtype):
    """A call that reads and writes more than 256 MB loads its rows otherwise: the same bits as four calls of a quarter,
    whose form the other tests compare with the formula."""
    Hq, Hkv, ps = 6, 2, 64
    N = ((128 << 20) // ((Hq + 2 * Hkv) * D * (2 if dtype == BF else 4)) // 4 + 1) * 4
    print(f"[case] large writes {dtype} D={D} {N} rows", flush=True)
    g = torch.Generator(device=DEV).manual_seed(D)
    q, k, v = (torch.randn(N, h, D, device=DEV, generator=g).to(dtype) for h in (Hq, Hkv, Hkv))
    width = N // ps + 1
    table = torch.randperm(width, device=DEV, generator=g).int().view(1, width)
    angles = torch.rand(N, D // 2, device=DEV, generator=g) * 6
    cos, sin = angles.cos(), angles.sin()
    def pages():
        return (torch.zeros(width, ps, Hkv, D, dtype=dtype, device=DEV), torch.zeros(width, ps, Hkv, D, dtype=dtype, device=DEV),
                *(torch.zeros(sparda.q4_page_shape(width, ps, Hkv, D), dtype=torch.uint8, device=DEV) for _ in range(2)))
    def write(p, a, b):
        cu = dev([0, b - a])
        pos = dev([a])
        x = sparda.rotate_append_paged(p[0], p[1], table, pos, q[a:b], k[a:b], v[a:b], cos, sin, cu)
        y = sparda.append_paged_q4(p[2], table, pos, k[a:b], v[a:b], cu, q[a:b], cos, sin)
        sparda.append_paged_q4(p[3], table, pos, k[a:b], v[a:b], cu)
        assert torch.equal(x, y)
        return x
    whole, parts = pages(), pages()
    out = write(whole, 0, N)
    assert torch.equal(out, torch.cat([write(parts, i * N // 4, (i + 1) * N // 4) for i in range(4)]))
    assert all(torch.equal(a, b) for a, b in zip(whole, parts)) and sparda.status() == 0


def test_refusals_of_ranks_and_gradients():
    print("[case] serving refusals", flush=True)
    cos, sin = (dev(x) for x in rope_tables(64, 40))
    pages, table, pos = torch.zeros(sparda.q4_page_shape(4, 16, 2, 64), dtype=torch.uint8, device=DEV), dev([[0, 1], [2, 3]]), dev([0, 0])
    kp, vp = (torch.zeros(4, 16, 2, 64, dtype=BF, device=DEV) for _ in range(2))
    q, k, v = (randn(2, h, 64, dtype=BF, seed=h).to(DEV) for h in (4, 2, 2))
    for bad in (k[0, 0, 0], k[0, 0], k[0], k[None]):
        with pytest.raises(ValueError):
            sparda.append_paged_q4(pages, table, pos, bad, bad)
        with pytest.raises(ValueError):
            sparda.rotate_append_paged(kp, vp, table, pos, q, bad, bad, cos, sin)
    for bad in (q[0, 0, 0], q[0, 0], q[0], q[None, None]):
        with pytest.raises(ValueError):
            sparda.decode_paged_q4(bad, pages, table, pos)
    learned = cos.clone().requires_grad_()
    for call in (lambda c: sparda.rotate_append_paged(kp, vp, table, pos, q, k, v, c, sin),
                 lambda c: sparda.rotate_append_paged(kp, vp, table, pos, q, k, v, cos, c),
                 lambda c: sparda.append_paged_q4(pages, table, pos, k, v, None, q, c, sin)):
        with pytest.raises(RuntimeError):
            call(learned)
        with torch.no_grad():
            assert call(learned).shape == q.shape


def _models(vocab=500):
    base = dict(vocab_size=vocab, n_embd=256, n_head=8, n_kv_head=2, head_dim=32, ffn_dim=512, forecast_heads=2,
                forecast_dim=32, context_length=64, block_size=16, top_k_blocks=8)
    torch.manual_seed(5)
    target = SparDAResearchModel(ModelConfig(n_layer=3, **base)).to(DEV)
    return target, SparDAResearchModel(ModelConfig(n_layer=1, **base)).to(DEV)


@pytest.mark.parametrize("temperature,top_k", [(0.8, 50), (1.0, 0), (0.0, 50)])
def test_drafted_generation_runs(temperature, top_k):
    print(f"[case] drafted generation T={temperature} top_k={top_k}", flush=True)
    target, draft = _models()
    prompt = torch.randint(0, 500, (1, 9), device=DEV)
    for n, drafts in ((1, 4), (17, 4), (30, 0), (75, 7)):       # the last past the context
        out = target.generate(prompt, max_new_tokens=n, temperature=temperature, top_k=top_k, draft_model=draft, num_drafts=drafts)
        assert out.shape == (1, 9 + n) and torch.equal(out[:, :9], prompt) and 0 <= int(out.min()) and int(out.max()) < 500


@torch.no_grad()
def test_drafted_generation_is_the_target_s_own():
    """Greedy: every token is the target's largest logit behind the tokens before it, whatever was drafted."""
    print("[case] drafted generation, greedy", flush=True)
    target, draft = _models()
    prompt = torch.randint(0, 500, (1, 12), device=DEV)
    plain = target.generate(prompt, max_new_tokens=24, temperature=0.0)
    for d in (draft, target):
        out = target.generate(prompt, max_new_tokens=24, temperature=0.0, draft_model=d, num_drafts=3)
        x = target(out)["logits"][0, 11:-1]
        picked = x.gather(1, out[0, 12:, None])[:, 0]
        assert (x.max(-1).values - picked <= 1e-4).all()         # (fp32 forwards of other lengths, logits of about 1)
        near = x.topk(2).values
        if ((near[:, 0] - near[:, 1]) > 1e-3).all():             # no tie for rounding to break
            assert torch.equal(out, plain)
    stop = int(plain[0, 15])
    cut = target.generate(prompt, max_new_tokens=24, temperature=0.0, eos_token_id=stop, draft_model=target, num_drafts=5)
    first = 12 + int((cut[0, 12:] == stop).nonzero()[0])
    assert cut.shape[1] == first + 1


def test_drafted_generation_refusals():
    target, draft = _models()
    other = _models(vocab=400)[1]
    prompt = torch.randint(0, 400, (1, 9), device=DEV)
    for kw in (dict(draft_model=other), dict(draft_model=draft, num_drafts=65), dict(draft_model=draft, num_drafts=-1),
               dict(draft_model=draft, kv_caches=[None] * 3)):
        with pytest.raises(ValueError):
            target.generate(prompt, max_new_tokens=4, **kw)
    with pytest.raises(ValueError):
        target.generate(prompt.repeat(2, 1), max_new_tokens=4, draft_model=draft)
