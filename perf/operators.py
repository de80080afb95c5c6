"""The serving operators for batches of requests of different lengths, as cases
that can be timed: causal attention over packed prompts, the write of new keys
and values into a paged cache, and single-token attention over that cache.

``run`` computes them in plain torch operations, or with ``own`` through the
library's entry points. The sizes are those of the repository's configurations
(12 query heads over 4 KV heads of dimension 64, contexts up to 16K and 32K)
and generic ones: 32 heads over 8 of dimension 128, pages of 16 to 128 tokens.
"""

import math
import os
import random
import sys

import torch

own = False

_BF, _F32 = torch.bfloat16, torch.float32


def listed():
    return [
        # the smallest prompt that a server sees alone: latency
        {"name": "prompt 1x37", "op": "prefill", "n": 1, "N": 37, "Hq": 12, "Hkv": 4, "D": 64, "dtype": "bf16"},
        # a prefill step of a server: prompts of mixed lengths within a token budget
        {"name": "prompts 16, 4099 tokens", "op": "prefill", "n": 16, "N": 4099, "Hq": 12, "Hkv": 4, "D": 64,
         "dtype": "bf16"},
        # one long prompt, the largest context of a dense layer
        {"name": "prompt 1x16384", "op": "prefill", "n": 1, "N": 16384, "Hq": 12, "Hkv": 4, "D": 64, "dtype": "bf16"},
        # the same server with a larger model's heads
        {"name": "prompts 8, 16000 tokens, 32/8x128", "op": "prefill", "n": 8, "N": 16000, "Hq": 32, "Hkv": 8,
         "D": 128, "dtype": "bf16"},
        # an evaluation in float32 over documents of mixed lengths
        {"name": "prompts 3, 1501 tokens f32", "op": "prefill", "n": 3, "N": 1501, "Hq": 12, "Hkv": 4, "D": 64,
         "dtype": "f32"},
        # a token of one short conversation: latency
        {"name": "decode 1x1000", "op": "decode", "B": 1, "S": 1000, "Hq": 12, "Hkv": 4, "D": 64, "ps": 16,
         "dtype": "bf16"},
        # a batch at the decode benchmark's context
        {"name": "decode 8x16384", "op": "decode", "B": 8, "S": 16384, "Hq": 12, "Hkv": 4, "D": 64, "ps": 64,
         "dtype": "bf16"},
        # one long document
        {"name": "decode 1x131000", "op": "decode", "B": 1, "S": 131000, "Hq": 12, "Hkv": 4, "D": 64, "ps": 64,
         "dtype": "bf16"},
        # a full server with a larger model's heads
        {"name": "decode 32x16384, 32/8x128", "op": "decode", "B": 32, "S": 16384, "Hq": 32, "Hkv": 8, "D": 128,
         "ps": 16, "dtype": "bf16"},
        # a small batch in float32
        {"name": "decode 5x3001 f32", "op": "decode", "B": 5, "S": 3001, "Hq": 12, "Hkv": 4, "D": 64, "ps": 32,
         "dtype": "f32"},
        # the write of a decode step: one token of every sequence
        {"name": "append 64x1", "op": "append", "n": 64, "N": 64, "Hkv": 4, "D": 64, "ps": 64, "dtype": "bf16"},
        # the write of a prefill step: whole prompts behind cached prefixes
        {"name": "append 16, 16000 tokens", "op": "append", "n": 16, "N": 16000, "Hkv": 8, "D": 128, "ps": 16,
         "dtype": "bf16"},
    ]


# the largest listed prefill (multiply-adds) and decode (cache elements read): no drawn case costs more
_PREFILL_MOST = 16384 * 16385 // 2 * 12 * 64
_DECODE_MOST = 16384 * 18 * 8 * 128


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "prefill", "decode", "decode", "decode", "append"])
    Hq, Hkv, D = rng.choice([(12, 4, 64), (12, 4, 64), (4, 4, 64), (8, 4, 64), (16, 4, 64), (32, 8, 128), (8, 1, 128)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    ps = rng.choice([16, 32, 64, 128])
    if op == "prefill":
        N = _log(rng, 8, 16384 if dtype == "bf16" else 4000)
        n = _log(rng, 1, max(1, min(32, N // 4)))
        while sum(t * (t + 1) // 2 for t in _prompts(n, N)) * Hq * D > _PREFILL_MOST * (1 if dtype == "bf16" else 0.1):
            N = N * 7 // 10
        return {"op": op, "n": n, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype}
    if op == "decode":
        B, S = _log(rng, 1, 128), _log(rng, 1, 131000)
        while B * S * Hkv * D * (1 if dtype == "bf16" else 2) > _DECODE_MOST:
            S = S * 7 // 10
        return {"op": op, "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "ps": ps, "dtype": dtype}
    n = _log(rng, 1, 128)
    N = n if rng.random() < 0.5 else max(n, _log(rng, n, 16000))
    return {"op": op, "n": n, "N": N, "Hkv": Hkv, "D": D, "ps": ps, "dtype": dtype}


# ---------------------------------------------------------------------------
# lengths and inputs
# ---------------------------------------------------------------------------

def _prompts(n, N):
    """n lengths of N tokens in all, most between a quarter and twice the mean."""
    if n == N:
        return [1] * n
    rng = random.Random(1000 * n + N)
    w = [rng.uniform(0.25, 1.75) for _ in range(n)]
    cut, at, out = 0.0, 0, []
    for x in w:
        cut += x
        to = round(N * cut / sum(w))
        out.append(to - at)
        at = to
    return out


def _contexts(B, S):
    """B cached lengths: the longest S, the others from a quarter of it."""
    rng = random.Random(1000 * B + S)
    return [S] + [max(1, int(S * rng.uniform(0.25, 1.0))) for _ in range(B - 1)]


def _prefixes(n):
    """Tokens already cached before an append."""
    rng = random.Random(n)
    return [rng.randrange(0, 200) for _ in range(n)]


def _dtype(case):
    return _F32 if case["dtype"] == "f32" else _BF


def _cumulative(lengths):
    out = [0]
    for t in lengths:
        out.append(out[-1] + t)
    return out


def _table(lengths, ps, g):
    """Pages in random order, as a server that has run for a while hands them out."""
    need = [(t + ps - 1) // ps for t in lengths]
    order = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    cols = torch.arange(max(need), device="cuda")
    table[cols[None, :] < torch.tensor(need, device="cuda")[:, None]] = order
    return table, sum(need)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    dt, Hkv, D = _dtype(case), case["Hkv"], case["D"]

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    if case["op"] == "prefill":
        N, lengths = case["N"], _prompts(case["n"], case["N"])
        return {"op": "prefill", "q": randn(N, case["Hq"], D, std=2.0), "k": randn(N, Hkv, D), "v": randn(N, Hkv, D),
                "cu": ints(_cumulative(lengths)), "longest": max(lengths)}
    if case["op"] == "decode":
        lengths = _contexts(case["B"], case["S"])
        table, pages = _table(lengths, case["ps"], g)
        return {"op": "decode", "q": randn(case["B"], case["Hq"], D, std=2.0), "k": randn(pages, case["ps"], Hkv, D),
                "v": randn(pages, case["ps"], Hkv, D), "table": table, "lengths": ints(lengths)}
    new, old = _prompts(case["n"], case["N"]), _prefixes(case["n"])
    table, pages = _table([a + b for a, b in zip(new, old)], case["ps"], g)
    return {"op": "append", "k": randn(pages, case["ps"], Hkv, D), "v": randn(pages, case["ps"], Hkv, D),
            "table": table, "positions": ints(old), "k_new": randn(case["N"], Hkv, D), "v_new": randn(case["N"], Hkv, D),
            "cu": None if case["N"] == case["n"] else ints(_cumulative(new))}


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------

def _sequence_of(cu, N):
    """Sequence and place in it of every packed token."""
    t = torch.arange(N, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    return seq, t - cu.long()[seq]


def _plain_prefill(s):
    q, k, v, cu, L = s["q"], s["k"], s["v"], s["cu"], s["longest"]
    (N, Hq, D), Hkv, n = q.shape, k.shape[1], cu.numel() - 1
    R = Hq // Hkv
    seq, pos = _sequence_of(cu, N)
    qp = q.new_zeros((n, Hkv, R, L, D), dtype=_F32)
    kp, vp = (q.new_zeros((n, Hkv, L, D), dtype=_F32) for _ in range(2))
    qp[seq, :, :, pos] = q.float().view(N, Hkv, R, D)
    kp[seq, :, pos] = k.float()
    vp[seq, :, pos] = v.float()
    x = torch.matmul(qp.view(n, Hkv, R * L, D), kp.transpose(2, 3).contiguous()).view(n, Hkv, R, L, L)
    x *= 1.0 / math.sqrt(D)
    at = torch.arange(L, device=q.device)
    x.masked_fill_(at[None, :] > at[:, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    z = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(n, Hkv, R * L, L), vp).view(n, Hkv, R, L, D) / z
    return o[seq, :, :, pos].reshape(N, Hq * D).to(q.dtype)


def _plain_decode(s):
    q, table, lengths = s["q"], s["table"], s["lengths"]
    (B, Hq, D), (_, ps, Hkv, _) = q.shape, s["k"].shape
    pages = table.clamp(min=0).long()
    k, v = (s[n][pages].view(B, -1, Hkv, D).transpose(1, 2).float().contiguous() for n in ("k", "v"))
    x = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    at = torch.arange(k.shape[2], device=q.device)
    x.masked_fill_((at[None, :] >= lengths[:, None])[:, None, None, :], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    return o.reshape(B, Hq * D).to(q.dtype)


def _plain_append(s):
    n, ps = s["positions"].numel(), s["k"].shape[1]
    if s["cu"] is None:
        seq, pos = torch.arange(n, device=s["k"].device), s["positions"].long()
    else:
        seq, pos = _sequence_of(s["cu"], s["k_new"].shape[0])
        pos = pos + s["positions"].long()[seq]
    page = s["table"].long()[seq, pos // ps]
    s["k"][page, pos % ps] = s["k_new"]
    s["v"][page, pos % ps] = s["v_new"]
    return s["k"], s["v"]


def run(state):
    if own:
        lib = _library()
        if state["op"] == "prefill":
            return lib.prefill_packed(state["q"], state["k"], state["v"], state["cu"])
        if state["op"] == "decode":
            return lib.decode_paged(state["q"], state["k"], state["v"], state["table"], state["lengths"])
        lib.append_paged(state["k"], state["v"], state["table"], state["positions"], state["k_new"], state["v_new"],
                         cu_seqlens=state["cu"])
        return state["k"], state["v"]
    return {"prefill": _plain_prefill, "decode": _plain_decode, "append": _plain_append}[state["op"]](state)


_lib = None


def _library():
    global _lib
    if _lib is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          "local-research-small-language-model_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import sparda
        _lib = sparda
    return _lib


def work(case):
    size, Hkv, D = (4 if case["dtype"] == "f32" else 2), case["Hkv"], case["D"]
    if case["op"] == "prefill":
        pairs = sum(t * (t + 1) // 2 for t in _prompts(case["n"], case["N"]))
        return {"bytes": 2 * case["N"] * (case["Hq"] + Hkv) * D * size + 4 * case["n"], "flops": 4 * D * case["Hq"] * pairs}
    if case["op"] == "decode":
        tokens = sum(_contexts(case["B"], case["S"]))
        return {"bytes": (2 * tokens * Hkv + 2 * case["B"] * case["Hq"]) * D * size, "flops": 4 * D * case["Hq"] * tokens}
    return {"bytes": 4 * case["N"] * Hkv * D * size, "flops": 0}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    D = case["D"]
    if case["op"] == "append":
        want = {}
        new, old = _prompts(case["n"], case["N"]), _prefixes(case["n"])
        table, ps = s["table"].cpu(), case["ps"]
        for name in ("k", "v"):
            pages, rows, at = s[name].double().cpu(), s[name + "_new"].double().cpu(), 0
            for i, (t, p) in enumerate(zip(new, old)):
                for j in range(t):
                    pages[table[i, (p + j) // ps], (p + j) % ps] = rows[at + j]
                at += t
            want[name] = pages
        return want["k"], want["v"]
    R = case["Hq"] // case["Hkv"]
    if case["op"] == "prefill":
        out = torch.empty(case["N"], case["Hq"], D, dtype=torch.float64, device="cuda")
        at = 0
        for t in _prompts(case["n"], case["N"]):
            for h in range(case["Hq"]):
                q, k, v = (s[x][at:at + t, y].double() for x, y in (("q", h), ("k", h // R), ("v", h // R)))
                for r in range(0, t, 2048):  # rows r .. e-1 see the keys up to themselves
                    e = min(t, r + 2048)
                    x = q[r:e] @ k[:e].T / math.sqrt(D) + torch.full((e - r, e), -math.inf, dtype=torch.float64,
                                                                     device="cuda").triu(r + 1)
                    out[at + r:at + e, h] = torch.softmax(x, -1) @ v[:e]
            at += t
        return out.view(case["N"], -1)
    out = torch.empty(case["B"], case["Hq"], D, dtype=torch.float64, device="cuda")
    for b, t in enumerate(_contexts(case["B"], case["S"])):
        ids = s["table"][b, :(t + case["ps"] - 1) // case["ps"]].long()
        k, v = (s[x][ids].flatten(0, 1)[:t].double() for x in ("k", "v"))
        for h in range(case["Hq"]):
            x = torch.mv(k[:, h // R], s["q"][b, h].double()) / math.sqrt(D)
            out[b, h] = torch.softmax(x, 0) @ v[:, h // R]
    return out.view(case["B"], -1)
