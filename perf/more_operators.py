"""The operators of a server that keeps its keys and values in 4 bits and decodes
drafted tokens, as cases that can be timed: the write of new keys and values into
pages with the position rotation applied on the way (16-bit pages, and pages of 4-bit
codes), attention of one or a few tokens a sequence over the 4-bit pages, and the
verification of drafted tokens.

``run`` computes them in plain torch operations, or with ``own`` through the
library's entry points. The sizes are those of the repository's configurations
(12 query heads over 4 KV heads of dimension 64, contexts up to 16K and 32K, a
vocabulary of 32000) and generic ones: 32 heads over 8 of dimension 128, pages of 16 to
128 tokens, an odd vocabulary.

A page of 4-bit codes. Dims are taken in groups of 32. A group of a key or a value
stands for h (2 c - 15), c in 0 .. 15 per dim, h in 16-bit floating point: the group's
largest magnitude over 15, and c = floor(x / 2h) + 8 cut to the range, x being the (rotated) row in
bfloat16. A page holds [Hkv, page_size / 16] tiles of 16 positions of one head,
each 576 bytes per group of the head: the keys' codes, the values' codes, the keys' h
[16, groups], the values' h. Keys' codes: position, then four quarters of
the groups' eighths (see ``_key_bytes``); values' codes: four positions a word (see ``_value_bytes``).
"""

import math
import os
import random
import sys

import torch

own = False

_BF, _F32, _F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # the write of a decode step: one token of every sequence, a rotation and a copy
        {"name": "rotate 64x1", "op": "rotate", "n": 64, "N": 64, "Hq": 12, "Hkv": 4, "D": 64, "ps": 64,
         "dtype": "bf16"},
        # the write of a prefill step: whole prompts behind cached prefixes, a larger model's heads
        {"name": "rotate 16, 16000 tokens, 32/8x128", "op": "rotate", "n": 16, "N": 16000, "Hq": 32, "Hkv": 8,
         "D": 128, "ps": 16, "dtype": "bf16"},
        # an evaluation in float32 over documents of mixed lengths
        {"name": "rotate 3, 1501 tokens f32", "op": "rotate", "n": 3, "N": 1501, "Hq": 12, "Hkv": 4, "D": 64,
         "ps": 32, "dtype": "f32"},
        # a decode step's write into 4-bit pages, and its rows read back
        {"name": "append q4 64x1", "op": "append_q4", "n": 64, "N": 64, "Hq": 12, "Hkv": 4, "D": 64, "ps": 64,
         "dtype": "bf16"},
        # a prefill step of prompts in chunks: the new rows into 4-bit pages, then every row so far read back
        # for the chunk's attention
        {"name": "append q4 16, 16000 tokens, 32/8x128", "op": "append_q4", "n": 16, "N": 16000, "Hq": 32, "Hkv": 8,
         "D": 128, "ps": 16, "dtype": "bf16"},
        # a token of one short conversation: latency
        {"name": "decode q4 1x1000", "op": "decode_q4", "B": 1, "T": 1, "S": 1000, "Hq": 12, "Hkv": 4, "D": 64,
         "ps": 16, "dtype": "bf16"},
        # a batch at the decode benchmark's context
        {"name": "decode q4 8x16384", "op": "decode_q4", "B": 8, "T": 1, "S": 16384, "Hq": 12, "Hkv": 4, "D": 64,
         "ps": 64, "dtype": "bf16"},
        # a full server with a larger model's heads
        {"name": "decode q4 32x16384, 32/8x128", "op": "decode_q4", "B": 32, "T": 1, "S": 16384, "Hq": 32, "Hkv": 8,
         "D": 128, "ps": 16, "dtype": "bf16"},
        # four drafted tokens and the one before them, of every sequence
        {"name": "decode q4 16x5 at 8000, 32/8x128", "op": "decode_q4", "B": 16, "T": 5, "S": 8000, "Hq": 32,
         "Hkv": 8, "D": 128, "ps": 16, "dtype": "bf16"},
        # tokens looked up in the prompt for one conversation: latency
        {"name": "verify 1x4 of 32000", "op": "verify", "B": 1, "K": 4, "V": 32000, "drafts": "given",
         "temperature": 0.8, "dtype": "bf16"},
        # a small draft model beside a batch, logits in float32
        {"name": "verify 32x5 of 32000 f32", "op": "verify", "B": 32, "K": 5, "V": 32000, "drafts": "sampled",
         "temperature": 1.0, "dtype": "f32"},
        # a full server, a larger and odd vocabulary
        {"name": "verify 64x7 of 50257", "op": "verify", "B": 64, "K": 7, "V": 50257, "drafts": "sampled",
         "temperature": 0.8, "dtype": "bf16"},
    ]


# what the largest listed cases of each kind move: no drawn case costs more
_ROWS_MOST = 16000 * 8 * 128
_DECODE_MOST = 16384 * 32 * 8 * 128
_VERIFY_MOST = 64 * 8 * 50257


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "append_q4", "append_q4", "decode_q4", "decode_q4", "decode_q4", "verify", "verify"])
    Hq, Hkv, D = rng.choice([(12, 4, 64), (12, 4, 64), (4, 4, 64), (8, 4, 64), (16, 4, 64), (32, 8, 128), (8, 1, 128)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    ps = rng.choice([16, 32, 64, 128])
    if op == "verify":
        V = _log(rng, 1000, 129000)
        K = rng.choice([0, 1, 2, 3, 4, 5, 6, 7, 8])
        B = _log(rng, 1, max(1, min(64, _VERIFY_MOST // ((K + 1) * V * (2 if dtype == "f32" else 1)))))
        return {"op": op, "B": B, "K": K, "V": V, "drafts": rng.choice(["given", "sampled"]),
                "temperature": rng.choice([0.6, 0.8, 1.0]), "dtype": dtype}
    if op == "decode_q4":
        B, S, T = _log(rng, 1, 128), _log(rng, 8, 131000), rng.choice([1, 1, 1, 2, 3, 4, 6, 8])
        while B * S * Hkv * D * (1 + T // 2) > _DECODE_MOST:
            S = S * 7 // 10
        S = max(S, T)
        return {"op": op, "B": B, "T": T, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "ps": ps, "dtype": dtype}
    n = _log(rng, 1, 128)
    N = n if rng.random() < 0.5 else max(n, _log(rng, n, 16000))
    while N * Hkv * D * (1 if dtype == "bf16" else 2) > _ROWS_MOST:
        N = N * 7 // 10
    return {"op": op, "n": n, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D, "ps": ps, "dtype": dtype}


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


def _contexts(B, S, T):
    """B cached lengths: the longest S, the others from a quarter of it, the T new tokens among them."""
    rng = random.Random(1000 * B + S)
    return [S] + [max(T, int(S * rng.uniform(0.25, 1.0))) for _ in range(B - 1)]


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


def _angles(rows, D):
    """cos, sin [rows, D/2] in float32 of the model's rotation, angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=_F64, device="cuda") / D)
    a = torch.arange(rows, dtype=_F64, device="cuda")[:, None] * inv
    return torch.cos(a).to(_F32), torch.sin(a).to(_F32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 31)
    dt = _dtype(case)

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    if case["op"] == "verify":
        return _prepare_verify(case, g, dt)
    Hq, Hkv, D, ps = case["Hq"], case["Hkv"], case["D"], case["ps"]
    if case["op"] == "decode_q4":
        B, T = case["B"], case["T"]
        lengths = _contexts(B, case["S"], T)
        table, pages = _table(lengths, ps, g)
        packed = []
        for p0 in range(0, pages, 4096):
            n = min(4096, pages - p0)
            packed.append(_pack(*(torch.randn(n, ps, Hkv, D, generator=g, device="cuda").to(_BF) for _ in range(2))))
        q = randn(B, T, Hq, D, std=2.0)
        return {"op": "decode_q4", "q": q[:, 0] if T == 1 else q, "pages": torch.cat(packed), "table": table,
                "lengths": ints(lengths), "D": D}
    new, old = _prompts(case["n"], case["N"]), _prefixes(case["n"])
    whole = [a + b for a, b in zip(new, old)]
    table, pages = _table(whole, ps, g)
    cos, sin = _angles(max(whole), D)
    s = {"op": case["op"], "table": table, "positions": ints(old), "q": randn(case["N"], Hq, D),
         "k_new": randn(case["N"], Hkv, D), "v_new": randn(case["N"], Hkv, D), "cos": cos, "sin": sin,
         "cu": None if case["N"] == case["n"] else ints(_cumulative(new))}
    if case["op"] == "rotate":
        return {**s, "k": randn(pages, ps, Hkv, D), "v": randn(pages, ps, Hkv, D)}
    packed = _pack(*(torch.randn(pages, ps, Hkv, D, generator=g, device="cuda").to(_BF) for _ in range(2)))
    # what is read back: a decode step's rows, or for a prompt's chunk all of its sequence so far
    step = s["cu"] is None
    return {**s, "pages": packed, "D": D, "from": s["positions"] if step else torch.zeros_like(s["positions"]),
            "rows": None if step else ints(_cumulative(whole)), "count": case["N"] if step else sum(whole)}


def _prepare_verify(case, g, dt):
    B, K, V = case["B"], case["K"], case["V"]
    x = torch.randn(B, K + 1, V, generator=g, device="cuda") * 3.0
    logits = x.to(dt)
    temperature = torch.full((B,), case["temperature"], device="cuda")
    temperature[3::4] = 0.0                       # some of a batch's requests are greedy
    s = {"op": "verify", "logits": logits, "temperature": temperature, "probs": None,
         "uniform": torch.rand(B, K + 1, generator=g, device="cuda"),
         "counts": torch.randint((K + 1) // 2, K + 1, (B,), generator=g, device="cuda").to(torch.int32)}
    # the draft's distribution is near the target's
    near = torch.softmax((x[:, :K] + torch.randn(B, K, V, generator=g, device="cuda") * 0.7)
                         / temperature.clamp(min=0.25)[:, None, None], -1)
    if K == 0:
        s["drafts"] = torch.zeros((B, 0), dtype=torch.int32, device="cuda")
    else:
        s["drafts"] = torch.multinomial(near.view(B * K, V), 1, generator=g).view(B, K).to(torch.int32)
    if case["drafts"] == "sampled":
        s["probs"] = near
    return s


# ---------------------------------------------------------------------------
# a page of 4-bit codes
# ---------------------------------------------------------------------------

_E = [0, 2, 4, 6, 1, 3, 5, 7]        # the eight dims of a key word, by nibble
_I = [0, 2, 1, 3]                    # the four positions of a value word, by byte


def _codes(x, d):
    """Codes and h of rows x [..., D] in bfloat16, computed in type d."""
    x = x.to(d).unflatten(-1, (-1, 32))
    h = (x.abs().amax(-1) / 15).to(torch.float16)
    c = torch.floor(x / (2 * h.to(d)[..., None])).add_(8).clamp_(0, 15)
    c = torch.where(h[..., None] > 0, c, torch.full_like(c, 8))
    return c.to(torch.uint8), h


def _key_bytes(c):
    """Codes [..., G, 32] of keys to bytes [..., 16 G]: quarter, group, four bytes of eight dims."""
    c = c.unflatten(-1, (4, 8))[..., _E].unflatten(-1, (4, 2))
    return (c[..., 0] | c[..., 1] << 4).transpose(-3, -2).flatten(-3)


def _value_bytes(c):
    """Codes [..., G, 32] of values to bytes [..., 16, G], two dims each: they go to word (position / 4, pair)."""
    c = c.unflatten(-1, (16, 2))
    return (c[..., 0] | c[..., 1] << 4).transpose(-2, -1)


def _pack(k, v):
    """[pages, ps, Hkv, D] keys and values in bfloat16 to [pages, Hkv, ps/16, 576 G] bytes."""
    P, ps, Hkv, D = k.shape
    (ck, hk), (cv, hv) = (_codes(x.transpose(1, 2), _F32) for x in (k, v))
    kb = _key_bytes(ck).view(P, Hkv, ps // 16, -1)
    vb = _value_bytes(cv).view(P, Hkv, ps // 16, 4, 4, 16, -1)[:, :, :, :, _I].permute(0, 1, 2, 3, 5, 6, 4)
    parts = [kb, vb.reshape(P, Hkv, ps // 16, -1)]
    parts += [h.contiguous().view(torch.uint8).view(P, Hkv, ps // 16, -1) for h in (hk, hv)]
    return torch.cat(parts, -1)


def _places(D, device):
    """Bytes of position 0 .. 15 in a tile: keys' codes [16, D/2], values' codes [16, 16, G], h of both [16, 2 G]."""
    G = D // 32
    i = torch.arange(16, device=device)
    kb = i[:, None] * (16 * G) + torch.arange(16 * G, device=device)
    slot = torch.tensor([0, 2, 1, 3], device=device)[i % 4]
    vb = (256 * G + ((i // 4)[:, None, None] * 16 + torch.arange(16, device=device)[:, None]) * (4 * G)
          + torch.arange(G, device=device) * 4 + slot[:, None, None])
    hk = 512 * G + i[:, None] * (2 * G) + torch.arange(2 * G, device=device)
    return kb, vb, hk, hk + 32 * G


def _values(ck, cv, hk, hv, d):
    """Bytes of rows ([..., 16 G], [..., 16, G], [..., 2 G] twice) to keys and values [..., D] of type d."""
    G = cv.shape[-1]
    out = []
    b = ck.unflatten(-1, (4, G, 4)).transpose(-3, -2)
    k = torch.empty(*b.shape[:-1], 8, dtype=d, device=ck.device)
    k[..., _E] = torch.stack((b & 15, b >> 4), -1).flatten(-2).to(d)
    v = torch.stack((cv & 15, cv >> 4), -1).transpose(-3, -2).to(d)
    for c, h in ((k, hk), (v, hv)):
        h = h.contiguous().view(torch.float16).to(d)
        out.append((c.flatten(-2) * 2 - 15).mul_(h[..., None]).flatten(-2))
    return out


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------

def _sequence_of(cu, N):
    """Sequence and place in it of every packed token."""
    t = torch.arange(N, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    return seq, t - cu.long()[seq]


def _rows_of(table, positions, cu, N, ps):
    """Position, page and row in the page of N packed rows."""
    if cu is None:
        seq, pos = torch.arange(N, device=table.device), positions.long()
    else:
        seq, pos = _sequence_of(cu, N)
        pos = pos + positions.long()[seq]
    return pos, table.long()[seq, pos // ps], pos % ps


def _turned(x, cos, sin, pos, d):
    """Rows x [N,H,D] turned by their positions' angles: pairs (i, i + D/2)."""
    c, s = cos[pos].to(d)[:, None], sin[pos].to(d)[:, None]
    a, b = x.to(d).chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _plain_rotate(s, d=_F32):
    pos, page, row = _rows_of(s["table"], s["positions"], s["cu"], s["q"].shape[0], s["k"].shape[1])
    q, k = (_turned(s[x], s["cos"], s["sin"], pos, d).to(s["q"].dtype) for x in ("q", "k_new"))
    s["k"][page, row] = k
    s["v"][page, row] = s["v_new"]
    return q, s["k"], s["v"]


def _tile_bytes(s, page, row):
    """Index of every byte of N rows in the flat pages, by part."""
    _, Hkv, tiles, size = s["pages"].shape
    base = (page[:, None] * Hkv + torch.arange(Hkv, device=page.device)) * tiles + (row // 16)[:, None]
    return [base.view(*base.shape, *([1] * (p.dim() - 1))) * size + p[row % 16].unsqueeze(1)
            for p in _places(s["D"], page.device)]


def _plain_append_q4(s):
    ps, flat = s["pages"].shape[2] * 16, s["pages"].view(-1)
    pos, page, row = _rows_of(s["table"], s["positions"], s["cu"], s["q"].shape[0], ps)
    q, k = (_turned(s[x], s["cos"], s["sin"], pos, _F32) for x in ("q", "k_new"))
    (ck, hk), (cv, hv) = (_codes(x.to(_BF), _F32) for x in (k, s["v_new"]))
    parts = (_key_bytes(ck), _value_bytes(cv), hk.contiguous().view(torch.uint8), hv.contiguous().view(torch.uint8))
    for at, b in zip(_tile_bytes(s, page, row), parts):
        flat[at] = b
    _, page, row = _rows_of(s["table"], s["from"], s["rows"], s["count"], ps)
    k, v = _values(*(flat[at] for at in _tile_bytes(s, page, row)), _F32)
    return q.to(s["q"].dtype), k.to(_BF), v.to(_BF)


def _plain_decode_q4(s):
    q, table, lengths, D = s["q"], s["table"], s["lengths"], s["D"]
    q = q[:, None] if q.dim() == 3 else q
    B, T, Hq, _ = q.shape
    _, Hkv, tiles, _ = s["pages"].shape
    G, R, cap = D // 32, Hq // Hkv, table.shape[1] * tiles * 16
    out = torch.empty(B, T, Hq, D, dtype=_F32, device=q.device)
    few = max(1, (1 << 29) // (cap * Hkv * D))    # sequences at a time
    at = torch.arange(cap, device=q.device)
    for b0 in range(0, B, few):
        rows = table[b0:b0 + few].clamp(min=0).long()
        n = rows.shape[0]
        x = s["pages"][rows].transpose(1, 2).reshape(n, Hkv, -1, 576 * G)
        k, v = _values(*(x[..., p] for p in _places(D, q.device)), _F32)
        k, v = k.view(n, Hkv, cap, D), v.view(n, Hkv, cap, D)
        y = q[b0:b0 + n].to(_F32).view(n, T, Hkv, R, D).transpose(1, 2).reshape(n, Hkv, T * R, D)
        y = torch.matmul(y, k.transpose(2, 3).contiguous()).view(n, Hkv, T, R, cap) * (1.0 / math.sqrt(D))
        last = lengths[b0:b0 + n, None] - T + 1 + torch.arange(T, device=q.device)
        y.masked_fill_((at >= last[..., None])[:, None, :, None], -math.inf)
        y = torch.exp(y - y.amax(-1, keepdim=True))
        o = torch.matmul(y.view(n, Hkv, T * R, cap), v).view(n, Hkv, T, R, D) / y.sum(-1, keepdim=True)
        out[b0:b0 + n] = o.transpose(1, 2).reshape(n, T, Hq, D)
    out = out.to(q.dtype).view(B, T, Hq * D)
    return out[:, 0] if s["q"].dim() == 3 else out


def _plain_verify(s):
    """In 64 bits: a drawn token is where a long sum passes a number."""
    x, drafts, u, probs, temperature = s["logits"].to(_F64), s["drafts"].long(), s["uniform"].to(_F64), s["probs"], s["temperature"]
    B, K1, V = x.shape
    K = K1 - 1
    greedy = temperature == 0
    t = torch.where(greedy, torch.ones_like(temperature), temperature).to(_F64)
    top = x.amax(-1, keepdim=True)
    best = torch.where(x == top, torch.arange(V, device=x.device), V).amin(-1)     # ties: the lowest
    p = torch.exp((x - top) / t[:, None, None])
    p /= p.sum(-1, keepdim=True)
    pd = p[:, :K].gather(2, drafts[..., None])[..., 0]
    qd = torch.ones_like(pd) if probs is None else probs.gather(2, drafts[..., None])[..., 0].to(_F64)
    ok = torch.where(greedy[:, None], drafts == best[:, :K], u[:, :K] * qd < pd)
    ok &= torch.arange(K, device=x.device) < s["counts"][:, None]
    n = ok.long().cumprod(1).sum(1)               # drafts accepted
    rows = torch.arange(B, device=x.device)
    r = p[rows, n]
    if K > 0:
        short, at = n < s["counts"], n.clamp(max=K - 1)
        if probs is None:
            less = r.scatter(1, drafts[rows, at][:, None], 0.0)
        else:
            less = (r - probs[rows, at].to(_F64)).clamp_(min=0.0)
        r = torch.where((short & (less.sum(1) > 0))[:, None], less, r)
    r = r.cumsum(1)
    last = torch.searchsorted(r, r[:, -1:].contiguous())        # the last token that weighs anything
    drawn = torch.minimum(torch.searchsorted(r, u[:, K:] * r[:, -1:], right=True), last)[:, 0]
    tokens = torch.full((B, K1), -1, dtype=torch.long, device=x.device)
    if K > 0:
        tokens[:, :K] = torch.where(torch.arange(K, device=x.device) < n[:, None], drafts, -1)
    tokens[rows, n] = torch.where(greedy, best[rows, n], drawn)
    return tokens.to(torch.int32), n.to(torch.int32)


def run(state):
    s = state
    if own:
        lib = _library()
        if s["op"] == "rotate":
            q = lib.rotate_append_paged(s["k"], s["v"], s["table"], s["positions"], s["q"], s["k_new"], s["v_new"],
                                        s["cos"], s["sin"], cu_seqlens=s["cu"])
            return q, s["k"], s["v"]
        if s["op"] == "append_q4":
            q = lib.append_paged_q4(s["pages"], s["table"], s["positions"], s["k_new"], s["v_new"], cu_seqlens=s["cu"],
                                    q=s["q"], cos=s["cos"], sin=s["sin"])
            return (q, *lib.gather_paged_q4(s["pages"], s["table"], s["from"], s["count"], cu_seqlens=s["rows"]))
        if s["op"] == "decode_q4":
            return lib.decode_paged_q4(s["q"], s["pages"], s["table"], s["lengths"])
        return lib.verify_drafts(s["logits"], s["drafts"], s["uniform"], draft_probs=s["probs"], n_drafts=s["counts"],
                                 temperature=s["temperature"])
    return {"rotate": _plain_rotate, "append_q4": _plain_append_q4, "decode_q4": _plain_decode_q4,
            "verify": _plain_verify}[s["op"]](s)


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
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "verify":
        B, K, V = case["B"], case["K"], case["V"]
        # the logits, and of the draft's distributions the one that a rejected token is drawn against
        return {"bytes": B * (K + 1) * V * size + (B * V * 4 if case["drafts"] == "sampled" and K > 0 else 0),
                "flops": 3 * B * (K + 1) * V}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    row = 2 * Hkv * (D // 2 + D // 16)            # a position of 4-bit pages
    if case["op"] == "decode_q4":
        B, T = case["B"], case["T"]
        tokens = sum(_contexts(B, case["S"], T))
        return {"bytes": tokens * row + 2 * B * T * Hq * D * size, "flops": 4 * D * Hq * T * tokens}
    N = case["N"]
    if case["op"] == "rotate":
        return {"bytes": 2 * N * (Hq + 2 * Hkv) * D * size, "flops": 3 * N * (Hq + Hkv) * D}
    back = N if N == case["n"] else N + sum(_prefixes(case["n"]))
    return {"bytes": N * (2 * Hq + 2 * Hkv) * D * size + N * row + back * (row + 4 * Hkv * D),
            "flops": 3 * N * (Hq + Hkv) * D + 6 * N * Hkv * D + 4 * back * Hkv * D}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _held64(x):
    """What rows x [..., D] in bfloat16 are held as: the nearest odd multiple of h of its group."""
    x = x.double().unflatten(-1, (-1, 32))
    h = (x.abs().amax(-1, keepdim=True) / 15).half().double()
    odd = 2 * torch.floor(x / (2 * h)) + 1
    return torch.where(h > 0, odd.clamp(-15, 15) * h, 0.0).flatten(-2)


def _all64(pages, D):
    """Every key and value of 4-bit pages: [pages, Hkv, page_size, D] in 64 bits, nibble by nibble."""
    P, Hkv, tiles, size = pages.shape
    G = D // 32
    x = pages.view(P, Hkv, tiles, size)
    scale = x[..., 512 * G:].contiguous().view(torch.float16).double().view(P, Hkv, tiles, 2, 16, G)
    out = []
    for what in (0, 1):
        y = torch.empty(P, Hkv, tiles, 16, D, dtype=_F64, device=pages.device)
        for d in range(D):
            g, e = d // 32, d % 32
            for i in range(16):
                if what == 0:
                    nibble = (e % 8) // 2 + 4 * (e % 2)
                    byte = i * 16 * G + (e // 8) * 4 * G + g * 4 + nibble // 2
                else:
                    nibble = e % 2
                    byte = 256 * G + ((i // 4) * 16 + e // 2) * 4 * G + g * 4 + (0, 2, 1, 3)[i % 4]
                y[:, :, :, i, d] = ((x[..., byte] >> (4 * (nibble % 2))) & 15).double() * 2 - 15
        y *= scale[..., what, :, :].repeat_interleave(32, -1)
        out.append(y.view(P, Hkv, tiles * 16, D))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(s)
    D, ps = case["D"], case["ps"]
    if case["op"] == "decode_q4":
        B, T, R = case["B"], case["T"], case["Hq"] // case["Hkv"]
        if s["pages"].numel() > 1 << 30:
            return None                           # (pages of many gigabytes in 64 bits)
        k, v = _all64(s["pages"], D)
        q = s["q"].view(B, T, case["Hq"], D)
        out = torch.empty(B, T, case["Hq"], D, dtype=_F64, device="cuda")
        for b, n in enumerate(_contexts(B, case["S"], T)):
            ids = s["table"][b, :(n + ps - 1) // ps].long()
            for g in range(case["Hkv"]):
                kb, vb = (x[ids, g].flatten(0, 1) for x in (k, v))
                for t in range(T):
                    m = n - T + 1 + t
                    x = q[b, t, g * R:(g + 1) * R].double() @ kb[:m].T / math.sqrt(D)
                    out[b, t, g * R:(g + 1) * R] = torch.softmax(x, -1) @ vb[:m]
        out = out.view(B, T, -1)
        return out[:, 0] if T == 1 else out
    new, old = _prompts(case["n"], case["N"]), _prefixes(case["n"])
    q = torch.empty(s["q"].shape, dtype=_F64, device="cuda")
    coded = case["op"] == "append_q4"
    if coded:
        k, v = (x.transpose(1, 2).contiguous() for x in _all64(s["pages"], D))
    else:
        k, v = s["k"].double(), s["v"].double()
    at, rows = 0, []
    for i, (t, p) in enumerate(zip(new, old)):
        pos = torch.arange(p, p + t, device="cuda")
        page, row = s["table"][i].long()[pos // ps], pos % ps
        # (rows of one sequence at once: heads beside positions)
        c, z = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
        turn = torch.complex(c, z)
        both = []
        for x in ("q", "k_new"):
            a, b = s[x][at:at + t].double().chunk(2, -1)
            y = torch.complex(a, b) * turn
            both.append(torch.cat((y.real, y.imag), -1))
        q[at:at + t] = both[0]
        if coded:
            k[page, row], v[page, row] = _held64(both[1].to(_BF)), _held64(s["v_new"][at:at + t].to(_BF))
        else:
            k[page, row], v[page, row] = both[1], s["v_new"][at:at + t].double()
        first = p if case["N"] == case["n"] else 0
        pos = torch.arange(first, p + t, device="cuda")
        rows.append((s["table"][i].long()[pos // ps], pos % ps))
        at += t
    if not coded:
        return q, k, v
    return (q, *(torch.cat([x[page, row] for page, row in rows]) for x in (k, v)))


def _exact_verify(s):
    B, K1, V = s["logits"].shape
    tokens, counts = [], []
    for b in range(B):
        n, row, temperature = 0, [], float(s["temperature"][b])
        last = None
        for i in range(K1):
            x = s["logits"][b, i].double()
            p = None if temperature == 0 else torch.softmax(x / temperature, 0)
            if i == int(s["counts"][b]):
                last = p if p is not None else x
                break
            d = int(s["drafts"][b, i])
            if p is None:
                if d != int(torch.nonzero(x == x.max())[0]):
                    last = x
                    break
            else:
                mine = s["probs"][b, i].double() if s["probs"] is not None else None
                if not float(s["uniform"][b, i]) * (1.0 if mine is None else float(mine[d])) < float(p[d]):
                    r = p.clone()
                    if mine is None:
                        r[d] = 0.0
                    else:
                        r = (p - mine).clamp(min=0.0)
                    last = r if float(r.sum()) > 0 else p
                    break
            row.append(d)
            n += 1
        if temperature == 0:
            row.append(int(torch.nonzero(last == last.max())[0]))
        else:
            c = torch.cumsum(last, 0)
            above = torch.nonzero(c > float(s["uniform"][b, K1 - 1]) * float(c[-1]))
            row.append(int(above[0]) if above.numel() else int(torch.nonzero(last)[-1]))
        tokens.append(row + [-1] * (K1 - len(row)))
        counts.append(n)
    return (torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.tensor(counts, dtype=torch.int32, device="cuda"))
