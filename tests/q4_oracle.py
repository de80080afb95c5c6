"""Pages of 4-bit codes and attention over them, written from the format's definition
(include/sparda.h) byte by byte, in numpy and on the CPU."""

import numpy as np
import torch


def groups(D):
    return (D + 31) // 32


def bf16(x: np.ndarray) -> np.ndarray:
    """fp32 values rounded to bf16, as fp32."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).float().numpy()


def codes(x: np.ndarray):
    """Rows x [..., D] (rounded to bf16 here) -> codes [..., D], h [..., G] fp16."""
    x = bf16(x).astype(np.float64)
    D, G = x.shape[-1], groups(x.shape[-1])
    g = x.reshape(*x.shape[:-1], G, min(D, 32))
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        top = np.abs(g).max(-1)                             # (NaN passes through)
        h = np.where(np.isfinite(top), np.minimum((top.astype(np.float32) / np.float32(15)), 65504), np.nan).astype(np.float16)
        c = np.floor(g / (2 * h.astype(np.float64)[..., None])) + 8
    c = np.where((h > 0)[..., None], np.clip(c, 0, 15), 8)
    return c.reshape(x.shape).astype(np.uint8), h


def values(c: np.ndarray, h: np.ndarray) -> np.ndarray:
    D, G = c.shape[-1], h.shape[-1]
    return (2.0 * c - 15.0) * np.repeat(h.astype(np.float64), D // G, -1)


def put(page: np.ndarray, head: int, row: int, k: np.ndarray, v: np.ndarray) -> None:
    """Rows k, v [D] into row `row` of a head of a page [Hkv, tiles, 576 G]."""
    D, G, tile, i = k.shape[-1], groups(k.shape[-1]), page[head, row // 16], row % 16
    (ck, hk), (cv, hv) = codes(k), codes(v)
    for d in range(D):
        g, e = d // 32, d % 32
        n = e % 8 // 2 + 4 * (e % 2)
        at = 16 * G * i + 4 * G * (e // 8) + 4 * g + n // 2
        tile[at] = tile[at] & (0xF0 if n % 2 == 0 else 0x0F) | int(ck[d]) << 4 * (n % 2)
        at = 256 * G + 4 * G * (16 * (i // 4) + e // 2) + 4 * g + (0, 2, 1, 3)[i % 4]
        tile[at] = tile[at] & (0xF0 if e % 2 == 0 else 0x0F) | int(cv[d]) << 4 * (e % 2)
    at = 512 * G + 2 * G * i
    tile[at:at + 2 * G] = hk.view(np.uint8)
    tile[at + 32 * G:at + 34 * G] = hv.view(np.uint8)


def held(x: np.ndarray) -> np.ndarray:
    """What rows come back as, in float64."""
    return values(*codes(x))


def turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos) -> torch.Tensor:
    """Rows x [N,H,D] on the CPU turned by their positions, in fp32, not rounded to x's type."""
    c, s = cos[pos][:, None], sin[pos][:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def attend(q, k, v, hk, hv, scale):
    """q [R,D], the held k / v [n,D] in float64, their h [n,G] -> out [R,D] and the bounds for bf16 and
    fp32 queries (same shape).

    A score is sum_g 2 h_g (sum (128 + c) q - 135.5 sum q): every product and sum of a group in fp32, at most
    33 roundings of sums below 143 sum |q| and 33 of sums below 135.5 sum |q|, then G of the groups'
    sum and three of its scaling: an error x of the scores moves out by 2 x A at most, A = sum w |v|. An
    output is 2 sum P (128 + c) - 135.5 sum P over weights P = w h: (n + 16) 2^-24 of 2 (143 + 135.5) sum w h. Where
    bf16 queries are, P is rounded to bf16, 2^-8 of A, and the output, 2^-8 of |out|; for fp32 both
    2^-24 (three bf16 terms hold 24 bits)."""
    D, G, n = q.shape[1], hk.shape[1], k.shape[0]
    per = D // G
    s = q @ k.T * scale
    w = np.exp(s - s.max(axis=1, keepdims=True))
    w /= w.sum(axis=1, keepdims=True)
    out, A = w @ v, w @ np.abs(v)
    e = 2.0 ** -24
    qa = np.abs(q).reshape(-1, G, per).sum(-1)                    # [R,G]
    hq = qa @ hk.astype(np.float64).T                             # [R,n]: sum_g h sum|q|
    ds = abs(scale) * (2 * 33 * (143 + 135.5) + 2 * 15 * (G + 3)) * e * hq.max(axis=1) + 4 * e * np.abs(s).max(axis=1)
    P = np.repeat(w @ hv.astype(np.float64), per, 1)              # sum w h of a dim's group
    f32 = 2 * ds[:, None] * A + (n + 16) * e * (A + 2 * (143 + 135.5) * P) + e * (A + np.abs(out))
    return out, f32 + 2.0 ** -8 * (A + np.abs(out)), f32
