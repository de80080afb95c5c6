"""How far attention over 4-bit pages may be off from float64, as one relative number for a token's whole output
(||got - want|| / ||want|| over its heads and dims). Unlike a bound of every element by the sum of all magnitudes it
does not grow with the length, so that a lost share, a lost key or a lost term of a split shows at any length.

bf16. A weight times h and an output are each rounded to bf16: relative errors of at most 2^-8, spread evenly over a
step of 2^-8 .. 2^-7 of the value: rms 2^-8 / sqrt(3) / 1.44 = 0.0016. Weights' errors are independent from key to key,
as the values are, so that they move an output's norm by 0.0016 of itself; both together 0.0023. Over the 64 numbers of the
smallest outputs here the rms itself varies by 1 / sqrt(128) = 9%, and values that are not independent of their weights
may give up to both roundings' largest; 2^-8 = 0.0039 is five times that variation above 0.0023.

fp32. q and the weights keep 24 bits (three bf16 terms). What is left are sums: a score's G products of 32 with codes
16.5 + c against -24 times the sum of q, magnitudes up to 24 sqrt(32) |q| 2 h scale, and a step's sums of 32 weights times
16.5 + c against -24 times their sum, which cancel to (c - 7.5) P. With N(0,1) rows h = 0.15 and rms(c - 7.5) = 3.4:
    scores   G products of 32 and 3 roundings: sqrt(3 G) 2^-24 24 sqrt(32) 2 h / sqrt(D) rms(q): 0.7e-6 rms(q) at most, a
             weight's relative error, independent from key to key;
    outputs  six products a step, each rounded at 24 32 h / 2 rms 0.29 2^-23: sqrt(6 n / 32) of these against
             3.4 h sqrt(n) is 0.4 0.29 2^-23 768 / 3.4 = 3e-6 where the weights are alike (less where few keys hold them).
sqrt(9 + 2) 1e-6 for rms(q) = 2; three times that, 1e-5, is the limit.

That holds where a wavefront's walk is short. Over s steps the running sums are rounded at their own size, as any fp32 sum is:
an output seven times a step (three terms of two products, and their sum), the weights' sum eight times (a lane's
keys); independent errors of rms 2^-24 / sqrt(3) each, 15 s of them: 2.1e-6 at 256 steps, which the limit above
still leaves room for, 8.5e-6 at 4096. `walk_limit` is three times both together."""

import numpy as np

LIMIT = {"bf16": 2.0 ** -8, "f32": 1e-5}


def walk_limit(steps):
    return 3 * (11e-12 + 15 * steps * (2.0 ** -24 / 3 ** 0.5) ** 2) ** 0.5


def relative(got, want):
    """got, want [..., n] -> [...]"""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)


def attend64(q, k, v, scale, keep=None):
    """q [H,D], one KV head's k, v [n,D], all float64 -> [H,D]; keep: the keys that take part."""
    s = q @ k.T * scale
    if keep is not None:
        s[:, ~keep] = -np.inf
    w = np.exp(s - s.max(axis=1, keepdims=True))
    return (w / w.sum(axis=1, keepdims=True)) @ v


def aligned_queries(k, at, scale, gain=12.0):
    """One query per position in `at`, q = a k[at]: that key's score is `gain` and, rows of N(0,1) being nearly
    orthogonal, it holds most of the weight: exp(12) against the sum over n others of exp(N(0, 12 / sqrt(D)))."""
    x = k[list(at)]
    return x * (gain / scale / (x * x).sum(-1, keepdims=True))
