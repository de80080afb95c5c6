"""Attention in float64 for the packed and paged operators, with the bound that
their rounding allows: for output out = sum w v with A = sum w |v|,

* bf16: every weight is rounded to bf16 for the product with v, half a step
  (2^-8) of A at most, and the output once more, 2^-8 of |out|;
* both types: a score is a dot product of D terms in fp32, off by at most
  (D + 2) 2^-24 sum |q k| scale, and is scaled into log2 units and subtracted
  from a reference, 2^-22 of the largest |score|: an error x of the scores
  moves out by 2 x A at most (numerator and denominator); exponentials and
  sums over n keys add (n + 16) 2^-24 A, the fp32 output rounding 2^-24 |out|.
"""

import numpy as np


def attend(q, k, v, scale):
    """q [R, D], k / v [n, D] in float64 -> out [R, D], bounds for bf16 and fp32 (same shape)."""
    D, n = q.shape[1], k.shape[0]
    s = q @ k.T * scale
    with np.errstate(invalid="ignore"):
        w = np.exp(s - s.max(axis=1, keepdims=True))
    w /= w.sum(axis=1, keepdims=True)
    out, A = w @ v, w @ np.abs(v)
    ds = ((D + 2) * 2.0 ** -24 * (np.abs(q) @ np.abs(k).T).max(axis=1) * abs(scale)
          + 2.0 ** -22 * np.abs(s).max(axis=1))[:, None]
    f32 = (2 * ds + (n + 16) * 2.0 ** -24) * A + 2.0 ** -24 * np.abs(out)
    return out, f32 + 2.0 ** -8 * (A + np.abs(out)), f32
