"""The limits of q4_accuracy would show a fault: what a lost share, a lost last key, and a split with one
term instead of three do to the output, on the CPU."""

import numpy as np
import pytest

from q4_accuracy import LIMIT, aligned_queries, attend64, relative
from q4_oracle import bf16, held


def inputs(n, D, H, seed=1):
    g = np.random.default_rng(seed)
    k, v = (held(g.standard_normal((n, D))) for _ in range(2))
    return bf16(g.standard_normal((H, D)) * 2).astype(np.float64), k, v


@pytest.mark.parametrize("n", [33, 1000, 9000, 20011])
@pytest.mark.parametrize("D", [16, 64, 128])
def test_a_lost_share_or_key_is_seen(n, D):
    q, k, v = inputs(n, D, 4)
    scale = D ** -0.5
    want = attend64(q, k, v, scale)
    for lost in (slice(0, 128), slice(n - 128 if n > 256 else n // 2, n), slice(n // 2, n // 2 + 128)):
        keep = np.ones(n, bool)
        keep[lost] = False
        if keep.any():
            assert relative(attend64(q, k, v, scale, keep).ravel(), want.ravel()) > LIMIT["bf16"]
    # the last key, where it holds weight
    q = aligned_queries(k, [n - 1], scale)
    keep = np.ones(n, bool)
    keep[n - 1] = False
    assert relative(attend64(q, k, v, scale, keep).ravel(), attend64(q, k, v, scale).ravel()) > LIMIT["bf16"]


@pytest.mark.parametrize("n", [33, 1000, 20011])
@pytest.mark.parametrize("D", [16, 64, 128])
def test_a_split_of_one_term_is_seen(n, D):
    """q and the weights rounded to bf16 once, as bf16 calls have it: outside the fp32 limit, and in the bf16 one."""
    q, k, v = inputs(n, D, 4)
    scale = D ** -0.5
    q = q * (1 + 2.0 ** -9)                                       # not bf16 values
    want = attend64(q, k, v, scale)
    s = bf16(q).astype(np.float64) @ k.T * scale
    assert relative((lambda w: w / w.sum(1, keepdims=True) @ v)(np.exp(s - s.max(1, keepdims=True))).ravel(), want.ravel()) > LIMIT["f32"]
    s = q @ k.T * scale
    w = np.exp(s - s.max(1, keepdims=True))
    out = bf16(bf16(w).astype(np.float64) @ v / w.sum(1, keepdims=True))
    assert LIMIT["f32"] < relative(out.ravel(), want.ravel()) < LIMIT["bf16"]
