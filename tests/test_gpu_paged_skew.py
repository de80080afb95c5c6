"""Paged decode where one sequence holds nearly all of the batch's keys, and so
nearly all of its shares: hundreds of partials of one sequence are joined beside
sequences of one."""

import numpy as np
import pytest
import torch

import sparda
from test_gpu_paged import BF, DEV, F32, cache, check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("B,Hq,Hkv,D,at", [(16, 12, 4, 64, 0), (32, 12, 4, 64, 31), (6, 8, 2, 128, 3), (32, 6, 2, 16, 7),
                                           (16, 6, 3, 32, 15)])
def test_one_long_sequence_among_short_ones(dtype, B, Hq, Hkv, D, at):
    print(f"[case] paged skew {dtype} {B} {Hq}/{Hkv}x{D} at={at}", flush=True)
    r = np.random.default_rng(B + D)
    lengths = [int(x) for x in r.integers(0, 300, B)]
    lengths[at], lengths[at - 1] = 20011, 0
    kp, vp, table, ks, vs = cache(lengths, 32, Hkv, D, dtype, seed=B, width=2048)
    q = queries(B, Hq, D, dtype, seed=17) * 2
    args = [x.to(DEV) for x in (q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32))]
    sparda.status()
    got = sparda.decode_paged(*args)
    check(got, q, ks, vs)
    assert torch.equal(got, sparda.decode_paged(*args)) and sparda.status() == 0
