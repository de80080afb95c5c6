"""Where rows of one forward may judge drafts: the attention backends' own statement."""

import pytest

from model.config import ModelConfig
from model.model import SparDAResearchModel


def model(backend, n_layer=2, block=16, top_k=4):
    return SparDAResearchModel(ModelConfig(vocab_size=64, n_layer=n_layer, n_embd=64, n_head=2, n_kv_head=1, head_dim=32, ffn_dim=64,
                                           forecast_heads=1, forecast_dim=32, context_length=64, block_size=block,
                                           top_k_blocks=top_k, attention_backend=backend))


@pytest.mark.parametrize("backend,holds,fails", [
    ("hip_sparse", [1, 32, 64], [65, 80, 8192, 8193]),        # 4 blocks of 16, all of them chosen
    ("static", [1, 65, 8192], [8193]),
    ("dense", [1, 8193, 1 << 20], []),
    ("offload", [1, 8193], []),
    ("async_offload", [1, 8193], []),
])
def test_lengths_up_to_which_no_row_depends_on_a_later_token(backend, holds, fails):
    m = model(backend)
    assert all(m.rows_ignore_later(n) for n in holds) and not any(m.rows_ignore_later(n) for n in fails)


def test_two_blocks_and_the_first_layer_are_dense():
    m = model("hip_sparse", top_k=1)
    assert m.rows_ignore_later(32) and not m.rows_ignore_later(33)
    assert model("hip_sparse", n_layer=1, top_k=1).rows_ignore_later(8192)
    assert not model("hip_sparse", n_layer=1, top_k=1).rows_ignore_later(8193)
