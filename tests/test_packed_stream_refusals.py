"""Budgets that PackedStreamDecoder refuses before it makes anything, without a GPU."""
import pytest

from infllm_b200.utils import PackedStreamDecoder

SHAPE = dict(n_layers=1, hidden=64, n_heads=1, n_kv_heads=1, head_dim=64, ffn=64, vocab=16, max_tokens=64)


@pytest.mark.parametrize("more", [dict(budget=10, sink=-1), dict(budget=10, sink=4, recent=-2), dict(budget=10, sink=-5, recent=12),
                                  dict(budget=10, sink=5, recent=6), dict(budget=-1), dict(budget=40, slack=24), dict(budget=40, slack=-1)])
def test_budgets_that_no_eviction_takes(more):
    with pytest.raises(ValueError):
        PackedStreamDecoder(**SHAPE, **more)
