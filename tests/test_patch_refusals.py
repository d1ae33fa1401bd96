"""What patch_hf refuses, without a GPU."""
import types

import pytest

from infllm_b200.utils import patch_hf


@pytest.mark.parametrize("attn_type", ["paged", "packed"])
def test_types_that_need_a_batch_are_refused_when_a_model_is_patched(attn_type):
    """Not at its first forward: and the model is as it was."""
    attention = types.SimpleNamespace(forward=len)
    config = types.SimpleNamespace(hidden_size=128, num_attention_heads=2, num_key_value_heads=2)
    model = types.SimpleNamespace(layers=[types.SimpleNamespace(self_attn=attention)], config=config)
    with pytest.raises(ValueError, match="batch"):
        patch_hf(model, attn_type, base=1e4)
    assert attention.forward is len and not hasattr(attention, "_infllm_past") and not hasattr(model, "infllm_reset")
