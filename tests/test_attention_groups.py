"""The layer's decode where groups are named and nothing is shared."""

import pytest
import torch

from microserve_amd import attention as layer
from tests.test_attention_more import _layer, _step, calls  # noqa: F401


@pytest.mark.parametrize("dtype,name", [("fp8_e4m3", "fp8_decode_attention"),
                                        ("fp4_e2m1", "fp4_decode_attention")])
def test_a_bound_of_zero_is_the_plain_decode(calls, monkeypatch, dtype, name):  # noqa: F811
    monkeypatch.setattr(layer, "fp4_decode_attention",
                        lambda *a: calls.append(("fp4_decode_attention", a)) or torch.zeros(1))
    groups = dict(cu_groups=torch.tensor([0, 3], dtype=torch.int32),
                  prefix_lens=torch.zeros(1, dtype=torch.int32))
    _step(_layer(dtype), **groups, max_prefix_len=0)
    assert calls[-1][0] == name
    attn = _layer()
    _step(attn, **groups, max_prefix_len=128)
    assert calls[-1][0] == "fp8_shared_prefix_decode_attention"
    attn.attention_weights = torch.zeros(4, 2, 128)
    _step(attn, **groups, max_prefix_len=0)
    assert calls[-1][0] == "fp8_decode_attention_weights"
