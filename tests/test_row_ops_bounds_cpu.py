"""Refusals of the language-model row operators at the bounds of their arguments' types, which come
before any device is touched: with tensors of no memory, or on the host."""
import pytest
import torch

from hephaestus_b200 import InvalidConfiguration
from hephaestus_b200 import torch_ops as T


def refused(message, call, *args, **kw):
    with pytest.raises(InvalidConfiguration) as e:
        call(*args, **kw)
    assert message in e.value.message, e.value.message


def test_sizes_past_32_bits():
    """No size is taken for what its low 32 bits say."""
    def wide(cols, dtype):
        return torch.empty(1, cols, dtype=dtype, device="meta")
    past = 2 ** 32 + 8
    g, p = torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.int32)
    refused(f"2 of {past}", T.route_experts_backward, g, wide(past, torch.bfloat16), p)
    refused(f"{past} of 8", T.route_experts_backward, wide(past, torch.float32), torch.zeros(1, 8), wide(past, torch.int32))
    refused("chooses 1 to 32", T.route_experts_backward, torch.zeros(1, 0), torch.zeros(1, 8), p[:, :0])
    refused(f"2 of {past}", T.route_experts, wide(past, torch.bfloat16), 2)
    refused("1 to 1024", T.expert_order, p, past)
    refused("[rows, vocabulary]", T.sample_tokens, wide(past, torch.bfloat16), torch.zeros(1))
