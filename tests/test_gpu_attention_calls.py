"""Calls of the operators on a paged cache that are refused, or served, as their documentation says."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.fixture
def cache(hip, torch_cuda):
    return hip.KvCache(*(torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)))


def heads(tokens=2, n=4):
    return torch.ones(tokens, n, 64, dtype=torch.bfloat16, device="cuda")


@pytest.mark.parametrize("length", [0, 20])
def test_a_prefix_without_pages_is_refused(hip, cache, length):
    with pytest.raises(TypeError):
        hip.attention_shared(heads(), cache, None, length, ints([0, 1], [2, 3]), ints(5, 6))
