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


def test_out_in_the_memory_of_q_in_another_order_is_refused(hip, cache):
    """Rows would be written that others are still read from.  The same memory in the same order is q itself."""
    block = torch.ones(4 * 4 * 64, dtype=torch.bfloat16, device="cuda")
    q, out = block.view(4, 4, 64), block.view(4, 4, 64).transpose(0, 1)
    pages, lengths = ints([0], [1], [2], [3]), ints(5, 6, 7, 8)
    for call in (lambda out: hip.attention_paged(q, cache, pages, lengths, out=out), lambda out: hip.attention_shared(q, cache, ints(3), 7, pages, lengths, out=out)):
        with pytest.raises(hip.SarekHipError, match="other strides"):
            call(out)
        assert call(q.view(4, 4, 64)) is not None
