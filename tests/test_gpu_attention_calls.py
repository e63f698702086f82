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


@pytest.mark.parametrize("prefix", [0, 20])
def test_a_layer_of_no_tokens(hip, cache, prefix):
    from spoc_amd.attention import MxAttention
    random = lambda *shape: hip.mx_quantize(torch.randn(*shape, device="cuda"), "fp4")  # noqa: E731
    layer = MxAttention(torch.ones(256, dtype=torch.bfloat16, device="cuda"), random(8 * 64, 256), random(256, 4 * 64), 4, 2, hip.Rotary(64))
    none = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    shared = (ints(2, 3), prefix) if prefix else None
    for more in (dict(starts=ints(0, 0)), dict(starts=ints(0, 0), residual=none)):
        y, h = layer(none, cache, ints([0]), ints(5), prefix=shared, **more)
        assert y.shape == h.shape == (0, 256) and y.dtype == h.dtype == torch.bfloat16
    y, h = layer(none, cache, torch.empty(0, 1, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), prefix=shared)
    assert y.shape == h.shape == (0, 256) and (cache.keys == 0).all() and (cache.values == 0).all()


def test_a_place_for_q_without_a_q_is_refused(hip, cache):
    with pytest.raises(ValueError):
        hip.kv_append(heads(n=2), heads(n=2), cache, ints([0, 1], [2, 3]), ints(5, 6), q_out=heads())
    assert (cache.keys == 0).all()
    assert hip.kv_append(heads(n=2), heads(n=2), cache, ints([0, 1], [2, 3]), ints(5, 6)) is None
