"""Infinite and undefined values among those that every row sees: they are in the sums of their own columns and in nothing else."""
import math

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,heads,kv_heads", [(64, 4, 2), (128, 8, 2), (200, 2, 2)])
@pytest.mark.parametrize("tokens,causal", [(1, True), (3, False), (60, False)])
@pytest.mark.parametrize("prefix", [0, 64])
def test_seen_by_all(hip, torch_cuda, dtype, d, heads, kv_heads, tokens, causal, prefix):
    """Queries are small, so that every weight is near the others and none of them 0 in the type."""
    gen, n, page = torch.Generator().manual_seed(d + tokens), 333, 16
    pages = torch.randperm(30, generator=gen).int().cuda()
    cache = hip.KvCache(*(torch.randn(30, page, kv_heads, d, generator=gen).to(dtype).cuda() for _ in range(2)))
    before, own = pages[:prefix // page], pages[prefix // page:][None]
    for at, column, value in ((0, 1, math.inf), (100, 2, -math.inf), (n - 1, 3, math.inf), (170, 4, math.nan), (31, 5, math.inf), (299, 5, math.inf),
                              (40, 6, math.inf), (200, 6, -math.inf)):
        cache.values[own[0, at // page].long(), at % page, 0, column] = value
    if prefix:
        cache.values[before[2].long(), 5, kv_heads - 1, 7] = -math.inf
    q = (0.2 * torch.randn(tokens, heads, d, generator=gen)).to(dtype).cuda()
    starts = ints(0, tokens)
    if prefix:
        got = hip.attention_shared(q, cache, before, prefix, own, ints(n), starts=starts, causal=causal)
    else:
        got = hip.attention_paged(q, cache, own, ints(n), starts=starts, causal=causal)
    want, tol, _, _ = ref.attention(q, cache.keys, cache.values, own, [n], [0, tokens], causal, prefix=before, prefix_length=prefix)
    same, worst = ref.compare(got, want, tol)
    assert torch.isinf(want[:, 0, [1, 2, 3, 5]]).all() and torch.isnan(want[:, 0, [4, 6]]).all()
    assert same and worst <= 1, (same, worst)
