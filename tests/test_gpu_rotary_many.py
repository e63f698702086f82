"""Rotary positions and appending of so much that a thread takes four heads: groups of heads that are not whole, heads whose pairs and
whose values behind them are not whole pieces."""
import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MANY = 1 << 19      # pieces of a head, 8 pairs or 16 values behind them, from which a thread takes four heads


def pieces(d, dim):
    return -(-(dim // 2) // 8) + -(-(d - dim) // 16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,d,dim", [(6000, 33, 50, 38), (30000, 6, 64, 64), (20000, 7, 80, 40), (140000, 4, 16, 10), (4099, 41, 128, 6)])
def test_rotary(hip, torch_cuda, dtype, layout, tokens, heads, d, dim):
    assert tokens * heads * pieces(d, dim) >= MANY
    gen = torch.Generator(device="cuda")
    gen.manual_seed(tokens + d)
    t = TYPES[dtype]
    x = torch.randn(tokens, heads, d + 3, generator=gen, device="cuda").to(t)[..., :d]
    positions = torch.randint(-5, 1 << 20, (tokens,), generator=gen, device="cuda")
    plan = hip.Rotary(dim, layout=layout, amplitude=1.25)
    for inverse, call in ((False, hip.rotary), (True, hip.rotary_backward)):
        block = torch.full((tokens, heads + 1, d + 5), 7.0, dtype=t, device="cuda")
        got = call(x, positions, plan, out=block[:, :heads, :d])
        off = (got.double() - ref.rotate(x, positions, plan.frequencies, layout, 1.25, inverse)).abs()
        assert (off <= ref.rotate_tolerance(x, dim // 2, layout, 1.25)).all()
        assert torch.equal(got[..., dim:], x[..., dim:])
        assert (block[:, heads] == 7).all() and (block[..., d:] == 7).all()      # (nothing past the last head, or past a head's end)
        mine = x.clone()
        assert call(mine, positions, plan, out=mine) is mine and torch.equal(mine, got)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv_heads,d,dim,tokens", [(10, 5, 72, 38, 9000), (7, 2, 64, 64, 20000), (9, 6, 128, 12, 7000), (0, 5, 80, 80, 30000), (13, 13, 80, 0, 9000)])
def test_append(hip, torch_cuda, dtype, layout, heads, kv_heads, d, dim, tokens):
    each = pieces(d, dim) if dim else -(-d // 16)
    assert tokens * (heads + kv_heads) * each >= MANY
    gen = torch.Generator(device="cuda")
    gen.manual_seed(tokens + d)
    t, page, before = TYPES[dtype], 48, [5, 0, 1000]
    news = [tokens // 3, 1, tokens - tokens // 3 - 1]
    lengths, starts = [a + b for a, b in zip(before, news)], [0, news[0], news[0] + 1, tokens]
    held = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(held) + 2, generator=gen, device="cuda").int()
    pages = torch.full((3, max(held)), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(held):
        pages[b, :n] = order[sum(held[:b]):sum(held[:b + 1])]
    cache = hip.KvCache(*(torch.full((len(order), kv_heads, page, d), 5.0, dtype=t, device="cuda").transpose(1, 2) for _ in range(2)))
    random = lambda n: torch.randn(tokens + 2, n, d + 8, generator=gen, device="cuda").to(t)[..., :d]  # noqa: E731
    k, v, q = random(kv_heads), random(kv_heads), random(heads) if heads else None
    q_out = torch.full_like(q, 7.0) if heads else None
    plan = hip.Rotary(dim, layout=layout) if dim else None
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    assert hip.kv_append(k, v, cache, pages, ints(lengths), starts=ints(starts), rotary=plan, q=q, q_out=q_out, first=3) is q_out
    keys, values, tol = torch.full_like(cache.keys, 5.0).double(), torch.full_like(cache.values, 5.0), torch.zeros_like(cache.keys).double()

    def turned(x, at):
        if not dim:
            return x.double(), torch.zeros_like(x).double()
        return ref.rotate(x, at + 3, plan.frequencies, layout), ref.rotate_tolerance(x, dim // 2, layout, 1.0)

    for b, n in enumerate(lengths):
        mine, at = slice(starts[b], starts[b + 1]), torch.arange(n - news[b], n, device="cuda")
        where = pages[b].long()[at // page], at % page
        values[where] = v[mine]
        keys[where], tol[where] = turned(k[mine], at)
        if heads:
            want, bound = turned(q[mine], at)
            assert ((q_out[mine].double() - want).abs() <= bound).all()
    assert torch.equal(cache.values, values) and ((cache.keys.double() - keys).abs() <= tol).all()
    if heads:
        assert (q_out[tokens:] == 7).all()
        assert hip.kv_append(k, v, cache, pages, ints(lengths), starts=ints(starts), rotary=plan, q=q, q_out=q, first=3) is q
        assert torch.equal(q[:tokens], q_out[:tokens])
