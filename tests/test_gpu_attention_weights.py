"""How exactly attention holds the softmax's weights for the product with the values: bounds by element and by norm that a kernel which
rounds them once more than it says would not pass.

With p the weights relative to a row's largest, S their sum, and h = eps / 2 of the type, the largest error of a rounding, relative to the value:
  few rows (up to 16 to a sequence): a weight is two parts of the type, the first below it by up to 2 h of it and the second what is left, rounded: off by
  2 h^2 of itself;
  tiles of rows: it is rounded to the type once, off by h of itself;
  fp16: besides by 2^-32 of the largest at most, half of the smallest step 2^-24 of weights that are held 2^7 times as large.
The queries and keys are such that scores are exact sums: an exponent's argument is then off by 2^-24 of itself for the scale and for the product each, the
exponential and that of a join by 2^-22, 2^-21 (1 + |argument|) in all of the weight; sums of n terms by n 2^-24 of what they sum, and the division by 2^-22.  Then o
is rounded, by h of itself or half of fp16's smallest step."""
import math

import pytest
import torch

import attention_reference as ref

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def exactly(q, k, v, seen, scale, parts):
    """(o, bound of o, o's bound without its own rounding, the mean square that weights rounded at random add), all in float64, of q [rows, d]
    over k and v [n, d]; seen [rows, n]; parts: of which a weight is made."""
    h, n = torch.finfo(q.dtype).eps / 2, k.shape[0]
    x, y, v = q.double(), k.double(), v.double()
    s = torch.where(seen, x @ y.t() * scale, -math.inf)
    p = torch.where(seen, torch.exp(s - s.amax(1, keepdim=True)), 0.0)
    total = p.sum(1, keepdim=True)
    o, size = p @ v / total, p @ v.abs() / total
    exponent = torch.where(p > 0, p * 2.0 ** -21 * (1 + torch.where(p > 0, s.amax(1, keepdim=True) - s, 0.0)), 0.0)
    rest = (p * (2 * h * h if parts == 2 else h) + exponent) @ v.abs() / total + o.abs() * (exponent.sum(1, keepdim=True) / total + 2.0 ** -22) + (size + o.abs()) * n * 2.0 ** -24
    if q.dtype == torch.float16:
        rest = rest + 2.0 ** -32 * (seen.double() @ v.abs()) / total
    own = h * o.abs() + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    # (a weight's error is even over a step at random: h / sqrt(3) of it in the mean square, or less)
    return o, own + rest * (1 + h), rest, (p * p) @ (v * v) / total ** 2 * h * h / 3


def check(got, q, k, v, seen, scale, parts, alike=False):
    """got [tokens, heads, d] of q like it, k and v [n, kv_heads, d], by element and by norm; alike: many weights are equal, and so their errors."""
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    square = torch.zeros(5, dtype=torch.float64, device=q.device)
    for head in range(heads):
        o, bound, rest, random = exactly(q[:, head], k[:, head // group], v[:, head // group], seen, scale, parts)
        off = (got[:, head].double() - o).abs()
        assert (off <= bound).all(), f"head {head}: {float((off / bound).max()):.3f} of the bound"
        rounded = o.to(q.dtype).double() - o
        square += torch.stack([t.pow(2).sum() for t in (off, rounded, rest)] + [random.sum(), o.pow(2).sum()])
    if alike and parts == 1:
        return
    off, rounded, rest, random, size = square.tolist()
    # Roundings that do not know of each other add up by their squares; a tenth for what some thousands of them differ from their mean.
    most = 1.1 * math.sqrt(rounded + (random if parts == 1 else 0.0)) + math.sqrt(rest if parts == 2 else 0.0)
    assert math.sqrt(off) <= most, f"{math.sqrt(off / size):.6f} of the norm, {most / math.sqrt(size):.6f} expected"


def exact_queries(gen, *shape):
    """Multiples of a half up to 4; products with the keys below are multiples of 2^-4, sums of 256 of them below 2^16."""
    return torch.randint(-8, 9, shape, generator=gen) / 2


def exact_keys(gen, *shape):
    return torch.randint(-16, 17, shape, generator=gen) / 8


def made(hip, gen, dtype, n, heads, kv_heads, d, tokens, page=16):
    """A cache with one sequence of n keys in pages in no order, and queries for its last tokens."""
    count = -(-n // page)
    pages = torch.randperm(count, generator=gen).int()[None].cuda()
    cache = hip.KvCache(exact_keys(gen, count, page, kv_heads, d).to(dtype).cuda(), torch.randn(count, page, kv_heads, d, generator=gen).to(dtype).cuda())
    q = exact_queries(gen, tokens, heads, d).to(dtype).cuda()
    return cache, pages, q, ref.gather(cache.keys, pages[0], n), ref.gather(cache.values, pages[0], n)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def causal(tokens, n, device="cuda"):
    return torch.arange(n, device=device)[None] <= torch.arange(n - tokens, n, device=device)[:, None]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,kv_heads,n", [(64, 4, 4, 300), (128, 8, 2, 130), (80, 6, 3, 77), (256, 4, 1, 200), (64, 8, 8, 4000), (128, 4, 4, 33)])
def test_few_rows(hip, torch_cuda, dtype, d, heads, kv_heads, n):
    cache, pages, q, k, v = made(hip, torch.Generator().manual_seed(d + n), TYPES[dtype], n, heads, kv_heads, d, 4)
    got = hip.attention_paged(q, cache, pages, ints(n), starts=ints(0, 4))
    check(got, q, k, v, causal(4, n), d ** -0.5, 2)
    got = hip.attention_paged(q[3:], cache, pages, ints(n))
    check(got, q[3:], k, v, causal(1, n), d ** -0.5, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,kv_heads,n,tokens", [(64, 4, 4, 300, 100), (128, 8, 2, 500, 70), (80, 6, 3, 77, 77), (256, 4, 1, 200, 50), (64, 8, 2, 3000, 40)])
def test_tiles(hip, torch_cuda, dtype, d, heads, kv_heads, n, tokens):
    cache, pages, q, k, v = made(hip, torch.Generator().manual_seed(d + n), TYPES[dtype], n, heads, kv_heads, d, tokens)
    got = hip.attention_paged(q, cache, pages, ints(n), starts=ints(0, tokens))
    check(got, q, k, v, causal(tokens, n), d ** -0.5, 1)


@pytest.fixture
def uncut(hip, request):
    """Keys in one stretch, as in a batch that fills the card by itself, or cut, which keeps small weights apart from a large one."""
    if request.param:
        hip.set_tunable("attention.stream_workgroups", 0)
        hip.set_tunable("attention.tile_workgroups", 0)
    yield
    hip.set_tunable("attention.stream_workgroups", 512)
    hip.set_tunable("attention.tile_workgroups", 512)


@pytest.mark.gpu
@pytest.mark.parametrize("uncut", [True, False], indirect=True)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("below,n", [(12, 3000), (14, 3000), (16, 8193), (18, 131072), (20, 131072)])
def test_one_key_far_above_the_others(hip, torch_cuda, uncut, dtype, tokens, below, n):
    """A key of value 0 `below` (natural logarithm) above thousands of others, whose values are all of the result: below fp16's least number by itself from 18 on."""
    t, d, gen = TYPES[dtype], 64, torch.Generator().manual_seed(below)
    cache, pages, _, _, _ = made(hip, gen, t, n, 1, 1, d, 1, page=64)
    at = int(torch.randint(0, n, (1,), generator=gen))
    cache.keys.zero_()
    cache.values.copy_(cache.values.abs())
    where = pages[0, at // 64].long(), at % 64
    cache.keys[where], cache.values[where] = below / 8, 0.0      # (64 products of 1 and below / 8, by 8: exact)
    q, lse = torch.ones(tokens, 2, d, dtype=t, device="cuda"), torch.empty(tokens, 2, device="cuda")
    got = hip.attention_paged(q, cache, pages, ints(n), starts=ints(0, tokens), causal=False, lse=lse)
    k, v = ref.gather(cache.keys, pages[0], n), ref.gather(cache.values, pages[0], n)
    check(got, q, k, v, torch.ones(tokens, n, dtype=torch.bool, device="cuda"), d ** -0.5, 2 if tokens == 1 else 1, alike=True)
    want = below + math.log1p((n - 1) * math.exp(-below))
    assert (lse.double() - want).abs().max() <= n * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * want


@pytest.mark.gpu
@pytest.mark.parametrize("uncut", [True, False], indirect=True)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 40])
def test_behind_a_prefix(hip, torch_cuda, uncut, dtype, tokens):
    """The key far above is in the prefix, the others are a sequence's own, and the other way round: the planes' maxima are those of the weights."""
    t, d, n, prefix, gen = TYPES[dtype], 64, 4000, 96, torch.Generator().manual_seed(tokens)
    cache, pages, _, _, _ = made(hip, gen, t, n + prefix, 2, 1, d, 1)
    cache.keys.zero_()
    cache.values.copy_(cache.values.abs())
    q = torch.ones(tokens, 2, d, dtype=t, device="cuda")
    for at in (50, 2000):
        where = pages[0, at // 16].long(), at % 16
        cache.keys[where] = 2.0
        got = hip.attention_shared(q, cache, pages[0, :prefix // 16].contiguous(), prefix, pages[:, prefix // 16:].contiguous(), ints(n), starts=ints(0, tokens), causal=False)
        k, v = ref.gather(cache.keys, pages[0], n + prefix), ref.gather(cache.values, pages[0], n + prefix)
        # (the rows of all sequences are together before the prefix: two of them go by few rows, 80 by tiles)
        check(got, q, k, v, torch.ones(tokens, n + prefix, dtype=torch.bool, device="cuda"), d ** -0.5, 2 if tokens == 1 else 1, alike=True)
        cache.keys[where] = 0.0


def rounded_weights(q, k, v, scale, parts, raised):
    """The formula with weights of the type, in float64 otherwise."""
    x = torch.exp(q.double() @ k.double().t() * scale)
    x = x / x.amax(1, keepdim=True)
    held = (x * 2.0 ** raised).to(q.dtype).double()
    if parts == 2:
        held = torch.where(held < x * 2.0 ** raised, held, (held * (1 - torch.finfo(q.dtype).eps)).to(q.dtype).double())
        held = held + (x * 2.0 ** raised - held).to(q.dtype).double()
    return (held @ v.double() / 2.0 ** raised / x.sum(1, keepdim=True)).to(q.dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_bounds_tell_roundings_apart(dtype):
    """On the CPU: two parts pass as two, one part as one and not as two; without the 2^7 fp16 does not pass."""
    t, gen, n, d = TYPES[dtype], torch.Generator().manual_seed(3), 130, 64
    q, k, v = exact_queries(gen, 8, d).to(t), exact_keys(gen, n, d).to(t), torch.randn(n, d, generator=gen).to(t)
    seen = torch.ones(8, n, dtype=torch.bool)

    def passes(q, k, v, seen, parts, raised, as_parts, alike=False):
        got = rounded_weights(q, k, v, d ** -0.5, parts, raised)
        try:
            check(got[:, None], q[:, None], k[:, None], v[:, None], seen, d ** -0.5, as_parts, alike)
        except AssertionError:
            return False
        return True

    assert passes(q, k, v, seen, 2, 7, 2) and passes(q, k, v, seen, 1, 7, 1) and not passes(q, k, v, seen, 1, 7, 2)
    for below, n in ((16, 8193), (18, 131072)):
        k, v = torch.zeros(n, d), torch.randn(n, d, generator=gen).abs()
        k[77], v[77] = below / 8, 0.0
        for parts in (1, 2):
            args = torch.ones(1, d, dtype=t), k.to(t), v.to(t), torch.ones(1, n, dtype=torch.bool), parts
            assert passes(*args, 7, parts, True) and passes(*args, 0, parts, True) == (dtype == "bf16")
