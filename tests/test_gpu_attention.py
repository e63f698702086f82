"""Rotary positions, the paged cache and attention over it against float64."""
import math
import random

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def table(lengths, page, gen, spare=3, more=0, prefix=0):
    """(page table on the device, prefix pages, pages in all): every page a place of its own, in no order."""
    held = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(held) + spare + prefix, generator=gen)
    pages = torch.full((len(lengths), max(held + [0]) + more), -1, dtype=torch.int32)
    at = prefix
    for b, n in enumerate(held):
        pages[b, :n] = order[at:at + n].int()
        at += n
    return pages.cuda(), order[:prefix].int().cuda(), len(order)


def cache_of(hip, pages, page, heads, d, dtype, layout="plain", fill=math.nan):
    """A KvCache whose unused places hold `fill`."""
    if layout == "plain":
        keys, values = (torch.full((pages, page, heads, d), fill, dtype=dtype, device="cuda") for _ in range(2))
    elif layout == "heads first":
        keys, values = (torch.full((pages, heads, page, d), fill, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
    elif layout == "one block":
        block = torch.full((pages, 2, page, heads, d + 8), fill, dtype=dtype, device="cuda")
        keys, values = block[:, 0, ..., :d], block[:, 1, ..., :d]
    else:
        keys, values = (torch.full((heads, pages, page, d), fill, dtype=dtype, device="cuda").permute(1, 2, 0, 3) for _ in range(2))
    return hip.KvCache(keys, values)


def fill(cache, pages, lengths, gen, key=1.0):
    """Random keys and values in the places that the sequences hold."""
    size, pages = cache.page_size, pages.cpu()
    for b, n in enumerate(lengths):
        at = torch.arange(n)
        where = pages[b].long()[at // size].cuda(), (at % size).cuda()
        for t, std in ((cache.keys, key), (cache.values, 1.0)):
            t[where] = (torch.randn(n, cache.heads, cache.head_dim, generator=gen) * std).to(t.dtype).cuda()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def queries(gen, tokens, heads, d, dtype, std=2.0, apart=0):
    q = (torch.randn(tokens, heads + (1 if apart else 0), d + apart, generator=gen) * std).to(dtype).cuda()
    return q[:, :heads, :d]


def run(hip, gen, dtype, d, heads, kv_heads, page, lengths, news=None, causal=True, layout="plain", apart=0, prefix=0, std=2.0, pad=0, scale=None):
    """One call against the reference; tokens behind the last sequence keep what they held."""
    dtype = TYPES[dtype]
    pages, prefix_pages, n = table(lengths, page, gen, prefix=-(-prefix // page), more=1)
    cache = cache_of(hip, n, page, kv_heads, d, dtype, layout)
    fill(cache, pages, lengths, gen)
    fill(cache, prefix_pages[None], [prefix], gen)
    starts = None if news is None else [sum(news[:b]) for b in range(len(news) + 1)]
    tokens = len(lengths) if news is None else starts[-1]
    q = queries(gen, tokens + pad, heads, d, dtype, std, apart)
    out = torch.full((tokens + pad, heads, d + apart), 7.0, dtype=dtype, device="cuda")[..., :d]
    lse = torch.full((tokens + pad, heads), 7.0, device="cuda")
    more = dict(starts=None if starts is None else ints(starts), causal=causal, scale=scale, out=out, lse=lse)
    if prefix:
        got = hip.attention_shared(q, cache, prefix_pages, prefix, pages, ints(lengths), **more)
    else:
        got = hip.attention_paged(q, cache, pages, ints(lengths), **more)
    assert got is out
    want, tol, want_lse, lse_tol = ref.attention(q[:tokens], cache.keys, cache.values, pages, lengths, starts, causal, scale, prefix_pages, prefix)
    for name, g, w, t in (("out", out[:tokens], want, tol), ("lse", lse[:tokens], want_lse, lse_tol)):
        same, worst = ref.compare(g, w, t)
        assert same and worst <= 1, f"{name}: {worst:.3f} of the tolerance, {same}"
    assert (out[tokens:] == 7).all() and (lse[tokens:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,d,dim", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 80, 40), (7, 3, 50, 38), (61, 13, 72, 72), (2500, 33, 64, 48), (0, 4, 64, 64)])
def test_rotary(hip, torch_cuda, dtype, layout, tokens, heads, d, dim):
    gen = torch.Generator().manual_seed(tokens * 31 + d)
    x = torch.randn(tokens, heads, d + 3, generator=gen).to(TYPES[dtype]).cuda()[..., :d]
    positions = torch.randint(-5, 1 << 20, (tokens,), generator=gen).cuda()
    plan = hip.Rotary(dim, layout=layout, amplitude=1.25)
    for inverse, call in ((False, hip.rotary), (True, hip.rotary_backward)):
        want = ref.rotate(x, positions, plan.frequencies, layout, 1.25, inverse)
        tol = ref.rotate_tolerance(x, dim // 2, layout, 1.25)
        got = call(x, positions, plan)
        assert (got.double() - want).abs().sub(tol).max(dim=-1).values.le(0).all() if tokens else got.shape == x.shape
        assert torch.equal(got[..., dim:], x[..., dim:])
        mine = x.clone()
        assert call(mine, positions.int(), plan, out=mine) is mine
        assert torch.equal(mine, got)


def test_rotary_far_positions_and_scalings(hip, torch_cuda):
    x = torch.randn(6, 2, 64, generator=torch.Generator().manual_seed(0)).cuda()
    positions = torch.tensor([0, 1, 2 ** 31 - 1, 2 ** 31, 2 ** 40 + 1, -2 ** 33], device="cuda")
    for kw in (dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0), dict(scaling="ramp", factor=8.0),
               dict(frequencies=[2.0 ** -i for i in range(32)])):
        plan = hip.Rotary(64, **kw)
        # 2^-54 of the angle is what float64's product is off by itself (2^40 radians: 6e-5), so the angle is formed from exact parts
        f = plan.turns.cpu().tolist()
        t = torch.tensor([[(p * v % 2 ** 64) / 2 ** 64 * 2 * math.pi for v in f] for p in positions.tolist()], dtype=torch.float64)[:, None].cuda()
        a, b = x.double()[..., :32], x.double()[..., 32:]
        want = torch.cat((a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()), -1)
        assert ((hip.rotary(x, positions, plan).double() - want).abs() <= ref.rotate_tolerance(x, 32, "half", 1.0)).all()


def test_rotary_gradient_by_differences(hip, torch_cuda):
    """The turn is linear: the gradient of sum(rotary(x) dy) is what differences give, up to float32's roundings."""
    gen = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(5, 3, 24, generator=gen).cuda() for _ in range(2))
    positions, plan = torch.arange(100, 105).cuda(), hip.Rotary(16, layout="interleaved")
    dx = hip.rotary_backward(dy, positions, plan)
    for _ in range(10):
        step = torch.randn(5, 3, 24, generator=gen).cuda()
        change = (hip.rotary(x + step, positions, plan).double() - hip.rotary(x - step, positions, plan).double()).mul(dy.double()).sum() / 2
        size = (dy.abs().double() * (x.abs() + step.abs()).double()).sum()
        assert abs(float(change - (dx.double() * step.double()).sum())) <= 2.0 ** -20 * float(size)


def test_rotary_of_an_expanded_tensor(hip, torch_cuda):
    x = torch.randn(1, 1, 32, generator=torch.Generator().manual_seed(2)).cuda().expand(9, 4, 32)
    positions, plan = torch.arange(9).cuda(), hip.Rotary(32)
    assert torch.equal(hip.rotary(x, positions, plan), hip.rotary(x.contiguous(), positions, plan))
    with pytest.raises(hip.SarekHipError):
        hip.rotary(x.contiguous(), positions, plan, out=x)


@pytest.mark.parametrize("dtype,layout,d,dim,heads,kv_heads,page,lengths,news,rotary", [
    ("bf16", "plain", 128, 128, 32, 8, 16, [1, 17, 4000, 16], None, "half"),
    ("f16", "one block", 64, 32, 6, 3, 20, [5, 0, 41, 20, 77], [5, 0, 1, 20, 30], "interleaved"),
    ("bf16", "heads first", 80, 40, 4, 1, 1, [3, 9], [3, 2], "half"),
    ("f16", "heads outermost", 72, 72, 5, 5, 64, [700], [700], "interleaved"),
    ("bf16", "plain", 8, 8, 1, 1, 7, [100] * 70, None, "half"),
    ("bf16", "plain", 128, 0, 8, 8, 256, [3000, 513], [2999, 1], None)])
def test_append(hip, torch_cuda, dtype, layout, d, dim, heads, kv_heads, page, lengths, news, rotary):
    gen, t = torch.Generator().manual_seed(3), TYPES[dtype]
    pages, _, n = table(lengths, page, gen)
    cache = cache_of(hip, n, page, kv_heads, d, t, layout, fill=5.0)
    news = [1] * len(lengths) if news is None else news
    starts = [sum(news[:b]) for b in range(len(news) + 1)]
    pad = 2 if starts[-1] != len(lengths) else 0
    k, v = (torch.randn(starts[-1] + pad, kv_heads, d, generator=gen).to(t).cuda() for _ in range(2))
    q = queries(gen, starts[-1] + pad, heads, d, t, apart=5)
    q_out = torch.full_like(q, 7.0)
    plan = hip.Rotary(dim, layout=rotary) if rotary else None
    more = dict(starts=ints(starts) if pad else None, rotary=plan, first=11)
    got = hip.kv_append(k, v, cache, pages, ints(lengths), q=q, q_out=q_out, **more)
    assert got is q_out
    keys, values = torch.full_like(cache.keys, 5.0).double(), torch.full_like(cache.values, 5.0)
    key_tol = torch.zeros_like(keys)
    for b, length in enumerate(lengths):
        if not news[b]:
            continue
        mine, at = slice(starts[b], starts[b + 1]), torch.arange(length - news[b], length).cuda()
        where = pages[b].long()[at // page], at % page
        values[where] = v[mine]
        if plan is None:
            keys[where] = k[mine].double()
            assert torch.equal(q_out[mine], q[mine])
            continue
        keys[where] = ref.rotate(k[mine], at + 11, plan.frequencies, rotary)
        key_tol[where] = ref.rotate_tolerance(k[mine], dim // 2, rotary, 1.0)
        assert ((q_out[mine].double() - ref.rotate(q[mine], at + 11, plan.frequencies, rotary)).abs() <= ref.rotate_tolerance(q[mine], dim // 2, rotary, 1.0)).all()
    assert torch.equal(cache.values, values)
    assert ((cache.keys.double() - keys).abs() <= key_tol).all()
    assert (q_out[starts[-1]:] == 7).all()
    mine = q.clone()
    assert hip.kv_append(k, v, cache, pages, ints(lengths), q=mine, q_out=mine, **more) is mine
    assert torch.equal(mine[:starts[-1]], q_out[:starts[-1]]) and torch.equal(mine[starts[-1]:], q[starts[-1]:])
    assert hip.kv_append(k, v, cache, pages, ints(lengths), **more) is None


def test_append_leaves_out_what_has_no_place(hip, torch_cuda):
    """Entries that are no page, lengths past the table, and more tokens than keys: nothing else is written."""
    cache = cache_of(hip, 4, 8, 1, 64, torch.bfloat16, fill=5.0)
    k = torch.ones(12, 1, 64, dtype=torch.bfloat16, device="cuda")
    pages = ints([[0, -1], [4, 2 ** 31 - 1], [1, 2], [3, 3]])
    hip.kv_append(k, k, cache, pages, ints([9, 16, 17, 1]), starts=ints([0, 2, 6, 8, 12]))
    want = torch.full((4, 8), 5.0)
    want[0, 7] = want[2, 7] = want[3, 0] = 1.0
    assert torch.equal(cache.keys[:, :, 0, 0].float().cpu(), want) and torch.equal(cache.values[:, :, 0, 5].float().cpu(), want)
    hip.kv_append(k, k, cache, pages, ints([-5, 2 ** 31 - 1, 0, -2 ** 31]), starts=ints([0, 2, 6, 8, 12]))
    hip.kv_append(k, k, cache, ints([[], [], [], []]).view(4, 0), ints([1, 2, 3, 4]), starts=ints([0, 2, 6, 8, 12]))
    assert torch.equal(cache.keys[:, :, 0, 0].float().cpu(), want)


EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 0, 500]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [8, 40, 64, 80, 128, 136, 256])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 2), (16, 1), (40, 2)])
def test_single_tokens(hip, torch_cuda, dtype, d, heads, kv_heads):
    run(hip, torch.Generator().manual_seed(d + heads), dtype, d, heads, kv_heads, 16, EDGES)


@pytest.mark.parametrize("dtype,page,layout", [("bf16", 1, "plain"), ("f16", 7, "one block"), ("bf16", 33, "heads first"), ("f16", 64, "heads outermost"), ("bf16", 1000, "plain")])
def test_pages_and_layouts(hip, torch_cuda, dtype, page, layout):
    run(hip, torch.Generator().manual_seed(page), dtype, 64, 4, 2, page, EDGES, layout=layout, apart=3)
    run(hip, torch.Generator().manual_seed(page), dtype, 128, 4, 2, page, [200, 77, 0, 300], [200, 1, 0, 90], layout=layout, apart=3, pad=2)


@pytest.mark.parametrize("lengths", [[4095], [20000], [30000, 5, 0, 12345], [1] * 300, [70] * 129 + [9000]])
def test_long_and_many(hip, torch_cuda, lengths):
    run(hip, torch.Generator().manual_seed(7), "bf16", 128, 8, 2, 16, lengths)
    run(hip, torch.Generator().manual_seed(8), "f16", 64, 3, 3, 20, lengths, std=6.0)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,heads,kv_heads", [(64, 4, 1), (128, 4, 2), (80, 3, 3), (256, 2, 1), (128, 24, 1), (40, 7, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(hip, torch_cuda, dtype, d, heads, kv_heads, causal):
    gen = torch.Generator().manual_seed(d + heads)
    run(hip, gen, dtype, d, heads, kv_heads, 16, [300, 5, 64, 0, 129, 1, 31], [300, 2, 64, 0, 65, 1, 30], causal, pad=3)
    run(hip, gen, dtype, d, heads, kv_heads, 16, [513, 700], [3, 2], causal)
    run(hip, gen, dtype, d, heads, kv_heads, 16, [1000], [1000], causal)


def test_more_tokens_than_keys(hip, torch_cuda):
    """The tokens are the last of the keys: those before the first key see none."""
    gen = torch.Generator().manual_seed(4)
    for d in (64, 128):
        run(hip, gen, "bf16", d, 4, 2, 16, [5, 0, 40], [9, 3, 100])
        run(hip, gen, "f16", d, 4, 2, 16, [5, 0, 40], [9, 3, 100], causal=False)


@pytest.mark.parametrize("dtype,d,heads,kv_heads,lengths,news,prefix", [
    ("bf16", 128, 32, 8, [1, 17, 100, 0, 61], None, 1000), ("f16", 64, 4, 4, [3, 9, 61, 3], [3, 3, 3, 3], 1001),
    ("bf16", 80, 6, 2, [40] * 50, None, 3000), ("f16", 128, 2, 1, [300, 200], [300, 1], 33), ("bf16", 256, 8, 2, [1] * 20, None, 1),
    ("f16", 64, 3, 1, [5, 0, 2], [1, 2, 2], 64), ("bf16", 128, 8, 1, [20] * 200, None, 129)])
def test_shared_prefix(hip, torch_cuda, dtype, d, heads, kv_heads, lengths, news, prefix):
    gen = torch.Generator().manual_seed(prefix)
    run(hip, gen, dtype, d, heads, kv_heads, 16, lengths, news, prefix=prefix, pad=0 if news is None else 2)
    run(hip, gen, dtype, d, heads, kv_heads, 20, lengths, news, causal=False, prefix=prefix, scale=0.3)


@pytest.mark.parametrize("news", [None, [4, 2], [70, 200]])
def test_masked_places_take_no_part(hip, torch_cuda, news):
    """Infinite and undefined keys and values that some or all tokens do not see, beside tokens that do."""
    for dtype, bad in (("bf16", math.inf), ("f16", math.nan), ("bf16", -math.inf)):
        gen = torch.Generator().manual_seed(5)
        lengths, d = [130, 333], 64
        pages, _, n = table(lengths, 16, gen)
        cache = cache_of(hip, n, 16, 2, d, TYPES[dtype])
        fill(cache, pages, lengths, gen)
        counts = [1, 1] if news is None else news
        for b, length in enumerate(lengths):
            if counts[b] > 1:               # a value that only the last token sees, one that the later half does
                for at, column in ((length - 1, 3), (length - counts[b] // 2, 40)):
                    cache.values[pages[b, at // 16].long(), at % 16, 1, column] = bad
        starts = [0, counts[0], sum(counts)]
        q = queries(gen, sum(counts), 4, d, TYPES[dtype])
        got = hip.attention_paged(q, cache, pages, ints(lengths), starts=ints(starts))
        want, tol, _, _ = ref.attention(q, cache.keys, cache.values, pages, lengths, starts)
        same, worst = ref.compare(got, want, tol)
        assert same and worst <= 1, (worst, same)
        # and keys that the tokens before the last do not see
        for b, length in enumerate(lengths):
            if counts[b] > 1:
                cache.keys[pages[b, (length - 1) // 16].long(), (length - 1) % 16] = math.nan
        again = hip.attention_paged(q, cache, pages, ints(lengths), starts=ints(starts))
        for b in range(2):
            if counts[b] > 1:
                assert torch.equal(again[starts[b]:starts[b + 1] - 1].nan_to_num(9), got[starts[b]:starts[b + 1] - 1].nan_to_num(9))
                assert again[starts[b + 1] - 1].isnan().all()


def test_entries_that_are_no_page(hip, torch_cuda):
    gen = torch.Generator().manual_seed(6)
    cache = cache_of(hip, 4, 16, 2, 64, torch.bfloat16)
    pages = ints([[0, -1, 1], [2, 4, 3], [2 ** 31 - 1, -2 ** 31, 0]])
    for t in (cache.keys, cache.values):
        t.copy_(torch.randn(t.shape, generator=gen))
    for lengths, starts in (([48, 40, 33], None), ([48, 40, 33], [0, 20, 60, 90])):
        q = queries(gen, 3 if starts is None else 90, 4, 64, torch.bfloat16)
        got = hip.attention_paged(q, cache, pages, ints(lengths), starts=None if starts is None else ints(starts))
        want, tol, _, _ = ref.attention(q, cache.keys, cache.values, pages, lengths, starts)
        assert ref.compare(got, want, tol)[1] <= 1
    # lengths past the table see what it has; negative ones nothing
    got = hip.attention_paged(queries(gen, 3, 4, 64, torch.bfloat16), cache, pages, ints([2 ** 31 - 1, -1, -2 ** 31]))
    assert got[0].isfinite().all() and (got[1:] == 0).all()


def test_starts_that_do_not_fit_write_nothing_else(hip, torch_cuda):
    """Starts out of range or falling are bounded by the call's tokens."""
    gen = torch.Generator().manual_seed(9)
    cache = cache_of(hip, 8, 16, 2, 64, torch.bfloat16, fill=1.0)
    pages = ints([[0, 1], [2, 3], [4, 5]])
    block = torch.full((40, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    for starts in ([-5, 3, 1000, 2 ** 31 - 1], [0, 20, 4, 10], [2 ** 31 - 1, -2 ** 31, 5, 5], [0, 0, 0, 0]):
        for prefix in (0, 16):
            q = queries(gen, 20, 4, 64, torch.bfloat16)
            more = dict(starts=ints(starts), out=block[10:30])
            if prefix:
                hip.attention_shared(q, cache, ints([7]), prefix, pages, ints([30, 20, 10]), **more)
            else:
                hip.attention_paged(q, cache, pages, ints([30, 20, 10]), **more)
        k = torch.ones(20, 2, 64, dtype=torch.bfloat16, device="cuda")
        hip.kv_append(k, k, cache, pages, ints([30, 20, 10]), starts=ints(starts))
    assert (block[:10] == 7).all() and (block[30:] == 7).all() and (cache.keys == 1).all()


@pytest.mark.parametrize("prefix", [0, 40])
@pytest.mark.parametrize("news", [[1, 2, 1], [30, 0, 40]])
def test_tokens_before_the_first_sequence(hip, torch_cuda, prefix, news):
    """They are left alone like those behind the last: in a batch that was cut out of a larger one."""
    gen, dtype, lengths = torch.Generator().manual_seed(15), torch.bfloat16, [500, 20, 70]
    pages, prefix_pages, n = table(lengths, 16, gen, prefix=-(-prefix // 16))
    cache = cache_of(hip, n, 16, 2, 64, dtype)
    fill(cache, pages, lengths, gen)
    fill(cache, prefix_pages[None], [prefix], gen)
    ends = [5 + sum(news[:b]) for b in range(4)]
    q = queries(gen, ends[-1] + 3, 8, 64, dtype)
    out = torch.full_like(q, 7.0)
    if prefix:
        hip.attention_shared(q, cache, prefix_pages, prefix, pages, ints(lengths), starts=ints(ends), out=out)
    else:
        hip.attention_paged(q, cache, pages, ints(lengths), starts=ints(ends), out=out)
    want, tol, _, _ = ref.attention(q, cache.keys, cache.values, pages, lengths, ends, prefix=prefix_pages, prefix_length=prefix)
    same, worst = ref.compare(out[5:ends[-1]], want[5:ends[-1]], tol[5:ends[-1]])
    assert same and worst <= 1 and (out[:5] == 7).all() and (out[ends[-1]:] == 7).all()
    k = torch.full((ends[-1] + 3, 2, 64), 3.0, dtype=dtype, device="cuda")
    before, q_out = cache.keys.clone(), torch.full_like(q, 7.0)
    hip.kv_append(k, k, cache, pages, ints(lengths), starts=ints(ends), q=q, q_out=q_out)
    changed = (cache.keys != before).any(-1).any(-1) & ~before.isnan().any(-1).any(-1)
    assert int(changed.sum()) == sum(news)
    assert (q_out[:5] == 7).all() and (q_out[ends[-1]:] == 7).all() and torch.equal(q_out[5:ends[-1]], q[5:ends[-1]])


def test_no_tokens_and_no_sequences(hip, torch_cuda):
    cache = cache_of(hip, 4, 16, 2, 64, torch.bfloat16)
    none = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert hip.attention_paged(none, cache, ints([[0]]), ints([5]), starts=ints([0, 0])).shape == (0, 4, 64)
    assert hip.attention_paged(none, cache, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([])).shape == (0, 4, 64)
    assert hip.kv_append(none[:, :2], none[:, :2], cache, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([]), q=none).shape == (0, 4, 64)
    # tokens, and no sequence that has them
    out = torch.full((2, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q = torch.ones_like(out)
    hip.attention_paged(q, cache, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([]), starts=ints([0]), out=out)
    assert (out == 7).all()
    # and a table without a page
    assert (hip.attention_paged(q, cache, torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints([3, 4])) == 0).all()


def test_a_cache_past_four_gigabytes(hip, torch_cuda):
    """Offsets that pass 32 bits, for appending and reading."""
    gen = torch.Generator().manual_seed(10)
    pages_in_all, page = 3 << 14, 64                          # 49152 pages of 64 x 8 heads x 256 bytes: 6 GiB each of keys and values
    cache = hip.KvCache(*(torch.empty(pages_in_all, page, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    lengths = [300, 150]
    pages = ints([[pages_in_all - 1, 5, pages_in_all // 2 + 1, pages_in_all - 7, 1], [pages_in_all - 2, 0, 40000, -1, -1]])
    k, v = (torch.randn(450, 8, 128, generator=gen).bfloat16().cuda() for _ in range(2))
    starts = [0, 300, 450]
    hip.kv_append(k, v, cache, pages, ints(lengths), starts=ints(starts))
    for b in range(2):
        assert torch.equal(ref.gather(cache.keys, pages[b], lengths[b]), k[starts[b]:starts[b + 1]])
        assert torch.equal(ref.gather(cache.values, pages[b], lengths[b]), v[starts[b]:starts[b + 1]])
    for q, s in ((queries(gen, 2, 16, 128, torch.bfloat16), None), (queries(gen, 450, 8, 128, torch.bfloat16), starts)):
        got = hip.attention_paged(q, cache, pages, ints(lengths), starts=None if s is None else ints(s))
        want, tol, _, _ = ref.attention(q, cache.keys, cache.values, pages, lengths, s)
        same, worst = ref.compare(got, want, tol)
        assert same and worst <= 1


def step(hip, state, cache, pages, lengths, starts=None, prefix=None):
    """What a layer does between its products: append with the rotation, attention."""
    k, v, q, plan = state
    first = 0 if prefix is None else prefix[1]
    q = hip.kv_append(k, v, cache, pages, lengths, starts=starts, rotary=plan, q=q, first=first)
    if prefix is None:
        return hip.attention_paged(q, cache, pages, lengths, starts=starts)
    return hip.attention_shared(q, cache, *prefix, pages, lengths, starts=starts)


def test_generation_with_a_cache_is_the_whole_sequence_at_once(hip, torch_cuda):
    """A prompt in chunks, then token by token, against attention over the whole sequence in one call and against float64 without a cache."""
    gen, d, heads, kv_heads, n, dtype = torch.Generator().manual_seed(11), 64, 6, 2, 150, torch.bfloat16
    plan = hip.Rotary(d)
    k, v = (torch.randn(2, n, kv_heads, d, generator=gen).to(dtype).cuda() for _ in range(2))
    q = (2 * torch.randn(2, n, heads, d, generator=gen)).to(dtype).cuda()
    pages, _, count = table([n, n], 16, gen)
    cache = cache_of(hip, count, 16, kv_heads, d, dtype)
    rows, done = [], [0, 0]
    for news in ([100, 30], [0, 70], [17, 17]) + ([1, 1],) * 33:
        at = [slice(done[b], done[b] + news[b]) for b in range(2)]
        done = [done[b] + news[b] for b in range(2)]
        cat = lambda t: torch.cat([t[b, at[b]] for b in range(2)])  # noqa: E731
        starts = None if news == [1, 1] else ints([0, news[0], sum(news)])
        got = step(hip, (cat(k), cat(v), cat(q), plan), cache, pages, ints(done), starts)
        rows.append((at, news, got))
    assert done == [n, n]
    whole = torch.empty_like(q)
    for at, news, got in rows:
        whole[0, at[0]], whole[1, at[1]] = got[:news[0]], got[news[0]:]
    fresh = cache_of(hip, count, 16, kv_heads, d, dtype)
    once = step(hip, (k.flatten(0, 1), v.flatten(0, 1), q.flatten(0, 1), plan), fresh, pages, ints([n, n]), ints([0, n, 2 * n])).view(2, n, heads, d)
    place = torch.arange(n).cuda()
    for b in range(2):
        turned = [ref.rotate(t[b], place, plan.frequencies, "half").to(dtype) for t in (q, k)]
        want, tol, _, _ = ref.attention(turned[0], turned[1][None], v[b][None], torch.zeros(1, 1, dtype=torch.int32), [n], [0, n])
        for got in (whole[b], once[b]):
            same, worst = ref.compare(got, want, 3 * tol)      # (a turned value may be rounded the other way, once each for q and k)
            assert same and worst <= 1, worst


@pytest.mark.parametrize("shared", [False, True])
def test_captured_and_replayed(hip, torch_cuda, shared):
    """Lengths, pages and tokens change between the replays of one graph; every replay gives what the eager call does."""
    gen, dtype, plan, batch = torch.Generator().manual_seed(12), torch.float16, hip.Rotary(64), 5
    prefix = (ints([20, 21, 22]), 45) if shared else None
    pages = torch.arange(20, dtype=torch.int32).view(5, 4).cuda()
    caches = [cache_of(hip, 23, 16, 2, 64, dtype, fill=0.5) for _ in range(2)]
    lengths = ints([1] * batch)
    k, v, q = (torch.zeros(batch, h, 64, dtype=dtype, device="cuda") for h in (2, 2, 8))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(hip, (k, v, q, plan), caches[0], pages, lengths, prefix=prefix)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(hip, (k, v, q, plan), caches[0], pages, lengths, prefix=prefix)
    for turn in range(12):
        lengths.copy_(ints([turn * 5 + 1, 1 + turn, 64 - turn, 0 if turn == 4 else 33, 17]))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen))
        caches[1].keys.copy_(caches[0].keys)
        caches[1].values.copy_(caches[0].values)
        torch.cuda.synchronize()
        graph.replay()
        want = step(hip, (k, v, q, plan), caches[1], pages, lengths, prefix=prefix)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(caches[0].keys, caches[1].keys) and torch.equal(caches[0].values, caches[1].values)


def test_two_streams_at_once(hip, torch_cuda):
    """Calls on two streams, each with a workspace of its own, give what they give alone."""
    gen = torch.Generator().manual_seed(13)
    lengths = [3000, 100, 5, 2000]
    pages, prefix, n = table(lengths, 16, gen, prefix=20)
    cache = cache_of(hip, n, 16, 2, 128, torch.bfloat16)
    fill(cache, pages, lengths, gen)
    fill(cache, prefix[None], [320], gen)
    qs = [queries(gen, 4, 8, 128, torch.bfloat16) for _ in range(8)]
    on = ints(lengths)
    call = lambda q, i: hip.attention_shared(q, cache, prefix, 320, pages, on) if i % 2 else hip.attention_paged(q, cache, pages, on)  # noqa: E731
    alone = [call(q, i) for i, q in enumerate(qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i // 2 % 2]):
            got.append(call(q, i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, got))


def test_refusals_of_tensors(hip, torch_cuda):
    cache = cache_of(hip, 4, 16, 2, 64, torch.bfloat16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    kv, pages, lengths, plan = q[:, :2], ints([[0, 1], [2, 3]]), ints([5, 6]), hip.Rotary(64)
    wrong = [
        (TypeError, lambda: hip.attention_paged(q.half(), cache, pages, lengths)), (TypeError, lambda: hip.attention_paged(q.cpu(), cache, pages, lengths)),
        (TypeError, lambda: hip.attention_paged(q, cache, pages.long(), lengths)), (TypeError, lambda: hip.attention_paged(q, cache, pages, lengths.float())),
        (TypeError, lambda: hip.attention_paged(q, None, pages, lengths)), (ValueError, lambda: hip.attention_paged(q[:, :3], cache, pages, lengths)),
        (ValueError, lambda: hip.attention_paged(q[..., :56].contiguous(), cache, pages, lengths)), (ValueError, lambda: hip.attention_paged(q[:1], cache, pages, lengths)),
        (ValueError, lambda: hip.attention_paged(q, cache, pages[:1], lengths)), (ValueError, lambda: hip.attention_paged(q, cache, pages, lengths, starts=lengths)),
        (TypeError, lambda: hip.attention_paged(q.transpose(1, 2), cache, pages, lengths)), (ValueError, lambda: hip.attention_paged(q, cache, pages, lengths, out=q[:1])),
        (TypeError, lambda: hip.attention_paged(q, cache, pages, lengths, lse=q)), (ValueError, lambda: hip.attention_paged(q, cache, pages, lengths, lse=torch.zeros(2, 3, device="cuda"))),
        (hip.SarekHipError, lambda: hip.attention_paged(q, cache, pages, lengths, scale=0.0)), (hip.SarekHipError, lambda: hip.attention_paged(q, cache, pages, lengths, scale=math.inf)),
        (ValueError, lambda: hip.attention_shared(q, cache, ints([1]), 17, pages, lengths)), (ValueError, lambda: hip.attention_shared(q, cache, ints([1]), -1, pages, lengths)),
        (hip.SarekHipError, lambda: hip.attention_paged(q, cache, pages, lengths, out=q[:1].expand(2, 4, 64))),
        (ValueError, lambda: hip.kv_append(q, kv, cache, pages, lengths)), (ValueError, lambda: hip.kv_append(kv, kv[:1], cache, pages, lengths)),
        (TypeError, lambda: hip.kv_append(kv, kv, cache, pages, lengths, rotary=64)), (ValueError, lambda: hip.kv_append(kv, kv, cache, pages, lengths, rotary=hip.Rotary(66))),
        (TypeError, lambda: hip.kv_append(kv, kv.float(), cache, pages, lengths)), (ValueError, lambda: hip.kv_append(kv, kv, cache, pages, lengths, q=q, q_out=kv)),
        (ValueError, lambda: hip.rotary(q, lengths, hip.Rotary(66))), (TypeError, lambda: hip.rotary(q, lengths.float(), plan)), (ValueError, lambda: hip.rotary(q, lengths[:1], plan)),
        (TypeError, lambda: hip.rotary(q[0], lengths, plan)), (TypeError, lambda: hip.rotary(q, lengths, plan, out=q.float())),
        (ValueError, lambda: hip.KvCache(cache.keys, cache.values[:2])), (TypeError, lambda: hip.KvCache(cache.keys, cache.values.half())),
        (ValueError, lambda: hip.KvCache(cache.keys[..., :60], cache.values[..., :60])), (ValueError, lambda: hip.KvCache(cache.keys[..., 4:60], cache.values[..., 4:60])),
        (ValueError, lambda: hip.KvCache(cache.keys.expand(4, 16, 2, 64)[:1].expand(3, 16, 2, 64), cache.values[:1].expand(3, 16, 2, 64)))]
    for kind, call in wrong:
        with pytest.raises(kind):
            call()


def test_random_calls(hip, torch_cuda):
    rng = random.Random(14)
    for turn in range(60):
        gen = torch.Generator().manual_seed(turn)
        kv_heads, batch = rng.randint(1, 4), rng.randint(1, 9)
        news = None if rng.random() < 0.4 else [rng.choice([0, 1, 2, 5, 40, 130]) for _ in range(batch)]
        lengths = [max(rng.choice([0, 1, 30, 64, 200, 777]), 0 if news is None else news[b]) for b in range(batch)]
        case = dict(dtype=rng.choice(["bf16", "f16"]), d=8 * rng.randint(1, 32), heads=kv_heads * rng.choice([1, 2, 3, 4, 8, 20]), kv_heads=kv_heads,
                    page=rng.choice([1, 3, 16, 32, 100]), lengths=lengths, news=news, causal=rng.random() < 0.7, prefix=rng.choice([0, 0, 1, 64, 333]),
                    layout=rng.choice(["plain", "heads first", "one block", "heads outermost"]), apart=rng.choice([0, 1, 8]), std=rng.choice([0.5, 2.0, 8.0]))
        print(turn, case, flush=True)
        run(hip, gen, **case)


def test_many_sequences(hip, torch_cuda):
    """More sequences than a wave has lanes, several times over: tiles, stretches and planes are found across the blocks of 64."""
    gen = torch.Generator().manual_seed(16)
    lengths = [int(v) for v in torch.randint(0, 40, (700,), generator=gen)]
    lengths[333] = lengths[699] = 5000
    news = [min(v, 1 + i % 3) for i, v in enumerate(lengths)]
    run(hip, gen, "bf16", 64, 2, 1, 16, lengths)
    run(hip, gen, "f16", 64, 2, 1, 16, lengths, news, pad=1)
    run(hip, gen, "bf16", 64, 24, 1, 16, lengths[:200] + [4000], news[:200] + [3], prefix=200)


def test_many_small_weights(hip, torch_cuda):
    """One key far above 60000 others, whose weights of 2^-14 to 2^-17 (below fp16's normal numbers) are most of the sum."""
    for dtype in ("f16", "bf16"):
        gen = torch.Generator().manual_seed(17)
        n, d = 60000, 64
        pages, _, count = table([n], 64, gen)
        cache = cache_of(hip, count, 64, 1, d, TYPES[dtype])
        fill(cache, pages, [n], gen, key=0.1)
        cache.values[:] = cache.values.abs()
        for rows in (1, 40):
            q = torch.ones(rows, 2, d, dtype=TYPES[dtype], device="cuda")
            cache.keys[pages[0, 0].long(), 0, 0] = 11.0 / 8
            lse = torch.empty(rows, 2, device="cuda")
            starts = [0, rows]
            got = hip.attention_paged(q, cache, pages, ints([n]), starts=ints(starts), causal=False, lse=lse)
            want, tol, want_lse, lse_tol = ref.attention(q, cache.keys, cache.values, pages, [n], starts, False)
            assert ref.compare(got, want, tol)[1] <= 1 and ref.compare(lse, want_lse, lse_tol)[1] <= 1


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 3.0])
def test_scales(hip, torch_cuda, scale):
    gen = torch.Generator().manual_seed(18)
    run(hip, gen, "bf16", 128, 4, 2, 16, [300, 5, 0, 77], scale=scale)
    run(hip, gen, "f16", 128, 4, 2, 16, [300, 5, 77], [300, 2, 70], scale=scale)


def test_tables_with_rows_apart(hip, torch_cuda):
    """A page table that is a part of a wider one."""
    gen = torch.Generator().manual_seed(19)
    lengths = [40, 100]
    pages, _, n = table(lengths, 16, gen)
    wide = torch.full((2, pages.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + pages.shape[1]] = pages
    cache = cache_of(hip, n, 16, 2, 64, torch.bfloat16)
    fill(cache, pages, lengths, gen)
    q = queries(gen, 2, 4, 64, torch.bfloat16)
    assert torch.equal(hip.attention_paged(q, cache, wide[:, 2:2 + pages.shape[1]], ints(lengths)), hip.attention_paged(q, cache, pages, ints(lengths)))


def test_on_a_stream_of_its_own(hip, torch_cuda):
    """Everything runs on the current stream, behind what made its inputs there."""
    gen = torch.Generator().manual_seed(20)
    plan, pages = hip.Rotary(64), torch.arange(20, dtype=torch.int32).view(5, 4).cuda()
    k, v, q = (torch.randn(5, h, 64, generator=gen).bfloat16().cuda() for h in (2, 2, 8))
    want = step(hip, (k, v, q, plan), cache_of(hip, 20, 16, 2, 64, torch.bfloat16, fill=0.5), pages, ints([64, 33, 1, 20, 50]))
    cache = cache_of(hip, 20, 16, 2, 64, torch.bfloat16, fill=0.5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [t + 0 for _ in range(20) for t in (k, v, q)][-3:]
        got = step(hip, (*late, plan), cache, pages, ints([64, 33, 1, 20, 50]))
    side.synchronize()
    assert torch.equal(got, want)


def test_tables_with_rows_on_each_other(hip, torch_cuda):
    """An expanded page table has one row in memory: what lies behind it is not read as the others."""
    cache = cache_of(hip, 4, 16, 2, 64, torch.bfloat16, fill=0.0)
    q, lengths = torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda"), ints([20, 30])
    for pages in (ints([[0, 1]]).expand(2, 2), torch.arange(3, dtype=torch.int32, device="cuda").as_strided((2, 2), (1, 1))):
        for call in (lambda: hip.attention_paged(q, cache, pages, lengths), lambda: hip.attention_shared(q, cache, ints([3]), 16, pages, lengths),
                     lambda: hip.kv_append(q[:, :2], q[:, :2], cache, pages, lengths)):
            with pytest.raises(hip.SarekHipError):
                call()
    one = ints([[0, 1]]).as_strided((1, 2), (0, 1))      # (the only row may lie anyhow)
    assert torch.equal(hip.attention_paged(q[:1], cache, one, ints([20])), torch.zeros_like(q[:1]))


@pytest.mark.parametrize("news,prefix", [(None, 0), ([40, 3], 0), ([2, 2], 100), ([60, 70], 100)])
def test_out_may_be_q(hip, torch_cuda, news, prefix):
    gen = torch.Generator().manual_seed(21)
    lengths = [3000, 90]
    pages, prefix_pages, n = table(lengths, 16, gen, prefix=-(-prefix // 16))
    cache = cache_of(hip, n, 16, 2, 64, torch.bfloat16)
    fill(cache, pages, lengths, gen)
    fill(cache, prefix_pages[None], [prefix], gen)
    q = queries(gen, 2 if news is None else sum(news), 8, 64, torch.bfloat16)
    starts = None if news is None else ints([0, news[0], sum(news)])
    call = lambda out: hip.attention_shared(q, cache, prefix_pages, prefix, pages, ints(lengths), starts=starts, out=out)  # noqa: E731
    want = call(None)
    assert call(q) is q and torch.equal(q, want)


def test_many_heads(hip, torch_cuda):
    gen = torch.Generator().manual_seed(22)
    run(hip, gen, "f16", 8, 520, 520, 16, [70, 1, 0])
    run(hip, gen, "bf16", 16, 600, 1, 16, [70, 9, 300], [3, 1, 2])


@pytest.mark.parametrize("name,values", [("tile_workgroups", [-1, 0, 1, 7, 5000, 1 << 40]), ("stream_workgroups", [-1, 0, 1, 7, 5000, 1 << 40]), ("large_rows", [0, 1 << 40])])
def test_every_split_gives_the_same(hip, torch_cuda, name, values):
    """What decides how the keys are split and which tiles are taken is free to be set."""
    try:
        for v in values:
            hip.set_tunable("attention." + name, v)
            gen = torch.Generator().manual_seed(23)
            run(hip, gen, "bf16", 128, 8, 2, 16, [1500, 3, 400])
            run(hip, gen, "f16", 128, 8, 2, 16, [1500, 30, 400], [300, 30, 1])
            run(hip, gen, "bf16", 64, 8, 2, 16, [100, 3, 40], prefix=700)
            run(hip, gen, "bf16", 128, 8, 2, 16, [100, 3, 400], [90, 3, 300], prefix=700)
    finally:
        hip.set_tunable("attention." + name, {"tile_workgroups": 512, "stream_workgroups": 512, "large_rows": 25600}[name])


def test_large_tiles(hip, torch_cuda):
    """More than 25600 rows to a sequence that fill the card twice, so 256 to a workgroup."""
    gen = torch.Generator().manual_seed(24)
    run(hip, gen, "bf16", 72, 96, 6, 16, [1700], [1640])
    run(hip, gen, "f16", 128, 64, 4, 20, [1700, 1800], [1650, 1800], causal=False)


def test_more_keys_than_stretches_hold(hip, torch_cuda):
    """One head of keys and few rows: as many stretches as a row may have, of several units each."""
    gen = torch.Generator().manual_seed(25)
    run(hip, gen, "bf16", 64, 2, 1, 64, [70001])
    run(hip, gen, "f16", 256, 2, 1, 64, [9000, 30001])
