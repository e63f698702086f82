"""The operators on a paged cache as a server uses them: caches past 4 GiB under every head length and kernel, the layer in a graph, several threads."""
import threading

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,kv_heads,group,news", [(64, 2, 4, None), (64, 2, 4, [200, 40]), (96, 2, 2, [200, 40]), (96, 2, 2, None), (128, 4, 1, None), (192, 2, 3, None), (192, 2, 3, [200, 40]),
                                                   (256, 2, 2, None), (256, 2, 2, [200, 40])])
def test_caches_past_four_gigabytes(hip, torch_cuda, dtype, d, kv_heads, group, news):
    gen, page, lengths = torch.Generator().manual_seed(d), 64, [300, 150]
    count = (9 << 29) // (page * kv_heads * d * 2)                    # 4.5 GiB each of keys and values
    cache = hip.KvCache.empty(count, page, kv_heads, d, dtype=dtype)
    pages = ints([count - 1, 5, count // 2 + 1, count - 7, 1], [count - 2, 0, count * 8 // 9 + 3, -1, -1])
    prefix = ints(count - 9, count // 3)
    for which, n in ((pages[0], 300), (pages[1], 150), (prefix, 100)):
        at = torch.arange(n)
        where = which.cpu().long()[at // page].cuda(), (at % page).cuda()
        for t in (cache.keys, cache.values):
            t[where] = torch.randn(n, kv_heads, d, generator=gen).to(dtype).cuda()
    starts = None if news is None else [0, news[0], sum(news)]
    q = (2 * torch.randn(2 if news is None else sum(news), kv_heads * group, d, generator=gen)).to(dtype).cuda()
    more = dict(starts=None if starts is None else ints(*starts))
    for length in (0, 100):
        got = hip.attention_shared(q, cache, prefix, length, pages, ints(*lengths), **more)
        want, tol, _, _ = ref.attention(q, cache.keys, cache.values, pages, lengths, starts, prefix=prefix, prefix_length=length)
        same, worst = ref.compare(got, want, tol)
        assert same and worst <= 1, (worst, same)


def test_tiles_of_256_rows_past_four_gigabytes(hip, torch_cuda):
    """Values that some rows do not see are unbounded, so that they are read again from their places."""
    gen, page, n, heads, kv_heads, d = torch.Generator().manual_seed(1), 64, 1700, 64, 4, 128
    count = (9 << 29) // (page * kv_heads * d * 2)
    cache = hip.KvCache.empty(count, page, kv_heads, d)
    held = -(-n // page)
    pages = (count - 1 - torch.randperm(held, generator=gen)).int()[None].cuda()
    at = torch.arange(n)
    where = pages[0].cpu().long()[at // page].cuda(), (at % page).cuda()
    for t in (cache.keys, cache.values):
        t[where] = torch.randn(n, kv_heads, d, generator=gen).bfloat16().cuda()
    cache.values[pages[0, 1600 // page].long(), 1600 % page, 1, 5] = float("inf")
    q = (2 * torch.randn(1650, heads, d, generator=gen)).bfloat16().cuda()
    got = hip.attention_paged(q, cache, pages, ints(n), starts=ints(0, 1650))
    want, tol, _, _ = ref.attention(q, cache.keys, cache.values, pages, [n], [0, 1650])
    same, worst = ref.compare(got, want, tol)
    assert same and worst <= 1, (worst, same)


def layer_of(hip, gen):
    from spoc_amd.attention import MxAttention
    weight = (1 + 0.1 * torch.randn(256, generator=gen)).bfloat16().cuda()
    qkv, output = (hip.mx_quantize((0.08 * torch.randn(rows, 256, generator=gen)).cuda(), "fp4") for rows in (8 * 64, 256))
    return MxAttention(weight, qkv, output, 4, 2, hip.Rotary(64))


@pytest.mark.parametrize("prefix", [0, 45])
def test_layer_captured_and_replayed(hip, torch_cuda, prefix):
    """Lengths, pages, the places of a batch that are used and what is in them change between the replays of one graph."""
    gen = torch.Generator().manual_seed(2)
    layer = layer_of(hip, gen)
    caches = [hip.KvCache(*(torch.randn(24, 16, 2, 64, generator=torch.Generator().manual_seed(3 + i)).bfloat16().cuda() for i in range(2))) for _ in range(2)]
    shared = (ints(20, 21, 22), prefix) if prefix else None
    pages, lengths, starts = torch.zeros(5, 4, dtype=torch.int32, device="cuda"), ints(*[1] * 5), ints(0, 1, 2, 3, 4, 5)
    x, residual = (torch.zeros(9, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer(x, caches[0], pages, lengths, starts, residual, shared)
    side.synchronize()
    for own, other in zip((caches[1].keys, caches[1].values), (caches[0].keys, caches[0].values)):
        own.copy_(other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = layer(x, caches[0], pages, lengths, starts, residual, shared)
    for turn in range(8):
        news = [1, turn % 3, 0, 2, 1 + turn % 2]
        lengths.copy_(ints(turn * 5 + 1, 2 + turn, 0, 64 - turn, 17))
        starts.copy_(ints(*(sum(news[:b]) for b in range(6))))
        pages.copy_(torch.randperm(20, generator=gen).int().view(5, 4))
        for t in (x, residual):
            t.copy_(torch.randn(t.shape, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        want_y, want_h = layer(x, caches[1], pages, lengths, starts, residual, shared)
        torch.cuda.synchronize()
        assert torch.equal(y, want_y) and torch.equal(h, want_h)
        assert torch.equal(caches[0].keys, caches[1].keys) and torch.equal(caches[0].values, caches[1].values)


def test_two_graphs_at_once(hip, torch_cuda):
    """Each has its workspace: replayed on two streams they give what they give alone."""
    gen = torch.Generator().manual_seed(4)
    cache = hip.KvCache(*(torch.randn(300, 16, 2, 128, generator=gen).bfloat16().cuda() for _ in range(2)))
    pages, lengths = torch.randperm(300, generator=gen).int().view(3, 100).cuda(), ints(1600, 77, 900)
    qs = [torch.randn(3, 8, 128, generator=gen).bfloat16().cuda() for _ in range(2)]
    want = [hip.attention_paged(q, cache, pages, lengths) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, q in zip(graphs, qs):
        with torch.cuda.graph(graph):
            outs.append(hip.attention_paged(q, cache, pages, lengths))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for out in outs:
            out.fill_(7)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_threads(hip, torch_cuda):
    """Calls let other threads run while they launch; each has its own stream, arguments and result, and a refusal names its own fault."""
    gen = torch.Generator().manual_seed(5)
    cache = hip.KvCache(*(torch.randn(60, 16, 2, 64, generator=gen).bfloat16().cuda() for _ in range(2)))
    pages, lengths = torch.randperm(60, generator=gen).int().view(3, 20).cuda(), ints(300, 77, 9)
    qs = [torch.randn(3, 8, 64, generator=gen).bfloat16().cuda() for _ in range(4)]
    want = [hip.attention_paged(q, cache, pages, lengths) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for turn in range(50):
                if not torch.equal(hip.attention_paged(qs[i], cache, pages, lengths), want[i]):
                    wrong.append((i, turn))
                try:
                    hip.attention_paged(qs[i], cache, pages, lengths, scale=0.0 if i % 2 else None, out=None if i % 2 else qs[i][:1].expand(3, 8, 64))
                    wrong.append((i, turn, "served"))
                except hip.SarekHipError as e:
                    if ("scale" if i % 2 else "strides") not in str(e):
                        wrong.append((i, turn, str(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
