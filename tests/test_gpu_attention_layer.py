"""The attention layer: norm, products, cache and attention as one, against the same steps in float64 with the layer's roundings."""
import pytest
import torch


pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def layer_of(hip, width, heads, kv_heads, d, dtype, gen):
    from spoc_amd.attention import MxAttention
    weight = (1 + 0.1 * torch.randn(width, generator=gen)).to(dtype).cuda()
    qkv = hip.mx_quantize((0.08 * torch.randn((heads + 2 * kv_heads) * d, width, generator=gen)).cuda(), "fp4")
    output = hip.mx_quantize((0.08 * torch.randn(width, heads * d, generator=gen)).cuda(), "fp4")
    return MxAttention(weight, qkv, output, heads, kv_heads, hip.Rotary(d // 2 // 2 * 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix", [0, 50])
def test_layer_is_its_steps(hip, torch_cuda, dtype, prefix):
    """Each step is checked for itself elsewhere: here that the layer puts them together as it says, bit for bit."""
    gen = torch.Generator().manual_seed(1)
    heads, kv, d, width = 6, 2, 40, 200
    layer = layer_of(hip, width, heads, kv, d, dtype, gen)
    caches = [hip.KvCache(*(torch.randn(12, 16, kv, d, generator=torch.Generator().manual_seed(2 + i)).to(dtype).cuda() for i in range(2))) for _ in range(2)]
    pages, lengths, starts = ints([0, 1, 2], [3, 4, 5]), ints(40, 33), ints(0, 40, 70)
    x, residual = (torch.randn(72, width, generator=gen).to(dtype).cuda() for _ in range(2))
    shared = (ints(8, 9, 10, 11), prefix) if prefix else None
    y, h = layer(x, caches[0], pages, lengths, starts, residual, shared)
    q8, want_h, _ = hip.rms_norm_mx(x, layer.weight, residual=residual)
    qkv = hip.gemm_mx(q8, layer.qkv, dtype=dtype).view(72, -1, d)
    q = hip.kv_append(qkv[:, heads:heads + kv].contiguous(), qkv[:, heads + kv:].contiguous(), caches[1], pages, lengths, starts=starts, rotary=layer.rotary,
                      q=qkv[:, :heads].contiguous(), first=prefix)
    out = torch.zeros(72, heads, d, dtype=dtype, device="cuda")
    if prefix:
        hip.attention_shared(q, caches[1], *shared, pages, lengths, starts=starts, out=out)
    else:
        hip.attention_paged(q, caches[1], pages, lengths, starts=starts, out=out)
    want = hip.gemm_mx(hip.mx_quantize(out.flatten(1), "fp8"), layer.output, dtype=dtype)
    assert torch.equal(h, want_h) and torch.equal(y, want) and (out[70:] == 0).all()
    assert all(torch.equal(a, b) for a, b in ((caches[0].keys, caches[1].keys), (caches[0].values, caches[1].values)))


def test_a_prompt_in_pieces_is_the_prompt(hip, torch_cuda):
    """Chunks and single tokens through the layer against the whole prompt: they differ by roundings of the turned and weighted values alone."""
    gen = torch.Generator().manual_seed(3)
    heads, kv, d, width, n = 4, 1, 64, 256, 75
    layer = layer_of(hip, width, heads, kv, d, torch.bfloat16, gen)
    x = torch.randn(n, width, generator=gen).bfloat16().cuda()
    pages = ints([4, 0, 3, 1, 2])
    whole, _ = layer(x, hip.KvCache.empty(5, 16, kv, d), pages, ints(n), ints(0, n))
    cache, rows, at = hip.KvCache.empty(5, 16, kv, d), [], 0
    for step in (30, 17, 1, 1, 20, 1, 5):
        rows.append(layer(x[at:at + step], cache, pages, ints(at + step), None if step == 1 else ints(0, step))[0])
        at += step
    # 16 bits of attention's output, then codes of 3 mantissa bits: a rounding the other way is 2^-3 of a value, of a few values
    got, want = torch.cat(rows).double(), whole.double()
    assert at == n and float((got - want).norm() / want.norm()) < 2.0 ** -5


def test_command(hip, torch_cuda, capsys):
    from spoc_amd import attention
    assert attention.main([]) == 0 and attention.main(["1", "512", "3"]) == 0 and attention.main(["300", "1000", "2"]) == 0
    assert "output within" in capsys.readouterr().out


def test_refusals(hip, torch_cuda):
    from spoc_amd.attention import MxAttention
    gen = torch.Generator().manual_seed(4)
    layer = layer_of(hip, 256, 4, 2, 64, torch.bfloat16, gen)
    for bad in (dict(heads=3), dict(kv_heads=3), dict(heads=8), dict(weight=layer.weight[:128].clone()), dict(output=layer.qkv)):
        with pytest.raises(ValueError):
            MxAttention(**{**dict(weight=layer.weight, qkv=layer.qkv, output=layer.output, heads=4, kv_heads=2), **bad})
    with pytest.raises(TypeError):
        MxAttention(layer.weight.float(), layer.qkv, layer.output, 4, 2)
