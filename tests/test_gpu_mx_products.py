"""Products of microscaled rows on every tile: how their sums are held, the tiles' rings and spans of scales all the way round, and
results at the ends of the formats, against float64.

Tolerances.  eps = 2^-24.  The products of a block of 32 are exact and add up exactly; blocks (those of 8-bit rows in two parts) are added
one after the other, each with a rounding of at most a float32's last bit, 2 eps, and so are the sums of a workgroup's eight waves and the
bias, four being spare: (2 ceil(k / 32) + 13) 2 eps of the sum of the magnitudes.  C is then rounded to its type.  Rows of codes that are
drawn so that every partial sum is a float32 have no tolerance."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half the smallest step
SHAPES = list(range(7))                    # gemm_mx.shape: 16 x 16 to 256 x 256
KINDS = [("fp8", torch.bfloat16), ("fp8", torch.float16), ("fp4", torch.bfloat16), ("fp4", torch.float16), ("fp4", torch.float32)]


@contextlib.contextmanager
def tuned(hip, **values):
    for name, value in values.items():
        hip.set_tunable("gemm_mx." + name, value)
    try:
        yield
    finally:
        for name, value in {"shape": -1, "past_caches_mib": 200}.items():
            hip.set_tunable("gemm_mx." + name, value)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def operands(hip, m, n, k, fmt, seed):
    """Activations with a few features that are much larger than the others, weights whose rows differ in size."""
    g = generator(seed)
    a, b = (torch.empty(r, k, device="cuda").normal_(generator=g) for r in (m, n))
    a = a * torch.where(torch.rand(k, device="cuda", generator=g) < 0.02, 20.0, 1.0)
    b = b * torch.exp(torch.empty(n, 1, device="cuda").normal_(0, 0.5, generator=g))
    return hip.mx_quantize(a, fmt), hip.mx_quantize(b, "fp4"), torch.empty(n, device="cuda").normal_(0, 3, generator=g)


def check(hip, c, a, b, bias, relu):
    va, vb = hip.mx_dequantize(a, torch.float32).double(), hip.mx_dequantize(b, torch.float32).double()
    want, size = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    if relu:
        want = want.clamp(min=0)
    off = (2 * -(-a.k // 32) + 13) * 2 * EPS32 * size
    assert bool(((c.double() - want).abs() <= off + HALF_ULP[c.dtype] * (want.abs() + off) + LEAST[c.dtype]).all())


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_sums_are_held_in_32_bits(hip, torch_cuda, shape, fmt, dtype):
    for m, n, k in ((70, 90, 600), (33, 300, 4000), (300, 270, 1100)):
        a, b, bias = operands(hip, m, n, k, fmt, m + k)
        with tuned(hip, shape=shape):
            check(hip, hip.gemm_mx(a, b, dtype=dtype), a, b, None, False)
            check(hip, hip.gemm_mx(a, b, bias=bias, relu=True, dtype=dtype), a, b, bias, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_large_products_that_cancel_leave_the_small_ones(hip, torch_cuda, shape, dtype):
    """At most five pairs of 448 x 6 and -448 x 6 to a row, side by side or apart, between values from 2^-9 on times 0.5 and more: all
    partial sums, in any order, are multiples of 2^-10 below 2^14, so float32 holds each, and C is what is left, rounded once."""
    m, n, k = 70, 90, 1536
    g = generator(shape)
    pick = lambda high, *size: torch.randint(0, high, size, device="cuda", generator=g)  # noqa: E731
    codes = torch.zeros(m, k, dtype=torch.uint8, device="cuda")
    for r in range(m):
        at = torch.randperm(k // 8, device="cuda", generator=g)[:5] * 8          # five runs of eight
        for q, start in enumerate(at.tolist()):
            codes[r, start:start + 8] = (pick(16, 8) | pick(2, 8) << 7).to(torch.uint8)     # up to 15/8 2^-6
            one, other = torch.randperm(8, device="cuda", generator=g)[:2].tolist()
            codes[r, start + one], codes[r, start + other] = 0x7E, 0xFE
            if q == 4:                                                             # the last pair in runs of eight that are apart
                codes[r, start + other], codes[r, (start + k // 2) % k] = 0, 0xFE
    weights = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    weights[:] = torch.where(pick(2, n, 1) == 1, 0x7, 0xF)                         # 6 or -6 in all of a row
    weights = torch.where((codes.unsqueeze(1).bitwise_and(0x7F) >= 0x7E).any(0), weights, (pick(2, n, k) << 3 | 1 + pick(2, n, k)).to(torch.uint8))
    a = hip.MxTensor(codes.contiguous(), torch.full((m, k // 32), 127, dtype=torch.uint8, device="cuda"), "fp8", k)
    b = hip.MxTensor((weights[:, 0::2] | weights[:, 1::2] << 4).contiguous(), torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda"), "fp4", k)
    want = hip.mx_dequantize(a, torch.float32).double() @ hip.mx_dequantize(b, torch.float32).double().t()
    with tuned(hip, shape=shape):
        assert torch.equal(hip.gemm_mx(a, b, dtype=dtype), want.float().to(dtype))
