"""Products of microscaled rows on every tile: how their sums are held, the tiles' rings and spans of scales all the way round, and
results at the ends of the formats, against float64; and large quantisations against those of a few rows.

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


# kp of 512 (one span of scales) to 4096 (the tiles' rings and periods all round), an odd multiple of 256 (a last span of 8 bytes) among them
@pytest.mark.parametrize("k", [505, 768, 1530, 1792, 3300, 4090])
@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_every_tile_and_length_of_k(hip, torch_cuda, shape, fmt, dtype, k):
    m, n = 300, 333
    a, b, bias = operands(hip, m, n, k, fmt, k)
    whole = torch.full((m * (n + 7) + 9,), 7.0, dtype=dtype, device="cuda")
    c = whole[3:3 + m * (n + 7)].view(m, n + 7)[:, :n]
    with tuned(hip, shape=shape):
        check(hip, hip.gemm_mx(a, b, bias=bias, dtype=dtype, out=c), a, b, bias, False)
        plain = hip.gemm_mx(a, b, dtype=dtype)
        check(hip, plain, a, b, None, False)
        assert torch.equal(plain, hip.gemm_mx(a, b, dtype=dtype))
    c.fill_(7.0)
    assert bool((whole == 7.0).all())


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_c_past_the_caches(hip, torch_cuda, fmt, dtype):
    """Rows of C that are whole 128-byte lines, the last ones of a tile missing, and the same bits as through the caches; rows
    that are not, where nothing changes."""
    for m, n in ((700, 768), (300, 333)):
        a, b, bias = operands(hip, m, n, 1100, fmt, n)
        with tuned(hip, shape=6):
            want = hip.gemm_mx(a, b, bias=bias, relu=True, dtype=dtype)
        check(hip, want, a, b, bias, True)
        out = torch.full((m + 3, n), 7.0, dtype=dtype, device="cuda")
        with tuned(hip, shape=6, past_caches_mib=0):
            hip.gemm_mx(a, b, bias=bias, relu=True, dtype=dtype, out=out[:m])
        assert torch.equal(out[:m], want) and bool((out[m:] == 7.0).all())


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("shape", [0, 3, 5, 6])
def test_scales_far_apart(hip, torch_cuda, shape, fmt):
    """Scales of A and B that cancel, results below the normal numbers (a rounding to a multiple of 2^-149 for each addition) and past the
    largest one (of magnitudes only, so that no part of a sum passes it before the sum does)."""
    m, n, k = 40, 70, 600
    for up, down, kind in ((60, -60, "cancel"), (-70, 72, "cancel"), (-66, -66, "least"), (60, 66, "largest"), (60, 59, "largest")):
        a, b, _ = operands(hip, m, n, k, fmt, 3)
        if kind == "largest":
            a.codes.bitwise_and_(0x7F if fmt == "fp8" else 0x77), b.codes.bitwise_and_(0x77)
        for q, by in ((a, up), (b, down)):
            q.scales.copy_(torch.where(q.scales > 0, q.scales.int() + by, 0).to(torch.uint8))
        want = hip.mx_dequantize(a, torch.float32).double() @ hip.mx_dequantize(b, torch.float32).double().t()
        size = hip.mx_dequantize(a, torch.float32).double().abs() @ hip.mx_dequantize(b, torch.float32).double().abs().t()
        for dtype in (torch.bfloat16,) if fmt == "fp8" else (torch.bfloat16, torch.float32):
            with tuned(hip, shape=shape):
                c = hip.gemm_mx(a, b, dtype=dtype).double()
            off = (2 * 19 + 13) * (2 * EPS32 * size + 2.0 ** -149)
            bound = off + HALF_ULP[dtype] * (want.abs() + off) + LEAST[dtype]
            top = torch.finfo(dtype).max
            sure, never = want.abs() - off > top * (1 + 2 * HALF_ULP[dtype]), want.abs() + off < top
            assert bool(((c - want).abs() <= bound)[never].all()) and bool((c.abs() == float("inf"))[sure].all())
            assert bool(sure.any()) == (kind == "largest")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_quantise_several_pieces_to_a_thread(hip, torch_cuda, fmt, dtype):
    """A matrix of 2^16 pieces of 256 values and more, whose threads take several each, is what its rows are a few at a time."""
    rows, k = 4099, 4100
    x = torch.empty(rows, k, device="cuda").normal_(generator=generator(1)).mul_(torch.exp(torch.empty(rows, 1, device="cuda").normal_(0, 2, generator=generator(2)))).to(dtype)
    q = hip.mx_quantize(x, fmt)
    back = hip.mx_dequantize(q, dtype)
    for first in range(0, rows, 1000):
        part = hip.mx_quantize(x[first:first + 1000], fmt)
        assert torch.equal(q.codes[first:first + 1000], part.codes) and torch.equal(q.scales[first:first + 1000], part.scales)
        assert torch.equal(back[first:first + 1000], hip.mx_dequantize(part, dtype))


@pytest.mark.parametrize("shape", SHAPES)
def test_undefined_codes(hip, torch_cuda, shape):
    """A code that is a NaN, in a block with a scale like any other, makes NaN of its row of C and of nothing else."""
    m, n, k = 70, 90, 900
    a, b, _ = operands(hip, m, n, k, "fp8", 9)
    a.codes[3, 899], a.codes[40, 17] = 0x7F, 0xFF
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[3], want[40] = True, True
    with tuned(hip, shape=shape):
        assert torch.equal(torch.isnan(hip.gemm_mx(a, b)), want)
