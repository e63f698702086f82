"""Microscaled rows on the GPU: quantisation, the norm that writes 8-bit rows, its gradient, products with 4-bit weights, and
the layer made of them, against float64 from the formats' definitions (mx_reference.py).

Tolerances.  Quantisation has none: codes and scale bytes are the definition's.  eps = 2^-24 is float32's relative rounding.
Norm: 1 / rms goes through k squares (one rounding each), sums of at most k / 64 + 16 terms in a row, a division, an addition, a
square root and a division; with k / 64 + 16 <= 1040 that is (k / 64 + 24) eps, halved by the square root, taken whole here, and
two more roundings to the normed value.  A normed value may then be rounded to 8 bits from anywhere within that relative
distance.  Gradient: the mean of products likewise, relative to the sum of magnitudes; the final rounding to the type.
Products: float32 sums of k terms in any order are within k eps of the sum of magnitudes (4-bit rows); with 8-bit rows the
matrix unit adds 128 products on a grid that is measured at 2^-14.4 of their sum of magnitudes at the worst: 2^-13; then the
bias and the type's rounding."""
import numpy as np
import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half the smallest step
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 255), (4, 256), (7, 257), (61, 1001), (1, 4096), (3, 11007), (130, 2048), (2, 20011),
         (1, 70001)]


def host(t):
    return t.detach().double().cpu().numpy()


def random_rows(rows, k, dtype, seed, spread=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.empty(rows, k, device="cuda").normal_(generator=g)
    return (x * torch.exp(torch.empty(rows, k, device="cuda").normal_(0, spread, generator=g).clamp(-6, 6))).to(dtype)


def guarded(rows, k, dtype, extra=5, offset=1):
    """A matrix inside a larger one (rows `extra` further apart, starting at an odd element) and a check that the rest stays."""
    whole = torch.full((rows * (k + extra) + offset + 8,), 7.0, dtype=dtype, device="cuda")
    view = whole[offset:offset + rows * (k + extra)].view(rows, k + extra)[:, :k]
    rest = torch.ones_like(whole, dtype=torch.bool)
    rest[offset:offset + rows * (k + extra)].view(rows, k + extra)[:, :k] = False
    return view, lambda: bool((whole[rest] == 7.0).all())


def check_codes(q, want_codes, want_scales, fmt):
    assert np.array_equal(q.scales.cpu().numpy(), want_scales)
    assert np.array_equal(q.codes.cpu().numpy(), ref.pack(want_codes, fmt))


# ---- to 8 and 4 bits and back ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SIZES)
def test_quantise(hip, torch_cuda, rows, k, dtype, fmt):
    x = random_rows(rows, k, dtype, rows + k)
    q = hip.mx_quantize(x, fmt)
    check_codes(q, *ref.quantise(host(x), fmt), fmt)
    want = ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), fmt, k)
    for out_type in TYPES:
        got = host(hip.mx_dequantize(q, out_type))
        assert (np.abs(got - want) <= (np.abs(want) * HALF_ULP[out_type] + LEAST[out_type]) * (out_type == torch.float16)).all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantise_strides_and_alignment(hip, torch_cuda, dtype, fmt):
    for rows, k, extra, offset in ((9, 300, 3, 1), (4, 257, 0, 1), (3, 64, 1, 5)):
        x = random_rows(rows, k, dtype, 5)
        view, rest = guarded(rows, k, dtype, extra, offset)
        view.copy_(x)
        q = hip.mx_quantize(view, fmt)
        check_codes(q, *ref.quantise(host(x), fmt), fmt)
        view.fill_(3.0)
        hip.mx_dequantize(q, dtype, out=view)
        assert torch.equal(view, hip.mx_dequantize(q, dtype)) and rest()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_quantise_every_scale_tie_and_special(hip, torch_cuda, fmt):
    """A block for every exponent a float32 has, each holding the grid, the middles between its values and what saturates;
    subnormal numbers; blocks with a NaN, an infinity; zeros of both signs."""
    g = ref.grid(fmt)
    pool = np.concatenate([g, (g[1:] + g[:-1]) / 2, [ref.LARGEST[fmt] * 1.07, ref.LARGEST[fmt] * 1.1]])
    blocks = []
    for e in range(-149 - 8, 127 - 8):
        for part in range(0, len(pool), 31):
            b = np.zeros(32)
            b[1:1 + len(pool[part:part + 31])] = pool[part:part + 31] * np.where(np.arange(len(pool[part:part + 31])) % 2, 1, -1)
            b[0] = 2.0 ** ref.EMAX[fmt]
            blocks.append(b * 2.0 ** e)
    x = np.concatenate(blocks).astype(np.float32)
    x = np.concatenate([x, np.zeros(32, np.float32), -np.zeros(32, np.float32), np.float32([np.nan] + [1.0] * 31),
                        np.float32([1.0] * 31 + [-np.inf]), np.float32([3.4e38] * 32), np.float32([1e-45] * 32)])
    t = torch.from_numpy(x).cuda().view(1, -1)
    q = hip.mx_quantize(t, fmt)
    check_codes(q, *ref.quantise(x.astype(np.float64)[None], fmt), fmt)
    want = ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), fmt, len(x)).astype(np.float32)
    got = hip.mx_dequantize(q, torch.float32).cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)


def test_no_rows(hip, torch_cuda):
    for fmt in ("fp8", "fp4"):
        q = hip.mx_quantize(torch.empty(0, 77, device="cuda"), fmt)
        assert q.rows == 0 and hip.mx_dequantize(q).shape == (0, 77)
    w = torch.ones(77, device="cuda")
    q, h, rstd = hip.rms_norm_mx(torch.empty(0, 77, device="cuda"), w, residual=torch.empty(0, 77, device="cuda"))
    assert q.rows == 0 and h.shape == (0, 77) and rstd.shape == (0,)
    dx, dw = hip.rms_norm_backward(h, h, w, rstd)
    assert dx.shape == (0, 77) and bool((dw == 0).all())
    b = hip.mx_quantize(torch.randn(5, 77, device="cuda"), "fp4")
    assert hip.gemm_mx(q, b).shape == (0, 5)


def test_quantise_rows_past_32_bit_offsets(hip, torch_cuda):
    rows, k = 131200, 16400                             # 2.15 10^9 values, 4.3 GB
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = random_rows(3, k, torch.bfloat16, 1)
    q = hip.mx_quantize(x, "fp8")
    last = hip.MxTensor(q.codes[-3:], q.scales[-3:], "fp8", k)
    check_codes(last, *ref.quantise(host(x[-3:]), "fp8"), "fp8")
    x.fill_(1.0)
    hip.mx_dequantize(q, torch.bfloat16, out=x)
    assert torch.equal(x[-3:], hip.mx_dequantize(last)) and bool((x[:-3] == 0).all())


# ---- norm ------------------------------------------------------------------------------------------------------------

def check_norm(hip, q, h, rstd, x, residual, weight, eps):
    """h is the rounded sum; rstd and the 8-bit rows are near enough (see the top of the file)."""
    k = x.shape[1]
    want_h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    assert torch.equal(h, want_h)
    near = (k / 64 + 24) * EPS32
    want_r, y = ref.norm(host(h), host(weight), eps)
    assert (np.abs(host(rstd) - want_r) <= near * want_r).all()
    near += 4 * EPS32
    bytes_ = q.scales.cpu().numpy().astype(np.int64)
    low, high = (ref.scale_bytes(y * f, "fp8").astype(np.int64) for f in (1 - near, 1 + near))
    assert ((bytes_ >= low) & (bytes_ <= high)).all()
    got = ref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy(), "fp8", k)
    scale = np.repeat(2.0 ** (bytes_ - 127.0), 32, axis=1)[:, :k]
    inside = np.clip(y, -448 * scale, 448 * scale)
    step = scale * 2.0 ** (np.maximum(np.frexp(np.maximum(np.abs(got), np.abs(inside)) / scale)[1] - 1, -6) - 3)
    assert (np.abs(got - inside) <= step / 2 + near * np.abs(y)).all()
    assert not ref.unpack(q.codes.cpu().numpy(), "fp8")[:, k:].any()           # zeros behind k


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SIZES + [(700, 512), (1500, 96), (300, 4100), (5, 16384), (9, 33000)])
def test_norm(hip, torch_cuda, rows, k, dtype, residual):
    x = random_rows(rows, k, dtype, rows + k, 0.7)
    more = random_rows(rows, k, dtype, rows + k + 1, 0.7) if residual else None
    weight = random_rows(1, k, dtype, 3, 0.2)[0].contiguous()
    q, h, rstd = hip.rms_norm_mx(x, weight, residual=more, eps=1e-5)
    check_norm(hip, q, h, rstd, x, more, weight, 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(2048, 1025), (2051, 1536), (2047, 1536), (2049, 4100), (2048, 6144), (5, 8200), (40, 12288), (3, 12289)])
def test_norm_of_three_loads_to_a_thread(hip, torch_cuda, rows, k, dtype):
    test_norm(hip, torch_cuda, rows, k, dtype, True)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_in_place_and_strided(hip, torch_cuda, dtype):
    for rows, k in ((6, 300), (3, 2049), (2, 18001)):
        a, b = random_rows(rows, k, dtype, 1, 0.5), random_rows(rows, k, dtype, 2, 0.5)
        weight = random_rows(1, k, dtype, 3, 0.2)[0].contiguous()
        want = hip.rms_norm_mx(a, weight, residual=b)
        for into in ("x", "residual", "other"):
            (x, rx), (r, rr), (o, ro) = guarded(rows, k, dtype), guarded(rows, k, dtype, 2, 3), guarded(rows, k, dtype, 9, 2)
            x.copy_(a), r.copy_(b)
            q, h, rstd = hip.rms_norm_mx(x, weight, residual=r, h={"x": x, "residual": r, "other": o}[into])
            assert torch.equal(h, want[1]) and torch.equal(q.codes, want[0].codes) and torch.equal(q.scales, want[0].scales)
            assert torch.equal(rstd, want[2]) and rx() and rr() and ro()


def test_norm_of_zeros_infinities_and_nan(hip, torch_cuda):
    k = 300
    x = torch.ones(5, k, device="cuda")
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    x[4] = 1e30                                                                # squares past float32: 1 / rms is 0
    q, h, rstd = hip.rms_norm_mx(x, torch.ones(k, device="cuda"), eps=0.0)
    v = hip.mx_dequantize(q, torch.float32).cpu().numpy()
    assert (v[0] == 1).all() and np.isnan(v[2]).all() and np.isnan(v[3, :32]).all() and (v[3, 32:] == 0).all() and (v[4] == 0).all()
    assert np.isnan(v[1]).all()                                                # 0 / 0 with no eps
    assert not q.codes[:, k:].any()
    q, _, rstd = hip.rms_norm_mx(x, torch.ones(k, device="cuda"), eps=1e-6)
    assert not q.codes[1].any() and abs(float(rstd[1]) - 1e3) < 1e-2


# ---- gradient --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("with_dh", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SIZES + [(1100, 512), (1500, 96), (600, 4100), (5, 16384)])
def test_norm_backward(hip, torch_cuda, rows, k, dtype, with_dh):
    h, dy = random_rows(rows, k, dtype, 1, 0.5), random_rows(rows, k, dtype, 2, 0.5)
    dh = random_rows(rows, k, dtype, 3, 0.5) if with_dh else None
    weight = random_rows(1, k, dtype, 4, 0.2)[0].contiguous()
    rstd = torch.rsqrt(h.float().pow(2).mean(1) + 1e-6)
    dx, dw = hip.rms_norm_backward(dy, h, weight, rstd, dh=dh)
    args = (host(dy), host(h), host(weight), host(rstd), None if dh is None else host(dh))
    want_dx, want_dw = ref.norm_backward(*args)
    n, g, r = args[1] * args[3][:, None], args[2] * args[0], args[3][:, None]
    size = r * (np.abs(g) + np.abs(n) * np.abs(n * g).mean(1, keepdims=True)) + (0 if dh is None else np.abs(args[4]))
    assert (np.abs(host(dx) - want_dx) <= (k / 64 + 24) * EPS32 * size + HALF_ULP[dtype] * np.abs(want_dx) + LEAST[dtype]).all()
    assert (np.abs(host(dw) - want_dw) <= (rows + 4) * EPS32 * np.abs(args[0] * n).sum(0)).all()
    assert torch.equal(dw, hip.rms_norm_backward(dy, h, weight, rstd, dh=dh)[1])    # the same bits again


def test_norm_backward_against_differences(hip, torch_cuda):
    """The gradient along random directions against central differences of sum(dy norm(h)) in float64: the formula's third
    derivative times step^2 is below 1e-7 of it at a step of 1e-4."""
    rows, k, eps = 5, 300, 1e-3
    h, dy, weight = random_rows(rows, k, torch.float32, 1, 0.3), random_rows(rows, k, torch.float32, 2, 0.3), random_rows(1, k, torch.float32, 3, 0.2)[0]
    rstd = hip.rms_norm_mx(h, weight, eps=eps)[2]
    dx, dw = hip.rms_norm_backward(dy, h, weight, rstd)
    f = lambda a, w: (host(dy) * ref.norm(a, w, eps)[1]).sum()  # noqa: E731
    rng, step = np.random.default_rng(0), 1e-4
    for _ in range(6):
        d, e = rng.normal(size=(rows, k)), rng.normal(size=k)
        along_h = (f(host(h) + step * d, host(weight)) - f(host(h) - step * d, host(weight))) / (2 * step)
        along_w = (f(host(h), host(weight) + step * e) - f(host(h), host(weight) - step * e)) / (2 * step)
        assert abs((host(dx) * d).sum() - along_h) <= 1e-5 * np.abs(host(dx) * d).sum()
        assert abs((host(dw) * e).sum() - along_w) <= 1e-5 * np.abs(host(dw) * e).sum()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1024, 1025), (1030, 1536), (1023, 1536), (2051, 1100), (5, 8200), (40, 12288), (3, 12289)])
def test_norm_backward_of_three_loads_to_a_thread(hip, torch_cuda, rows, k, dtype):
    test_norm_backward(hip, torch_cuda, rows, k, dtype, True)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_backward_strided_and_in_place(hip, torch_cuda, dtype):
    for rows, k in ((7, 300), (3, 2049), (530, 65)):
        h, dy, dh = (random_rows(rows, k, dtype, s, 0.5) for s in (1, 2, 3))
        weight = random_rows(1, k, dtype, 4, 0.2)[0].contiguous()
        rstd = torch.rsqrt(h.float().pow(2).mean(1) + 1e-6)
        want = hip.rms_norm_backward(dy, h, weight, rstd, dh=dh)
        for into in ("dy", "dh", "other"):
            views = [guarded(rows, k, dtype, e, o) for e, o in ((5, 1), (0, 3), (2, 2), (7, 5))]
            (vh, _), (vy, _), (vd, _), (vo, _) = views
            vh.copy_(h), vy.copy_(dy), vd.copy_(dh)
            dx, dw = hip.rms_norm_backward(vy, vh, weight, rstd, dh=vd, out={"dy": vy, "dh": vd, "other": vo}[into])
            assert torch.equal(dx, want[0]) and torch.equal(dw, want[1]) and all(rest() for _, rest in views)


# ---- products --------------------------------------------------------------------------------------------------------

def operands(hip, m, n, k, fmt, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    a, b = (torch.empty(r, k, device="cuda").normal_(generator=g) for r in (m, n))
    a = a * torch.where(torch.rand(k, device="cuda", generator=g) < 0.02, 20.0, 1.0)
    b = b * torch.exp(torch.empty(n, 1, device="cuda").normal_(0, 0.5, generator=g))
    return hip.mx_quantize(a, fmt), hip.mx_quantize(b, "fp4")


def check_product(hip, c, a, b, bias, relu, rows=None):
    """C (all rows or those asked for) against float64 on the GPU."""
    pick = slice(None) if rows is None else rows
    va = hip.mx_dequantize(a, torch.float32)[pick].double()
    vb = hip.mx_dequantize(b, torch.float32).double()
    want, size = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    if relu:
        want = want.clamp(min=0)
    off = (a.k + 2) * EPS32 if a.fmt == "fp4" else 2.0 ** -13 + (a.k + 2) * EPS32
    bound = off * size + HALF_ULP[c.dtype] * (want.abs() + off * size) + LEAST[c.dtype]
    assert bool(((c[pick].double() - want).abs() <= bound).all())


PRODUCTS = [(1, 1, 1), (1, 5, 33), (2, 16, 256), (3, 17, 257), (5, 100, 100), (16, 16, 512), (17, 31, 1000), (33, 65, 300), (61, 1007, 4095),
            (64, 256, 256), (65, 130, 2100), (100, 250, 64), (129, 257, 513), (200, 875, 1932), (255, 300, 700), (300, 520, 1300),
            (257, 1025, 260), (513, 770, 1537), (1000, 64, 900), (1, 8192, 2048), (8, 4099, 11008), (1030, 1290, 512)]


@pytest.mark.parametrize("fmt,dtype", [("fp8", torch.bfloat16), ("fp8", torch.float16), ("fp4", torch.bfloat16), ("fp4", torch.float16),
                                       ("fp4", torch.float32)])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(hip, torch_cuda, m, n, k, fmt, dtype):
    a, b = operands(hip, m, n, k, fmt, m + n + k)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    bias = torch.empty(n, device="cuda").normal_(0, 3, generator=g)
    for use_bias, relu in ((False, False), (True, True), (True, False), (False, True)):
        c, rest = guarded(m, n, dtype, *((5, 1) if relu else (0, 0)))
        got = hip.gemm_mx(a, b, bias=bias if use_bias else None, relu=relu, dtype=dtype, out=c)
        check_product(hip, got, a, b, bias if use_bias else None, relu)
        assert rest()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("m,n,k", [(4095, 11008, 1024), (2048, 2048, 4096), (4100, 4100, 300), (1, 4096, 16384), (130, 16384, 1000)])
def test_large_products(hip, torch_cuda, m, n, k, fmt):
    a, b = operands(hip, m, n, k, fmt)
    bias = torch.randn(n, device="cuda")
    c = hip.gemm_mx(a, b, bias=bias, relu=True)
    check_product(hip, c, a, b, bias, True, rows=torch.randint(0, m, (600,), device="cuda") if m > 600 else None)
    assert torch.equal(c, hip.gemm_mx(a, b, bias=bias, relu=True))             # the same bits again


@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_of_undefined_blocks(hip, torch_cuda, m):
    """A block that stands for NaNs makes NaN of its row (of A) or its column (of B) and of nothing else; ReLU keeps it."""
    n, k = 300, 700
    for fmt in ("fp8", "fp4"):
        x = torch.randn(m, k, device="cuda")
        w = torch.randn(n, k, device="cuda")
        x[m // 2, 601], w[17, 5] = float("nan"), float("inf")
        c = hip.gemm_mx(hip.mx_quantize(x, fmt), hip.mx_quantize(w, "fp4"), relu=True)
        want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        want[m // 2], want[:, 17] = True, True
        assert torch.equal(torch.isnan(c), want)


@pytest.mark.parametrize("m", [1, 70])
def test_product_weights_past_32_bit_offsets(hip, torch_cuda, m):
    n, k = (1 << 20) + 40, 4096                          # 2.1 GB of codes
    codes = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    tail = hip.mx_quantize(torch.randn(300, k, device="cuda"), "fp4")
    scales = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    codes[-300:], scales[-300:] = tail.codes, tail.scales
    a = hip.mx_quantize(torch.randn(m, k, device="cuda"), "fp8")
    c = hip.gemm_mx(a, hip.MxTensor(codes, scales, "fp4", k))
    check_product(hip, c[:, -300:], a, tail, None, False)
    assert not c[:, :-300].any()


def test_streams_and_graphs(hip, torch_cuda):
    """The layer's calls on a stream of their own, then captured once and replayed between eager calls."""
    k, n = 1000, 777
    x, r, w = random_rows(37, k, torch.bfloat16, 1, 0.5), random_rows(37, k, torch.bfloat16, 2, 0.5), random_rows(1, k, torch.bfloat16, 3, 0.1)[0]
    b = hip.mx_quantize(torch.randn(n, k, device="cuda") * 0.05, "fp4")
    dy = random_rows(37, k, torch.bfloat16, 4, 0.5)

    def step():
        q, h, rstd = hip.rms_norm_mx(x, w, residual=r)
        c = hip.gemm_mx(q, b, relu=True)
        return [h, rstd, c, hip.mx_dequantize(hip.mx_quantize(c, "fp4"))] + list(hip.rms_norm_backward(dy, h, w, rstd, dh=h))
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        x.copy_(random_rows(37, k, torch.bfloat16, 10 + turn, 0.5))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(held, eager))


# ---- the layer -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,inner", [(1, 300, 777), (16, 512, 1000), (300, 256, 520)])
def test_feed_forward(hip, torch_cuda, rows, k, inner, dtype):
    """The layer is its operators one after the other; its gradients are those of the layer with the ReLU's choices it made and
    no rounding to 8 bits: three roundings to the type on the way (2^-9 of a value each in bf16), within 2 % of their norms."""
    from spoc_amd.feed_forward import MxFeedForward
    x, res = random_rows(rows, k, dtype, 1, 0.3), random_rows(rows, k, dtype, 2, 0.3)
    weight = (1 + random_rows(1, k, dtype, 3, 0.1)[0].float() * 0.1).to(dtype)
    up, down = hip.mx_quantize(torch.randn(inner, k, device="cuda") * 0.05, "fp4"), hip.mx_quantize(torch.randn(k, inner, device="cuda") * 0.05, "fp4")
    up_bias, down_bias = torch.randn(inner, device="cuda") * 0.1, torch.randn(k, device="cuda") * 0.1
    layer = MxFeedForward(weight, up, down, up_bias, down_bias)
    y, h, kept = layer.train(x, res)
    q, h2, rstd = hip.rms_norm_mx(x, weight, residual=res)
    u = hip.gemm_mx(q, up, bias=up_bias, relu=True, dtype=dtype)
    assert torch.equal(h, h2) and torch.equal(y, hip.gemm_mx(hip.mx_quantize(u, "fp8"), down, bias=down_bias, dtype=dtype))
    assert all(torch.equal(a, b) for a, b in zip(layer(x, res), (y, h)))
    dy, dh = random_rows(rows, k, dtype, 5, 0.3), random_rows(rows, k, dtype, 6, 0.3)
    got = layer.backward(kept, dy, dh)
    leaf = {n: t.double().detach().clone().requires_grad_() for n, t in (("dx", h), ("dweight", weight), ("dup_bias", up_bias), ("ddown_bias", down_bias))}
    n = leaf["dx"] * torch.rsqrt(leaf["dx"].pow(2).mean(1, keepdim=True) + 1e-6) * leaf["dweight"]
    wu, wd = (hip.mx_dequantize(t, torch.float32).double() for t in (up, down))
    out = ((n @ wu.t() + leaf["dup_bias"]) * (kept[2] > 0)) @ wd.t() + leaf["ddown_bias"]
    ((out * dy.double()).sum() + (leaf["dx"] * dh.double()).sum()).backward()
    for name, t in leaf.items():
        assert float((got[name].double() - t.grad).norm()) <= 0.02 * float(t.grad.norm()), name
    with pytest.raises(ValueError):
        MxFeedForward(weight, down, down)
    with pytest.raises(TypeError):
        MxFeedForward(weight.float(), up, down)


def test_feed_forward_command(hip, torch_cuda, capsys):
    from spoc_amd import feed_forward
    assert feed_forward.main(["5", "300", "700"]) == 0
    assert "gradients" in capsys.readouterr().out


def test_refusals_on_the_device(hip, torch_cuda):
    x = torch.randn(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    q8, q4 = hip.mx_quantize(x, "fp8"), hip.mx_quantize(x, "fp4")
    for error, call in [
            (ValueError, lambda: hip.mx_quantize(x, "fp6")), (TypeError, lambda: hip.mx_quantize(x.t(), "fp8")),
            (TypeError, lambda: hip.mx_quantize(x.double(), "fp8")), (TypeError, lambda: hip.mx_quantize(x[0], "fp8")),
            (ValueError, lambda: hip.mx_quantize(x, "fp8", out=q4)), (TypeError, lambda: hip.mx_dequantize(q8, torch.float64)),
            (ValueError, lambda: hip.mx_dequantize(hip.MxTensor(q8.codes, q8.scales, "fp4", 64))),
            (ValueError, lambda: hip.mx_dequantize(q8, torch.float32, out=torch.empty(4, 65, device="cuda"))),
            (TypeError, lambda: hip.rms_norm_mx(x, w.half())), (ValueError, lambda: hip.rms_norm_mx(x, w[:63].contiguous())),
            (ValueError, lambda: hip.rms_norm_mx(x, w, residual=x[:3])), (TypeError, lambda: hip.rms_norm_mx(x, w, residual=x.half())),
            (hip.SarekHipError, lambda: hip.rms_norm_mx(x, w, eps=-1.0)),
            (ValueError, lambda: hip.rms_norm_backward(x, x, w, torch.ones(3, device="cuda"))),
            (TypeError, lambda: hip.rms_norm_backward(x.half(), x, w, torch.ones(4, device="cuda"))),
            (ValueError, lambda: hip.gemm_mx(q4, q8)), (ValueError, lambda: hip.gemm_mx(q4, hip.mx_quantize(x[:, :63], "fp4"))),
            (TypeError, lambda: hip.gemm_mx(q4, q4, dtype=torch.float64)), (hip.SarekHipError, lambda: hip.gemm_mx(q8, q4, dtype=torch.float32)),
            (ValueError, lambda: hip.gemm_mx(q4, q4, bias=w)), (TypeError, lambda: hip.gemm_mx(q4, q4, bias=torch.ones(4, device="cuda").half())),
            (ValueError, lambda: hip.gemm_mx(q4, q4, out=torch.empty(4, 5, device="cuda", dtype=torch.bfloat16)))]:
        with pytest.raises(error):
            call()
