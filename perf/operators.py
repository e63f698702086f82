"""The operators of a feed-forward layer in microscaled 8- and 4-bit floating point, as a list of cases that can be timed.

An operator is called as a program calls it: `hip.rms_norm_mx` (residual's addition, root-mean-square norm, 8-bit output
with a scale for each 32 values), `hip.rms_norm_backward`, `hip.mx_quantize` and `hip.mx_dequantize`, `hip.gemm_mx` (8- or
4-bit rows times 4-bit weights), and `feed_forward.MxFeedForward`, which runs them one after the other.  With `own = False`
the same outputs come from elementary torch operations in 32 bits.

Sizes come from the 16-bit products that this library is measured on (4095 x 11008 x 4096 with its epilogue, 8192^3, 16 rows
against 8192 x 8192) and from the odd ones its kernels are tested at; between them they are drawn.
"""
import math

import torch

own = False

F32 = torch.float32
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 32            # values that share a scale
ROW = 256             # rows of codes are padded with zeros to a whole number of these
EMAX = {"fp8": 8, "fp4": 2}              # exponent of the largest value: 448 = 1.75 2^8, 6 = 1.5 2^2
EMIN = {"fp8": -6, "fp4": 0}             # exponent of the smallest normal one
BITS = {"fp8": 3, "fp4": 1}              # of the mantissa
LARGEST = {"fp8": 448.0, "fp4": 6.0}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


def listed():
    return [
        # the norm in front of a layer while one token is generated: what a launch costs
        dict(name="norm_one_token", op="norm", rows=1, k=4096, dtype="bf16", residual=True),
        # the same for a prompt: one read of both inputs, one write of the sum and of the 8-bit rows
        dict(name="norm_prompt", op="norm", rows=4095, k=4096, dtype="bf16", residual=True),
        # 32-bit rows of an odd length, no residual
        dict(name="norm_odd_rows_f32", op="norm", rows=999, k=11007, dtype="f32", residual=False),
        # a training step's norm, backwards: a small batch of odd rows
        dict(name="norm_backward_small", op="norm_backward", rows=61, k=1001, dtype="f16", residual=False),
        # and a large one, with the gradient that comes down the residual stream
        dict(name="norm_backward_large", op="norm_backward", rows=8192, k=4096, dtype="bf16", residual=True),
        # a layer's weights, brought to 4 bits once
        dict(name="quantise_weights", op="quantise", rows=11008, k=4096, dtype="bf16", fmt="fp4"),
        # a few tokens' activations, brought to 8 bits before the second product
        dict(name="quantise_few_rows", op="quantise", rows=16, k=11008, dtype="f16", fmt="fp8"),
        # one token against a square of weights: the weights have to be read, little else
        dict(name="product_one_token", op="product", m=1, n=8192, k=8192, fmt="fp8", out="bf16", bias=False, relu=False),
        # a batch of tokens, sizes that are nobody's multiples
        dict(name="product_batch_odd", op="product", m=61, n=11007, k=4095, fmt="fp8", out="f16", bias=True, relu=True),
        # a prompt through the first product of a layer, with its bias and ReLU
        dict(name="product_prompt", op="product", m=4095, n=11008, k=4096, fmt="fp8", out="bf16", bias=True, relu=True),
        # both operands in 4 bits
        dict(name="product_fp4_8192", op="product", m=8192, n=8192, k=8192, fmt="fp4", out="f32", bias=False, relu=False),
        # the layer: norm, product, ReLU, 8 bits again, product, for the tokens of a small batch
        dict(name="feed_forward_16", op="feed_forward", rows=16, k=4096, inner=11008, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform over [lo, hi]; every second one rounded to a multiple of 64 where it can be."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 256:
        v = v // 64 * 64
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_backward", "quantise", "product", "product", "product", "product", "feed_forward"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    while True:
        if op in ("norm", "norm_backward"):
            c = dict(op=op, rows=_log(rng, 1, 8192), k=_log(rng, 40, 16384), dtype=dtype, residual=rng.random() < 0.5)
            if c["rows"] * c["k"] <= 8192 * 4096:
                return c
        elif op == "quantise":
            c = dict(op=op, rows=_log(rng, 1, 11008), k=_log(rng, 40, 16384), dtype=dtype, fmt=rng.choice(["fp8", "fp4"]))
            if c["rows"] * c["k"] <= 11008 * 4096:
                return c
        elif op == "product":
            fmt = rng.choice(["fp8", "fp4"])      # products with 8-bit rows go to 16 bits
            c = dict(op=op, m=_log(rng, 1, 8192), n=_log(rng, 64, 16384), k=_log(rng, 64, 16384), fmt=fmt,
                     out=dtype if fmt == "fp4" else rng.choice(["bf16", "f16"]), bias=rng.random() < 0.5, relu=rng.random() < 0.5)
            if c["m"] * c["n"] * c["k"] <= 8192 ** 3 // 2:
                return c
        else:
            c = dict(op=op, rows=_log(rng, 1, 4096), k=_log(rng, 256, 8192), inner=_log(rng, 256, 16384),
                     dtype=rng.choice(["bf16", "f16"]))
            if c["rows"] * c["k"] * c["inner"] <= 8192 ** 3 // 8:
                return c


def _up(a, b):
    return (a + b - 1) // b * b


# ---- the plain form: 32 bits, elementary operations ------------------------------------------------------------------

def _power(e):
    """2^e for whole e in [-127, 127], from the bits."""
    return torch.where(e > -127, ((e + 127) << 23).view(F32), torch.full((), 2.0 ** -127, dtype=F32, device=e.device))


def _exponent(v):
    """floor(log2 v) of v >= 0, -127 for what is below the smallest normal number."""
    return (v.view(torch.int32) >> 23) - 127


def _blocks(y):
    """[rows, k] -> [rows, blocks, 32], zeros behind k."""
    rows, k = y.shape
    return torch.nn.functional.pad(y, (0, _up(k, ROW) - k)).view(rows, -1, BLOCK)


def _round_mx(y, fmt):
    """The nearest 8- or 4-bit values times 2^-e, and e, of each block: e from the block's largest value, ties to even."""
    y = _blocks(y)
    e = (_exponent(y.abs().amax(-1, keepdim=True)) - EMAX[fmt]).clamp(min=-127)
    q = y * _power(-e)
    step = _power(_exponent(q.abs()).clamp(min=EMIN[fmt]) - BITS[fmt])
    return (torch.round(q / step) * step).clamp(-LARGEST[fmt], LARGEST[fmt]), e


def _quantised(y, fmt):
    """The values that y's 8- or 4-bit form stands for."""
    q, e = _round_mx(y, fmt)
    return (q * _power(e)).view(y.shape[0], -1)[:, :y.shape[1]]


def _codes(y, fmt):
    """(codes, scales) of a matrix as a program keeps them: rows of 8-bit codes, or two 4-bit ones to a byte (the first in
    the low half), and a byte e + 127 for each 32 of them; both run over the padded row."""
    q, e = _round_mx(y, fmt)
    q = q.view(y.shape[0], -1)
    if fmt == "fp8":
        c = q.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        code = torch.searchsorted(torch.tensor(E2M1, device=q.device), q.abs()).to(torch.uint8)
        code = code | (torch.signbit(q).to(torch.uint8) << 3)
        c = code[:, 0::2] | (code[:, 1::2] << 4)
    return c.contiguous(), (e.view(y.shape[0], -1) + 127).to(torch.uint8)


def _values(codes, scales, fmt, k):
    """What codes and scales stand for, in 32 bits."""
    if fmt == "fp8":
        v = codes.view(torch.float8_e4m3fn).to(F32)
    else:
        table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
        v = table[torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1).to(torch.int32)]
    v = v.view(codes.shape[0], -1, BLOCK) * _power(scales.to(torch.int32) - 127).unsqueeze(-1)
    return v.view(codes.shape[0], -1)[:, :k]


def _norm(x, residual, weight):
    """The sum in x's type, its rows' 1 / root mean square, and the norm in 32 bits."""
    h = x if residual is None else (x.to(F32) + residual.to(F32)).to(x.dtype)
    h32 = h.to(F32)
    rstd = torch.rsqrt((h32 * h32).mean(-1) + EPS)
    return h, rstd, h32 * rstd[:, None] * weight.to(F32)


def _product(a, b, bias, relu):
    c = a @ b.t()
    if bias is not None:
        c = c + bias
    return c.clamp(min=0) if relu else c


# ---- what a program has before the call ------------------------------------------------------------------------------

def _normal(gen, std, *shape):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=gen)


def _rows(gen, rows, k):
    """Activations: normal, with a few features that are much larger than the others, as layers have them."""
    x = _normal(gen, 1.0, rows, k)
    return x * torch.where(torch.rand(k, device="cuda", generator=gen) < 0.01, 20.0, 1.0)


def _weight(gen, k, dtype):
    return (1 + _normal(gen, 0.1, k)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, s = case["op"], dict(case)
    if op in ("norm", "norm_backward"):
        rows, k, dtype = case["rows"], case["k"], TYPES[case["dtype"]]
        more = (lambda: _rows(gen, rows, k).to(dtype)) if case["residual"] else (lambda: None)
        s.update(x=_rows(gen, rows, k).to(dtype), weight=_weight(gen, k, dtype), more=more())
        if op == "norm_backward":
            x32 = s["x"].to(F32)
            s.update(dy=_normal(gen, 1e-2, rows, k).to(dtype), rstd=torch.rsqrt((x32 * x32).mean(-1) + EPS))
    elif op == "quantise":
        s.update(x=_rows(gen, case["rows"], case["k"]).to(TYPES[case["dtype"]]))
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s.update(a=_codes(_rows(gen, m, k), case["fmt"]), b=_codes(_normal(gen, 0.02, n, k), "fp4"),
                 bias_row=_normal(gen, 0.1, n) if case["bias"] else None)
    else:
        rows, k, inner, dtype = case["rows"], case["k"], case["inner"], TYPES[case["dtype"]]
        s.update(x=_normal(gen, 1.0, rows, k).to(dtype), more=_rows(gen, rows, k).to(dtype), weight=_weight(gen, k, dtype),
                 up=_codes(_normal(gen, 0.02, inner, k), "fp4"), down=_codes(_normal(gen, 0.02, k, inner), "fp4"),
                 up_bias=_normal(gen, 0.1, inner), down_bias=_normal(gen, 0.1, k))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    op = s["op"]
    if op == "norm":
        h, rstd, y = _norm(s["x"], s["more"], s["weight"])
        return {"h": h, "rstd": rstd, "y": _quantised(y, "fp8").to(torch.bfloat16)}
    if op == "norm_backward":
        h, w, dy, r = s["x"].to(F32), s["weight"].to(F32), s["dy"].to(F32), s["rstd"][:, None]
        n, g = h * r, w * dy
        dx = r * (g - n * (n * g).mean(-1, keepdim=True))
        if s["more"] is not None:
            dx = dx + s["more"].to(F32)
        return {"dx": dx.to(s["x"].dtype), "dweight": (dy * n).sum(0)}
    if op == "quantise":
        return _quantised(s["x"].to(F32), s["fmt"]).to(torch.bfloat16)
    if op == "product":
        a, b = _values(*s["a"], s["fmt"], s["k"]), _values(*s["b"], "fp4", s["k"])
        return _product(a, b, s["bias_row"], s["relu"]).to(TYPES[s["out"]])
    h, _, y = _norm(s["x"], s["more"], s["weight"])
    dtype = h.dtype
    u = _product(_quantised(y, "fp8"), _values(*s["up"], "fp4", s["k"]), s["up_bias"], True).to(dtype)
    out = _product(_quantised(u.to(F32), "fp8"), _values(*s["down"], "fp4", s["inner"]), s["down_bias"], False).to(dtype)
    return {"y": out, "h": h}


def _run_own(s):
    from spoc_amd import feed_forward, hip
    op = s["op"]
    if op == "norm":
        q, h, rstd = hip.rms_norm_mx(s["x"], s["weight"], residual=s["more"], eps=EPS)
        return {"h": h, "rstd": rstd, "y": hip.mx_dequantize(q)}
    if op == "norm_backward":
        dx, dweight = hip.rms_norm_backward(s["dy"], s["x"], s["weight"], s["rstd"], dh=s["more"])
        return {"dx": dx, "dweight": dweight}
    if op == "quantise":
        return hip.mx_dequantize(hip.mx_quantize(s["x"], s["fmt"]))
    if op == "product":
        return hip.gemm_mx(hip.MxTensor(*s["a"], s["fmt"], s["k"]), hip.MxTensor(*s["b"], "fp4", s["k"]), bias=s["bias_row"],
                           relu=s["relu"], dtype=TYPES[s["out"]])
    layer = feed_forward.MxFeedForward(s["weight"], hip.MxTensor(*s["up"], "fp4", s["k"]), hip.MxTensor(*s["down"], "fp4", s["inner"]),
                                       up_bias=s["up_bias"], down_bias=s["down_bias"], eps=EPS)
    y, h = layer(s["x"], s["more"])
    return {"y": y, "h": h}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def _held(rows, k, fmt):
    """Bytes of a matrix in 8 or 4 bits, its scales among them."""
    return rows * k // (1 if fmt == "fp8" else 2) + rows * -(-k // BLOCK)


def work(case):
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=_held(m, k, case["fmt"]) + _held(n, k, "fp4") + m * n * TYPES[case["out"]].itemsize + (4 * n if case["bias"] else 0),
                    flops=2 * m * n * k)
    rows, k, size = case["rows"], case["k"], TYPES[case["dtype"]].itemsize
    if op == "norm":            # x, the residual, the weight; the sum where there is a residual, 8-bit rows, their values, 1 / rms
        return dict(bytes=rows * k * size * (3 if case["residual"] else 1) + k * size + _held(rows, k, "fp8") + rows * k * 2 + rows * 4,
                    flops=8 * rows * k)
    if op == "norm_backward":   # dy, the sum, the gradient from above, the weight, 1 / rms; dx, the weight's gradient
        return dict(bytes=rows * k * size * (4 if case["residual"] else 3) + k * (size + 4) + rows * 4, flops=12 * rows * k)
    if op == "quantise":        # the matrix; its codes and the values that they stand for
        return dict(bytes=rows * k * size + _held(rows, k, case["fmt"]) + rows * k * 2, flops=4 * rows * k)
    inner = case["inner"]
    return dict(bytes=4 * rows * k * size + k * size + _held(inner, k, "fp4") + _held(k, inner, "fp4") + 4 * (k + inner),
                flops=4 * rows * k * inner)


# ---- the same from the definition, in 64 bits ------------------------------------------------------------------------

def _two64(e):
    """2^e in 64 bits for whole e, from the bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _mx64(y, fmt):
    """[rows, k] in 64 bits -> the nearest values of its blocks' grids: the grid's magnitudes in order, the middle between
    two neighbours going to the one with the even index (whose last mantissa bit is 0)."""
    rows, k = y.shape
    top, low, bits = EMAX[fmt], EMIN[fmt], BITS[fmt]
    small = [j * 2.0 ** (low - bits) for j in range(2 ** bits)]
    grid = small + [(1 + j / 2 ** bits) * 2.0 ** e for e in range(low, top + 1) for j in range(2 ** bits)]
    grid = torch.tensor([g for g in grid if g <= LARGEST[fmt]], dtype=torch.float64, device=y.device)
    mid = (grid[1:] + grid[:-1]) / 2
    whole = torch.zeros(rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=y.device)
    whole[:, :k] = y
    z = whole.reshape(rows, -1, BLOCK)
    most = z.abs().max(-1, keepdim=True).values
    scale = _two64(torch.where(most > 0, torch.frexp(most).exponent - 1 - top, -127).clamp(min=-127))
    v = (z / scale).abs().contiguous()
    below, above = torch.searchsorted(mid, v), torch.searchsorted(mid, v, right=True)
    at = torch.where((below != above) & (below % 2 == 1), above, below)
    return (torch.sign(z) * grid[at] * scale).reshape(rows, -1)[:, :k]


def _held64(codes, scales, fmt, k):
    """What codes and scales stand for, decoded bit by bit in 64 bits."""
    c = codes.to(torch.int64)
    if fmt == "fp4":
        c = torch.stack((c % 16, c // 16), dim=-1).reshape(codes.shape[0], -1)
    bits, width = (3, 4) if fmt == "fp8" else (1, 2)
    mantissa, exponent = (c % 2 ** bits).double(), (c // 2 ** bits) % 2 ** width
    bias = 7 if fmt == "fp8" else 1
    v = torch.where(exponent > 0, (1 + mantissa / 2 ** bits) * _two64(exponent - bias), mantissa / 2 ** bits * 2.0 ** (1 - bias))
    v = torch.where(c // 2 ** (bits + width) == 1, -v, v)
    return (v * _two64(scales.to(torch.int64) - 127).repeat_interleave(BLOCK, dim=1))[:, :k]


def _norm64(x, residual, weight):
    """The sum, and the norm of the sum as the type holds it."""
    h = x.double() + (0 if residual is None else residual.double())
    held = h.to(x.dtype).double()
    rstd = 1 / torch.sqrt(held.pow(2).mean(dim=1) + EPS)
    return h, rstd, held * rstd.unsqueeze(1) * weight.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "norm":
        h, rstd, y = _norm64(s["x"], s["more"], s["weight"])
        return {"h": h, "rstd": rstd, "y": _mx64(y, "fp8")}
    if op == "norm_backward":
        # y_j = w_j h_j r, r = (mean h^2 + eps)^-1/2: dr/dh_j = -r^3 h_j / k
        h, dy, r, w = s["x"].double(), s["dy"].double(), s["rstd"].double(), s["weight"].double()
        along = torch.mv(h * dy, w)
        dx = dy * w * r.unsqueeze(1) - h * (r ** 3 * along / case["k"]).unsqueeze(1)
        return {"dx": dx if s["more"] is None else dx + s["more"].double(), "dweight": torch.mv((dy * h).t(), r)}
    if op == "quantise":
        return _mx64(s["x"].double(), s["fmt"])
    if op == "product":
        c = torch.mm(_held64(*s["a"], s["fmt"], s["k"]), _held64(*s["b"], "fp4", s["k"]).t())
        if s["bias_row"] is not None:
            c += s["bias_row"].double()
        return torch.relu(c) if s["relu"] else c
    dtype = s["x"].dtype
    h, _, y = _norm64(s["x"], s["more"], s["weight"])
    u = torch.relu(torch.mm(_mx64(y, "fp8"), _held64(*s["up"], "fp4", s["k"]).t()) + s["up_bias"].double())
    out = torch.mm(_mx64(u.to(dtype).double(), "fp8"), _held64(*s["down"], "fp4", s["inner"]).t()) + s["down_bias"].double()
    return {"y": out, "h": h}
