"""The feed-forward layer of a transformer block on microscaled matrices: the residual's addition and the root-mean-square
norm, a product with 4-bit weights, its bias and ReLU, 8 bits again, a second product.

    python -m spoc_amd.feed_forward [tokens] [width] [inner]    # one pass each way on random data, both checked against float64
"""
import torch

from . import hip


class MxFeedForward:
    """y = down(relu(up(norm(x + residual)))) with `up` [inner, width] and `down` [width, inner] held in 4 bits (MxTensor "fp4",
    from hip.mx_quantize(weights, "fp4")), float32 biases and a norm weight in the activations' type (bfloat16 or float16).

    Calling it serves a few tokens or a prompt; `train` keeps what `backward` needs.  The 4-bit weights stay as they are in
    training; gradients go to the inputs, to the norm's weight and to the biases, with every rounding to 8 bits taken as
    the identity."""

    def __init__(self, weight, up, down, up_bias=None, down_bias=None, eps=1e-6):
        if (up.rows, up.k) != (down.k, down.rows) or weight.shape != (up.k,):
            raise ValueError(f"MxFeedForward: up is {up.rows} x {up.k}, down {down.rows} x {down.k}, the norm's weight {tuple(weight.shape)}")
        if weight.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("MxFeedForward: activations are bfloat16 or float16")
        self.weight, self.up, self.down, self.up_bias, self.down_bias, self.eps = weight, up, down, up_bias, down_bias, eps

    def __call__(self, x, residual=None):
        """(y, h): the layer's output and h = x + residual, to which the caller's next layer adds it."""
        return self.train(x, residual)[:2]

    def train(self, x, residual=None):
        """(y, h, kept): as the call, and what backward() takes."""
        q, h, rstd = hip.rms_norm_mx(x, self.weight, residual=residual, eps=self.eps)
        u = hip.gemm_mx(q, self.up, bias=self.up_bias, relu=True, dtype=x.dtype)
        y = hip.gemm_mx(hip.mx_quantize(u, "fp8"), self.down, bias=self.down_bias, dtype=x.dtype)
        return y, h, (h, rstd, u)

    def backward(self, kept, dy, dh=None):
        """Gradients for dy (of y) and dh (of h, None where nothing else uses it): a dict of dx (x's and the residual's),
        dweight, dup_bias and ddown_bias.  The products go over the weights' values in 16 bits."""
        h, rstd, u = kept
        du = _product(dy.contiguous(), hip.mx_dequantize(self.down, h.dtype)).masked_fill_(u <= 0, 0)   # (adjacent rows for the products)
        dn = _product(du.to(h.dtype), hip.mx_dequantize(self.up, h.dtype)).to(h.dtype)
        dx, dweight = hip.rms_norm_backward(dn, h, self.weight, rstd, dh=dh)
        return {"dx": dx, "dweight": dweight, "dup_bias": du.sum(0), "ddown_bias": dy.float().sum(0)}


def _product(a, b):
    """a b of 16-bit matrices in float32; of no rows too, as the other operators serve them."""
    if a.shape[0] == 0:
        return a.new_empty(0, b.shape[1], dtype=torch.float32)
    return (hip.gemm_bf16 if a.dtype == torch.bfloat16 else hip.gemm_f16)(a, b)


def main(argv=None):
    import sys
    sizes = [int(v) for v in (sys.argv[1:] if argv is None else argv)]
    tokens, width, inner = sizes + [16, 1024, 4096][len(sizes):]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    random = lambda std, *shape: torch.empty(shape, device="cuda").normal_(0, std, generator=gen)  # noqa: E731
    x, residual = random(1, tokens, width).bfloat16(), random(1, tokens, width).bfloat16()
    weight = (1 + random(0.1, width)).bfloat16()
    up, down = hip.mx_quantize(random(0.02, inner, width), "fp4"), hip.mx_quantize(random(0.02, width, inner), "fp4")
    up_bias, down_bias = random(0.1, inner), random(0.1, width)
    layer = MxFeedForward(weight, up, down, up_bias, down_bias)
    y, h, kept = layer.train(x, residual)
    dy = random(0.1, tokens, width).bfloat16()
    grads = layer.backward(kept, dy, h)

    # float64, the ReLU as the layer chose, no rounding to 8 bits
    leaves = {"dx": h, "dweight": weight, "dup_bias": up_bias, "ddown_bias": down_bias}
    leaves = {name: t.double().detach().requires_grad_() for name, t in leaves.items()}
    values = lambda q: hip.mx_dequantize(q, torch.float32).double()  # noqa: E731
    n = leaves["dx"] / (leaves["dx"].pow(2).mean(1, keepdim=True) + layer.eps).sqrt() * leaves["dweight"]
    want = ((n @ values(up).t() + leaves["dup_bias"]) * (kept[2] > 0)) @ values(down).t() + leaves["ddown_bias"]
    ((want * dy.double()).sum() + (leaves["dx"] * h.double()).sum()).backward()
    away = lambda got, right: float((got.double() - right).norm() / right.norm())  # noqa: E731
    off = {"y": (away(y, want.detach()), 0.05), **{name: (away(grads[name], t.grad), 0.02) for name, t in leaves.items()}}
    print(f"{tokens} x {width} -> {inner} -> {width}: output and gradients within (of the layer in float64 without its roundings to 8 bits) "
          + ", ".join(f"{name} {far:.4f}" for name, (far, _) in off.items()))
    return 0 if all(far < most for far, most in off.values()) else 1


if __name__ == "__main__":
    raise SystemExit(main())
