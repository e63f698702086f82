"""The feed-forward layer on microscaled rows: its command's own check, and the forms of its arguments.

Gradients: those of the layer in float64 with the ReLU's choices that it made and no rounding to 8 bits.  Three roundings to the type on the
way (2^-9 of a value each in bf16): within 2 % of their norms."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def made(hip, rows, k, inner, dtype, biases, seed=0):
    from spoc_amd.feed_forward import MxFeedForward
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    random = lambda std, *shape: torch.empty(shape, device="cuda").normal_(0, std, generator=gen)  # noqa: E731
    weight = (1 + random(0.1, k)).to(dtype)
    up, down = hip.mx_quantize(random(0.05, inner, k), "fp4"), hip.mx_quantize(random(0.05, k, inner), "fp4")
    more = (random(0.1, inner), random(0.1, k)) if biases else (None, None)
    return MxFeedForward(weight, up, down, *more), *(random(1, rows, k).to(dtype) for _ in range(4))


def check_gradients(hip, layer, kept, got, dy, dh):
    h, _, u = kept
    k, inner = layer.up.k, layer.up.rows
    start = {"dx": h, "dweight": layer.weight, "dup_bias": torch.zeros(inner, device="cuda") if layer.up_bias is None else layer.up_bias,
             "ddown_bias": torch.zeros(k, device="cuda") if layer.down_bias is None else layer.down_bias}
    leaf = {n: t.double().detach().clone().requires_grad_() for n, t in start.items()}
    n = leaf["dx"] * torch.rsqrt(leaf["dx"].pow(2).mean(1, keepdim=True) + layer.eps) * leaf["dweight"]
    wu, wd = (hip.mx_dequantize(t, torch.float32).double() for t in (layer.up, layer.down))
    out = ((n @ wu.t() + leaf["dup_bias"]) * (u > 0)) @ wd.t() + leaf["ddown_bias"]
    total = (out * dy.double()).sum()
    (total if dh is None else total + (leaf["dx"] * dh.double()).sum()).backward()
    for name, t in leaf.items():
        assert float((got[name].double() - t.grad).norm()) <= 0.02 * float(t.grad.norm()), name


@pytest.mark.parametrize("wrong", ["dx", "dweight", "dup_bias", "ddown_bias", "nan"])
def test_the_command_checks_the_gradients(hip, torch_cuda, monkeypatch, wrong):
    from spoc_amd import feed_forward
    assert feed_forward.main(["5", "300", "700"]) == 0
    right = feed_forward.MxFeedForward.backward

    def off(self, *args):
        grads = right(self, *args)
        name = "dx" if wrong == "nan" else wrong
        grads[name] = grads[name] * (float("nan") if wrong == "nan" else 1.2)
        return grads
    monkeypatch.setattr(feed_forward.MxFeedForward, "backward", off)
    assert feed_forward.main(["5", "300", "700"]) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_of_strided_rows(hip, torch_cuda, dtype):
    """dy, dh and the inputs as rows of larger matrices, at odd elements: the same bits as from matrices of their own."""
    rows, k, inner = 37, 300, 520
    layer, x, residual, dy, dh = made(hip, rows, k, inner, dtype, True)
    apart = []
    for i, t in enumerate((x, residual, dy, dh)):
        whole = torch.full((rows * (k + 3 + i) + 9,), 5.0, dtype=dtype, device="cuda")
        apart.append(whole[1 + i:1 + i + rows * (k + 3 + i)].view(rows, k + 3 + i)[:, :k])
        apart[-1].copy_(t)
    y, h, kept = layer.train(x, residual)
    got = layer.train(*apart[:2])
    assert torch.equal(got[0], y) and torch.equal(got[1], h)
    want, grads = layer.backward(kept, dy, dh), layer.backward(got[2], *apart[2:])
    assert all(torch.equal(grads[name], v) for name, v in want.items())
    check_gradients(hip, layer, kept, want, dy, dh)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [0, 1, 19])
@pytest.mark.parametrize("residual,dh,biases", [(False, False, False), (True, False, True), (False, True, True), (True, True, False)])
def test_gradients_without_the_arguments_that_may_be_missing(hip, torch_cuda, rows, dtype, residual, dh, biases):
    layer, x, more, dy, above = made(hip, rows, 260, 390, dtype, biases, seed=rows)
    y, h, kept = layer.train(x, more if residual else None)
    assert torch.equal(h, x + more if residual else x) and y.shape == x.shape
    got = layer.backward(kept, dy, above if dh else None)
    assert got["dx"].shape == x.shape and got["dx"].dtype == dtype
    check_gradients(hip, layer, kept, got, dy, above if dh else None)
