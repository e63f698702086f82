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
