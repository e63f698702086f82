"""Cosines and sines of rotary positions against angles from whole numbers of any length."""
import math

import pytest
import torch

import rotary_exactly as exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_angles(hip, torch_cuda, layout):
    """Pairs (1, 0) become (cos, sin), which the library's functions give to 4 steps of 2^-23; what the angle is off goes into the sine whole where it is small."""
    f = [s * 10 ** (-9 * i / 47) for i in range(48) for s in (1, -1)]
    at = [0, 1, -1, 3, 17, 1000, 4095, 999999, 2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345]
    plan = hip.Rotary(192, layout=layout, frequencies=f)
    x = torch.zeros(len(at), 1, 192, device="cuda")
    first = x[..., :96] if layout == "half" else x[..., 0::2]
    first.fill_(1.0)
    positions = torch.tensor(at, device="cuda")
    y = hip.rotary(x, positions, plan).double().cpu()[:, 0]
    cos, sin = (y[:, :96], y[:, 96:]) if layout == "half" else (y[:, 0::2], y[:, 1::2])
    worst = 0.0
    for i, p in enumerate(at):
        for j, frequency in enumerate(f):
            angle = float(exact.turns(p, frequency) * exact.TWO_PI)
            off = 2 * math.pi * exact.angle_bound(p, angle)
            s, c = math.sin(angle), math.cos(angle)
            for got, want, slope in ((float(sin[i, j]), s, c), (float(cos[i, j]), c, s)):
                worst = max(worst, abs(got - want) / (off * (abs(slope) + off) + 4 * 2.0 ** -23 * abs(want) + 1e-30))
    assert worst <= 1, worst
