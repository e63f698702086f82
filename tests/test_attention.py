"""What the operators on a paged cache refuse, the frequencies of rotary positions, and the reference of the GPU tests."""
import ctypes as C
import math

import pytest
import torch

import attention_reference as ref

P = 1 << 20      # an aligned address that is never read: a refusal comes before any launch


def layout(hip, **kw):
    v = dict(keys=P, values=P, page_stride=16 * 2 * 64, slot_stride=2 * 64, head_stride=64, n_pages=4, page_size=16, heads=2, head_dim=64, type=1)
    v.update({k: kw.pop(k) for k in list(kw) if k in v})
    return hip.KvCacheLayout(**v), kw


def rotary(hip, plan=(P, 32, 0, 1.0), x=P, xt=256, xh=64, type=1, positions=P, size=8, out=P, ot=256, oh=64, tokens=2, heads=4, d=64):
    plan = None if plan is None else C.byref(hip.RotaryPlan(*plan))
    return hip.lib.sarek_hip_rotary(plan, x, xt, xh, type, positions, size, 0, out, ot, oh, tokens, heads, d, None)


def append(hip, plan=None, k=P, kt=128, kh=64, v=P, vt=128, vh=64, q=P, qt=256, qh=64, o=P, ot=256, oh=64, q_heads=4, pages=P, ps=2, mp=2,
           lengths=P, starts=None, batch=2, tokens=2, **cache):
    held, rest = layout(hip, **cache)
    assert not rest
    plan = None if plan is None else C.byref(hip.RotaryPlan(*plan))
    return hip.lib.sarek_hip_kv_append(C.byref(held), k, kt, kh, v, vt, vh, q, qt, qh, o, ot, oh, q_heads, plan, pages, ps, mp, lengths, starts, batch,
                                       tokens, 0, None)


def attend(hip, q=P, qt=256, qh=64, q_heads=4, out=P, ot=256, oh=64, pages=P, ps=2, mp=2, lengths=P, starts=None, batch=2, tokens=2, scale=0.125,
           workspace=P, held=1 << 40, prefix=None, n=0, **cache):
    kv, rest = layout(hip, **cache)
    assert not rest
    return hip.lib.sarek_hip_attention_shared(C.byref(kv), q, qt, qh, q_heads, out, ot, oh, None, prefix, n, pages, ps, mp, lengths, starts, batch,
                                              tokens, 1, scale, workspace, held, None)


CACHE = [dict(keys=None), dict(values=None), dict(type=0), dict(type=3), dict(n_pages=0), dict(page_size=0), dict(heads=0), dict(head_dim=0), dict(keys=P + 8),
         dict(values=P + 2), dict(page_stride=60), dict(slot_stride=100), dict(head_stride=56)]
SEQUENCES = [dict(pages=None), dict(lengths=None), dict(batch=-1), dict(tokens=-1), dict(mp=-1), dict(ps=1), dict(batch=3)]


@pytest.mark.parametrize("call,bad", [
    (rotary, dict(plan=None)), (rotary, dict(plan=(None, 32, 0, 1.0))), (rotary, dict(plan=(P, 0, 0, 1.0))), (rotary, dict(plan=(P, 33, 0, 1.0))),
    (rotary, dict(plan=(P, 32, 0, math.inf))), (rotary, dict(x=None)), (rotary, dict(positions=None)), (rotary, dict(out=None)), (rotary, dict(type=3)),
    (rotary, dict(size=2)), (rotary, dict(tokens=-1)), (rotary, dict(heads=0)), (rotary, dict(d=0)), (rotary, dict(xt=-1)), (rotary, dict(ot=255)),
    (rotary, dict(oh=63)), (rotary, dict(xt=512)),      # (out is x, but not as it lies)
    *[(append, v) for v in CACHE + SEQUENCES], (append, dict(k=None)), (append, dict(v=None)), (append, dict(o=None)), (append, dict(q_heads=0)),
    (append, dict(ot=200)), (append, dict(qt=512)), (append, dict(plan=(P, 40, 0, 1.0))), (append, dict(plan=(P, 4, 0, math.nan))),
    *[(attend, v) for v in CACHE + SEQUENCES], (attend, dict(q=None)), (attend, dict(out=None)), (attend, dict(q_heads=3)), (attend, dict(q_heads=0)),
    (attend, dict(scale=0.0)), (attend, dict(scale=-1.0)), (attend, dict(scale=math.nan)), (attend, dict(scale=math.inf)), (attend, dict(ot=64)), (attend, dict(oh=8)),
    (attend, dict(qh=-64)), (attend, dict(n=5)), (attend, dict(prefix=P, n=-1))],
    ids=lambda v: v.__name__ if callable(v) else "-".join(v))
def test_invalid_arguments(hip, call, bad):
    assert call(hip, **bad) == hip.E_INVALID_ARG
    assert hip.lib.sarek_hip_last_error()


@pytest.mark.parametrize("call,bad", [
    (rotary, dict(heads=65536, x=P, xh=64, oh=64, xt=1 << 23, ot=1 << 23)), (append, dict(head_dim=60)), (append, dict(head_dim=264, head_stride=264, slot_stride=528, page_stride=528 * 16)),
    (append, dict(tokens=1 << 24, starts=P)), (append, dict(batch=(1 << 16) + 1, tokens=(1 << 16) + 1)), (attend, dict(tokens=1 << 23, starts=P, q_heads=8)), (attend, dict(batch=1 << 17, tokens=1 << 17)), (attend, dict(mp=1 << 27, ps=1 << 27)),
    (attend, dict(prefix=P, n=(1 << 30) + 1)), (attend, dict(head_dim=4))], ids=lambda v: v.__name__ if callable(v) else "-".join(v))
def test_unsupported(hip, call, bad):
    assert call(hip, **bad) == hip.E_UNSUPPORTED


def test_nothing_to_do(hip):
    assert rotary(hip, tokens=0, x=None, out=None) == 0
    assert append(hip, batch=0, tokens=0, lengths=None, pages=None, k=None) == 0 and append(hip, tokens=0, starts=P) == 0
    assert attend(hip, batch=0, tokens=0, lengths=None, pages=None, q=None) == 0 and attend(hip, tokens=0, starts=P) == 0


def test_frequencies(hip):
    plain = hip.Rotary(64, device="cpu")
    assert plain.frequencies[0] == 1 and plain.frequencies[-1] == pytest.approx(10000 ** (-62 / 64))
    assert torch.equal(hip.Rotary(64, scaling="linear", factor=4.0, device="cpu").frequencies, plain.frequencies / 4)
    base = hip.Rotary(64, scaling="base", factor=8.0, device="cpu").frequencies
    assert base[0] == 1 and base[-1] == pytest.approx(float(plain.frequencies[-1]) / 8)
    ramp = hip.Rotary(64, scaling="ramp", factor=8.0, trained=4096, low=1.0, high=4.0, device="cpu").frequencies
    turns = 4096 * plain.frequencies / (2 * math.pi)
    assert torch.equal(ramp[turns >= 4], plain.frequencies[turns >= 4]) and torch.allclose(ramp[turns <= 1], plain.frequencies[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 4)
    assert between.any() and ((ramp > plain.frequencies / 8) & (ramp < plain.frequencies))[between].all()


def test_turns(hip):
    """2^-64 turns, of negative and of large frequencies too."""
    f = [1.0, -1.0, 0.0, 7.0, 1e-9, 1e6]
    got = [v % 2 ** 64 for v in hip.Rotary(12, frequencies=f, device="cpu").turns.tolist()]
    for v, radians in zip(got, f):
        want = radians / (2 * math.pi) % 1
        off = abs(v / 2 ** 64 - want)
        assert min(off, 1 - off) <= max(abs(radians), 1) * 2.0 ** -53
    assert got[0] + got[1] in (2 ** 64, 2 ** 64 - 1, 2 ** 64 + 1) and got[2] == 0


@pytest.mark.parametrize("bad", [dict(dim=3), dict(dim=0), dict(dim=4, layout="x"), dict(dim=4, scaling="x"), dict(dim=4, factor=0.0), dict(dim=4, base=-1.0),
                                 dict(dim=2, scaling="base", factor=2.0), dict(dim=4, low=2.0, high=2.0), dict(dim=4, frequencies=[1.0])], ids=str)
def test_rotary_refusals(hip, bad):
    with pytest.raises(ValueError):
        hip.Rotary(device="cpu", **bad)
    with pytest.raises(hip.SarekHipError):
        hip.Rotary(4, frequencies=[1.0, math.nan], device="cpu")


def test_cache_refuses_the_host(hip):
    with pytest.raises(TypeError):
        hip.KvCache(torch.zeros(1, 1, 1, 8, dtype=torch.bfloat16), torch.zeros(1, 1, 1, 8, dtype=torch.bfloat16))


def test_reference_rotation_is_a_rotation():
    x = torch.randn(4, 2, 10, generator=torch.Generator().manual_seed(0)).double()
    f, at = torch.tensor([1.0, 0.1, 0.01]).double(), torch.tensor([0, 1, 50, 1000])
    for kind in ("half", "interleaved"):
        y = ref.rotate(x, at, f, kind)
        assert torch.allclose(ref.rotate(y, at, f, kind, inverse=True), x, atol=1e-13) and torch.equal(y[0], x[0])
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[..., 6:], x[..., 6:])
    assert torch.allclose(ref.rotate(x, at, f, "half")[1, 0, 0], x[1, 0, 0] * math.cos(1) - x[1, 0, 3] * math.sin(1))


def test_reference_attention_by_hand():
    """Against the softmax written out, with a page table, a prefix, a row that sees nothing and values that a row does not see."""
    gen = torch.Generator().manual_seed(1)
    keys, values = (torch.randn(4, 2, 1, 8, generator=gen).double().to(torch.float16) for _ in range(2))
    values[3, 0] = math.inf                                      # key 2 of sequence 0: seen by its second token alone
    q = torch.randn(3, 2, 8, generator=gen).to(torch.float16)
    pages = torch.tensor([[1, 3], [-1, -1]])
    out, _, lse, _ = ref.attention(q, keys, values, pages, [3, 0], [0, 2, 3])
    k = torch.stack((keys[1, 0, 0], keys[1, 1, 0])).double()
    v = torch.stack((values[1, 0, 0], values[1, 1, 0])).double()
    for h in range(2):
        s = k @ q[0, h].double() / math.sqrt(8)
        assert torch.allclose(out[0, h], torch.softmax(s, 0) @ v) and torch.allclose(lse[0, h], torch.logsumexp(s, 0))
        assert torch.isinf(out[1, h]).all() and (out[2, h] == 0).all() and lse[2, h] == -math.inf
    out, _, _, _ = ref.attention(q[2:], keys, values, pages[1:], [0], None, prefix=torch.tensor([1]), prefix_length=2)
    assert torch.allclose(out[0, 0], torch.softmax(k @ q[2, 0].double() / math.sqrt(8), 0) @ v)
