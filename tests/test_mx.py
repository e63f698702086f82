"""What the microscaled operators refuse, the layout of their matrices, and the reference that the GPU tests compare with."""
import numpy as np
import pytest
import torch

import mx_reference as ref


@pytest.mark.parametrize("k,kp", [(-1, 0), (0, 0), (1, 256), (255, 256), (256, 256), (257, 512), (11008, 11008), (2 ** 31, 2 ** 31)])
def test_row_values(hip, k, kp):
    assert hip.lib.sarek_hip_mx_row_values(k) == kp
    if k > 0:
        assert hip.mx_row_values(k) == kp


def test_reference_grids():
    assert ref.grid("fp4").tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    g = ref.grid("fp8")
    assert len(g) == 127 and g[-1] == 448 and g[1] == 2.0 ** -9 and g[8] == 2.0 ** -6
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(codes, g)


def test_reference_ties_saturation_and_undefined_blocks():
    x = np.zeros((1, 64))
    x[0, :8] = [4, 5, 3.5, 2.5, 0.25, 0.75, -7.9, 1.25]        # E = 0: on the grid, and ties that go to the even code
    x[0, 40] = np.inf
    c, s = ref.quantise(x, "fp4")
    assert s[0, :3].tolist() == [127, 255, 0]
    assert ref.values(ref.pack(c, "fp4"), s, "fp4", 64)[0, :8].tolist() == [4, 4, 4, 2, 0, 1, -6, 1]
    assert np.isnan(ref.values(ref.pack(c, "fp4"), s, "fp4", 64)[0, 32:]).all()


P, Q = 1 << 20, (1 << 20) + 16      # aligned addresses that are never read: a refusal comes before any launch


def quantise(lib, x=P, type=1, stride=64, codes=P, scales=Q, fmt=0, rows=2, k=64):
    return lib.sarek_hip_mx_quantize(x, type, stride, codes, scales, fmt, rows, k, None)


def dequantise(lib, codes=P, scales=Q, fmt=0, out=P, type=1, stride=64, rows=2, k=64):
    return lib.sarek_hip_mx_dequantize(codes, scales, fmt, out, type, stride, rows, k, None)


def rms(lib, x=P, xs=64, residual=None, rs=0, weight=P, type=1, eps=1e-6, h=None, hs=0, codes=P, scales=Q, rows=2, k=64):
    return lib.sarek_hip_rms_norm_mx(x, xs, residual, rs, weight, type, eps, h, hs, codes, scales, None, rows, k, None)


def back(lib, dy=P, dys=64, h=P, hs=64, weight=P, rstd=P, dh=None, dhs=0, type=1, dx=P, dxs=64, dw=P, rows=2, k=64, ws=P,
         floats=1 << 20):
    return lib.sarek_hip_rms_norm_backward(dy, dys, h, hs, weight, rstd, dh, dhs, type, dx, dxs, dw, rows, k, ws, floats, None)


def product(lib, a=P, sa=Q, fmt=0, b=P, sb=Q, bias=None, c=P, type=1, stride=64, m=2, n=64, k=64):
    return lib.sarek_hip_gemm_mx(a, sa, fmt, b, sb, bias, 0, c, type, stride, m, n, k, None)


@pytest.mark.parametrize("call,bad", [
    (quantise, dict(x=None)), (quantise, dict(codes=None)), (quantise, dict(scales=None)), (quantise, dict(rows=-1)),
    (quantise, dict(k=0)), (quantise, dict(type=3)), (quantise, dict(type=-1)), (quantise, dict(fmt=2)), (quantise, dict(stride=63)),
    (quantise, dict(codes=P + 8)), (quantise, dict(scales=Q + 1)),
    (dequantise, dict(codes=None)), (dequantise, dict(scales=None)), (dequantise, dict(out=None)), (dequantise, dict(rows=-1)),
    (dequantise, dict(k=-1)), (dequantise, dict(type=7)), (dequantise, dict(fmt=-1)), (dequantise, dict(stride=0)), (dequantise, dict(codes=P + 1)),
    (rms, dict(x=None)), (rms, dict(weight=None)), (rms, dict(codes=None)), (rms, dict(scales=None)), (rms, dict(rows=-5)), (rms, dict(k=0)),
    (rms, dict(type=3)), (rms, dict(eps=-1.0)), (rms, dict(eps=float("nan"))), (rms, dict(xs=1)), (rms, dict(residual=P, rs=64)),
    (rms, dict(residual=P, rs=63, h=P, hs=64)), (rms, dict(h=P, hs=63)), (rms, dict(scales=Q + 4)),
    (back, dict(dy=None)), (back, dict(h=None)), (back, dict(weight=None)), (back, dict(rstd=None)), (back, dict(dx=None)),
    (back, dict(dw=None)), (back, dict(ws=None)), (back, dict(rows=-1)), (back, dict(k=0)), (back, dict(type=3)), (back, dict(dys=63)),
    (back, dict(hs=63)), (back, dict(dxs=63)), (back, dict(dh=P, dhs=63)),
    (product, dict(a=None)), (product, dict(sa=None)), (product, dict(b=None)), (product, dict(sb=None)), (product, dict(c=None)),
    (product, dict(m=-1)), (product, dict(n=0)), (product, dict(k=0)), (product, dict(fmt=2)), (product, dict(type=3)),
    (product, dict(stride=63)), (product, dict(a=P + 4)), (product, dict(b=P + 2)), (product, dict(sb=Q + 2))],
    ids=lambda v: v.__name__ if callable(v) else "-".join(v))
def test_invalid_arguments(hip, call, bad):
    assert call(hip.lib, **bad) == hip.E_INVALID_ARG
    assert hip.lib.sarek_hip_last_error()


def test_workspace_and_unsupported(hip):
    need = hip.lib.sarek_hip_rms_norm_backward_workspace_floats(2, 64)
    assert need > 0 and hip.lib.sarek_hip_rms_norm_backward_workspace_floats(0, 64) == 0
    assert back(hip.lib, floats=need - 1) == hip.E_WORKSPACE
    assert product(hip.lib, type=0) == hip.E_UNSUPPORTED                      # 8-bit rows to float32
    assert product(hip.lib, m=1 << 20) == hip.E_UNSUPPORTED
    assert quantise(hip.lib, rows=1 << 31) == hip.E_UNSUPPORTED
    assert rms(hip.lib, k=2 ** 31 - 1, xs=2 ** 31) == hip.E_UNSUPPORTED


def test_no_rows_is_no_error(hip):
    assert quantise(hip.lib, rows=0, x=None) == 0 and dequantise(hip.lib, rows=0, out=None) == 0
    assert rms(hip.lib, rows=0, x=None) == 0 and product(hip.lib, m=0, a=None, c=None) == 0


def test_the_front_end_refuses_host_tensors_and_wrong_kinds(hip):
    x = torch.zeros(2, 64)
    for call in (lambda: hip.mx_quantize(x, "fp8"), lambda: hip.rms_norm_mx(x, torch.ones(64)), lambda: hip.mx_dequantize(x),
                 lambda: hip.rms_norm_backward(x, x, torch.ones(64), torch.ones(2)), lambda: hip.gemm_mx(x, x)):
        with pytest.raises(TypeError):
            call()
    q = hip.MxTensor(torch.zeros(2, 256, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.uint8), "fp8", 64)
    assert q.rows == 2
    with pytest.raises(TypeError):
        hip.gemm_mx(q, q)                                                      # on the host


def test_mx_tensor_is_checked(hip):
    codes, scales = torch.zeros(2, 256, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.uint8)
    q = hip.MxTensor(codes, scales, "fp8", 64)
    assert (q.rows, q.k, q.fmt) == (2, 64, "fp8") and q.codes is codes and q.scales is scales
    assert hip.MxTensor(codes, torch.zeros(2, 16, dtype=torch.uint8), "fp4", 257).k == 257
    for bad in ((codes, scales, "fp8", 0), (codes, scales, "fp8", 257), (codes, scales, "fp4", 64), (codes, scales, "fp6", 64),
                (codes, scales[:1], "fp8", 64), (codes.view(-1), scales, "fp8", 64), (codes, scales.view(4, 4), "fp8", 64)):
        with pytest.raises(ValueError):
            hip.MxTensor(*bad)
    for bad in ((codes.float(), scales, "fp8", 64), (codes, scales.int(), "fp8", 64), (codes[:, ::2], scales, "fp4", 64), (None, scales, "fp8", 64)):
        with pytest.raises(TypeError):
            hip.MxTensor(*bad)


def test_a_made_tensor_has_its_parts_in_one_block(hip):
    for fmt, width in (("fp8", 512), ("fp4", 256)):
        q = hip.MxTensor._empty(3, 300, fmt, torch.zeros(1))
        at = q._at
        assert q.codes.shape == (3, width) and q.scales.shape == (3, 16) and q.codes.is_contiguous() and q.scales.is_contiguous()
        assert (q.codes.data_ptr(), q.scales.data_ptr()) == at and at[1] % 8 == 0
        q.codes.fill_(1), q.scales.fill_(2)
        assert int(q.codes.sum()) == 3 * width and int(q.scales.sum()) == 96


def test_native_calls_check_their_arguments(hip):
    """What goes to C through the extension: the number of the arguments, their kinds and their ranges; nothing is called else."""
    good = [None, 0, 64, None, None, 0, 0, 64, None]
    assert hip._host.mx_quantize(*good) == hip.OK
    for i, bad, error in ((1, 1 << 31, OverflowError), (2, 1 << 63, OverflowError), (0, "x", TypeError), (5, 1.5, TypeError), (7, None, TypeError)):
        with pytest.raises(error):
            hip._host.mx_quantize(*good[:i], bad, *good[i + 1:])
    for call, count in ((hip._host.mx_quantize, 9), (hip._host.mx_dequantize, 9), (hip._host.rms_norm_mx, 15),
                        (hip._host.rms_norm_backward, 17), (hip._host.gemm_mx, 14), (hip._host.bind_mx, 5)):
        for n in (0, count - 1, count + 1):
            with pytest.raises(TypeError):
                call(*[0] * n)


def test_workspaces_grow_with_rows_to_a_limit(hip):
    """A plane for each workgroup; what serves some rows serves fewer too."""
    f = hip.lib.sarek_hip_rms_norm_backward_workspace_floats
    for k in (1, 64, 1024, 1025, 1536, 1537, 4096, 4097, 20000):
        planes = [f(rows, k) // k for rows in (*range(1, 4200), 1 << 14, 1 << 20)]
        assert planes == sorted(planes) and planes[0] == 1 and planes[-1] == planes[-2] <= 512 and f(7, k) % k == 0
