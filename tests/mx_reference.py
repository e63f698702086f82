"""Microscaled rows, their norm and their products in float64 with numpy, from the formats' definitions: what the tests of
the kernels compare with."""
import numpy as np

EMAX, EMIN, BITS, LARGEST = {"fp8": 8, "fp4": 2}, {"fp8": -6, "fp4": 0}, {"fp8": 3, "fp4": 1}, {"fp8": 448.0, "fp4": 6.0}


def grid(fmt):
    """The magnitudes of a format in order: code c stands for grid(fmt)[c]."""
    p = 2 ** BITS[fmt]
    g = [j * 2.0 ** (EMIN[fmt] - BITS[fmt]) for j in range(p)]
    g += [(1 + j / p) * 2.0 ** e for e in range(EMIN[fmt], EMAX[fmt] + 1) for j in range(p)]
    return np.array([v for v in g if v <= LARGEST[fmt]])


def row_values(k):
    return -(-k // 256) * 256


def blocks(x):
    """[rows, k] -> [rows, kp / 32, 32], zeros behind k."""
    x = np.asarray(x, dtype=np.float64)
    out = np.zeros((x.shape[0], row_values(x.shape[1])))
    out[:, :x.shape[1]] = x
    return out.reshape(x.shape[0], -1, 32)


def scale_bytes(x, fmt):
    z = blocks(x)
    with np.errstate(all="ignore"):
        most = np.abs(z).max(-1)
        e = np.frexp(most)[1] - 1 - EMAX[fmt]
    e = np.where((most > 0) & (e >= -127), e, -127)
    return np.where(np.isfinite(z).all(-1), e + 127, 255).astype(np.uint8)


def quantise(x, fmt):
    """(codes one to an element [rows, kp], scale bytes [rows, kp / 32])."""
    z, s, g = blocks(x), scale_bytes(x, fmt), grid(fmt)
    with np.errstate(all="ignore"):
        v = np.abs(z) * 2.0 ** -(s.astype(np.float64) - 127)[..., None]
    v = np.where((s == 255)[..., None], 0.0, v)
    mid = (g[1:] + g[:-1]) / 2
    low, high = np.searchsorted(mid, v), np.searchsorted(mid, v, side="right")
    code = np.where((low != high) & (low % 2 == 1), high, low).astype(np.uint8)
    sign = np.signbit(z) & ~(s == 255)[..., None]
    top = 128 if fmt == "fp8" else 8
    return (code | sign * np.uint8(top)).reshape(z.shape[0], -1), s


def pack(codes, fmt):
    return codes if fmt == "fp8" else (codes[:, 0::2] | codes[:, 1::2] << 4)


def unpack(codes, fmt):
    return codes if fmt == "fp8" else np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)


def values(codes, scales, fmt, k):
    """What packed codes and scale bytes stand for."""
    c = unpack(codes, fmt)
    top = 128 if fmt == "fp8" else 8
    g = np.append(grid(fmt), np.nan) if fmt == "fp8" else grid(fmt)
    v = g[c & (top - 1)] * np.where(c & top, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(c.shape[0], -1, 32) * s[..., None]).reshape(c.shape[0], -1)[:, :k]


def norm(h, weight, eps):
    """(1 / rms of the rows, the norm)."""
    h = np.asarray(h, dtype=np.float64)
    rstd = 1 / np.sqrt((h * h).mean(1) + eps)
    return rstd, h * rstd[:, None] * np.asarray(weight, dtype=np.float64)


def norm_backward(dy, h, weight, rstd, dh):
    dy, h, w = (np.asarray(v, dtype=np.float64) for v in (dy, h, weight))
    r = np.asarray(rstd, dtype=np.float64)[:, None]
    n, g = h * r, w * dy
    dx = r * (g - n * (n * g).mean(1, keepdims=True))
    return dx + (0 if dh is None else np.asarray(dh, dtype=np.float64)), (dy * n).sum(0)
