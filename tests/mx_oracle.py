"""The microscaled formats in numpy, 64 bits: what the GPU kernels are held to. Written from the formats' definition."""
import numpy as np

GRID4 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
_c = np.arange(256)
_e, _m = _c >> 3 & 15, _c & 7
E4M3 = np.where(_e > 0, (1 + _m / 8) * 2.0 ** (_e - 7.0), _m / 8 * 2.0 ** -6) * np.where(_c >> 7, -1, 1)
E4M3[[127, 255]] = np.nan
GRID8 = E4M3[:127]


def _nearest(mag, grid):
    """Index of the nearest grid value, ties to the even index, beyond the last one: the last."""
    hi = np.clip(np.searchsorted(grid, mag), 1, len(grid) - 1)
    lo = hi - 1
    up = (mag - grid[lo] > grid[hi] - mag) | ((mag - grid[lo] == grid[hi] - mag) & (lo % 2 == 1))
    return np.where(up, hi, lo)


def quantize(x, four):
    """(codes [rows, K] one a byte, scales [rows, K/32]) of f32 rows."""
    b = np.asarray(x, np.float32).astype(np.float64).reshape(x.shape[0], -1, 32)
    big = np.abs(b).max(-1)
    bad = ~np.isfinite(big)
    _, e = np.frexp(np.where(bad, 1.0, big))
    s = np.where(big == 0, 0, np.maximum(e - 1 + 127 - (2 if four else 8), 0)).astype(np.int64)
    v = np.where(bad[..., None], 0, b) * 2.0 ** (127 - np.where(bad, 127, s))[..., None]
    codes = _nearest(np.abs(v), GRID4 if four else GRID8) | np.where(np.signbit(v), 8 if four else 128, 0)
    return codes.astype(np.uint8).reshape(x.shape), np.where(bad, 255, s).astype(np.uint8)


def pack(codes):
    return np.ascontiguousarray(codes[:, 0::2] | codes[:, 1::2] << 4)


def values(codes, scales, four):
    v = np.where(codes & 8, -1.0, 1.0) * GRID4[codes & 7] if four else E4M3[codes]
    f = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(v.shape[0], -1, 32) * f[..., None]).reshape(v.shape)


def norm(x, parts, w, eps):
    """(xout f32, h f32): the residual's sum in f32 in the order of the parts, the norm in 64 bits, rounded once."""
    x = x.astype(np.float32)
    if len(parts):
        t = parts[0].copy()
        for p in parts[1:]:
            t = t + p
        x = x + t
    d = x.astype(np.float64)
    h = d * (1.0 / np.sqrt((d * d).mean(-1, keepdims=True) + np.float64(np.float32(eps)))) * w.astype(np.float64)
    return x, h.astype(np.float32)


def swiglu(gu):
    ff = gu.shape[1] // 2
    g = gu[:, :ff]
    return g / (1 + np.exp(-g)) * gu[:, ff:]
