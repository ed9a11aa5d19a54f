"""Microscaled numbers on the host in 64 bits: the reference of the linear
layer's tests (MXFP4 from synthetic.py, MXFP8 here)."""
import numpy as np

import synthetic

FP4, FP8 = 0, 1


def e8m0(scales):
    """Scale bytes to values; 255 is NaN."""
    v = np.ldexp(1.0, scales.astype(np.int32) - 127)
    return np.where(scales == 255, np.nan, v)


def e4m3_values():
    c = np.arange(256)
    ex, man = (c >> 3) & 15, c & 7
    v = np.where(ex > 0, (8 + man) * np.ldexp(1.0, ex - 10), man * 2.0 ** -9)
    v[(c & 127) == 127] = np.nan
    return np.where(c >> 7, -v, v)


E4M3 = e4m3_values()
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6])


def quantize(x, fmt):
    """fp32 [rows, K] to (codes, scales [rows, K/32]) by the formats' definition."""
    x = np.ascontiguousarray(x, np.float32)
    rows, K = x.shape
    b = x.reshape(rows, K // 32, 32).astype(np.float64)
    bad = ~np.isfinite(b).all(axis=2)
    b = np.where(bad[:, :, None], 0.0, b)
    if fmt == FP4:
        codes, scales = synthetic.mxfp4_quantize(b.reshape(rows, K).astype(np.float32))
        scales = np.where(bad, 255, scales).astype(np.uint8)
        codes = codes.reshape(rows, K // 32, 16).copy()
        codes[bad] = 0
        return codes.reshape(rows, K // 2), scales
    amax = np.abs(b).max(axis=2)
    frac, ex = np.frexp(amax)
    e = np.where(amax > 0, np.clip(ex - 9 + (frac > 0.875), -127, 127), 0)
    v = np.ldexp(b, -e[:, :, None])
    mag = E4M3[:127]
    a = np.abs(v)
    hi = np.clip(np.searchsorted(mag, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    d_hi, d_lo = mag[hi] - a, a - mag[lo]
    code = np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    code = (code | (np.signbit(b) << 7)).astype(np.uint8)
    code[bad] = 0
    return code.reshape(rows, K), np.where(bad, 255, e + 127).astype(np.uint8)


def dequantize(codes, scales, fmt):
    """Values in 64 bits, scales [rows, K/32]."""
    if fmt == FP4:
        v = E2M1[np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[0], -1)]
    else:
        v = E4M3[codes]
    return v * np.repeat(e8m0(scales), 32, axis=1)
