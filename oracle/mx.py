"""CPU oracle of the microscaled operators, in float64 numpy from their definition: blocks of 32
values share 2^e with e = floor(log2(largest magnitude)) minus the element format's largest
exponent; elements are the nearest of the format's values, ties to the even code.  No reference
counterpart."""
import numpy as np

EMAX = {"mxfp4": 2, "mxfp8": 8}


def grid(fmt):
    """The format's non-negative finite values in ascending order; the index is the code."""
    if fmt == "mxfp4":
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
    e, m = np.divmod(np.arange(127), 8)
    return np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))


def nearest(v, fmt):
    """Codes (without sign) of the magnitudes v: nearest, ties to even, clamped."""
    g = grid(fmt)
    mid = (g[1:] + g[:-1]) / 2
    lo = np.searchsorted(mid, v, side="left")           # midpoints below v
    hi = np.searchsorted(mid, v, side="right")          # ... at or below
    return np.where(lo == hi, lo, lo + (lo & 1))


def quantize(x, fmt):
    """x [rows, K] -> (codes with sign uint8 [rows, nb, 32], scale bytes uint8 [rows, nb]); a
    block with a non-finite value has zero codes and byte 255."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    nb = -(-K // 32)
    b = np.zeros((rows, nb * 32))
    b[:, :K] = x
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 1 - EMAX[fmt], -127)
    e = np.maximum(e, -127)
    v = np.ldexp(b, -e[..., None])
    code = nearest(np.abs(v), fmt).astype(np.uint8)
    sign = (np.signbit(b) & ~bad[..., None]).astype(np.uint8)
    code |= sign << (3 if fmt == "mxfp4" else 7)
    return code, np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales, fmt):
    """Float64 values [rows, nb * 32] of codes [rows, nb, 32] and scale bytes [rows, nb]."""
    bits = 3 if fmt == "mxfp4" else 7
    mag = (codes & ((1 << bits) - 1)).astype(np.int64)
    g = np.append(grid(fmt), np.nan) if fmt == "mxfp8" else grid(fmt)
    v = np.where(codes >> bits, -g[mag], g[mag])
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    with np.errstate(invalid="ignore"):
        return (v * s[..., None]).reshape(codes.shape[0], -1)


def split_codes(data, fmt):
    """Packed bytes [rows, ...] -> codes [rows, nb, 32]."""
    rows = data.shape[0]
    if fmt == "mxfp4":
        c = np.empty((rows, data.shape[1] * 2), np.uint8)
        c[:, 0::2], c[:, 1::2] = data & 15, data >> 4
    else:
        c = data
    return c.reshape(rows, -1, 32)


def row_scales(tiled, rows, nb):
    """Scale bytes [rows, nb] out of the tiled layout [row tiles, groups, 32, 4, 4]."""
    r, j = np.arange(rows)[:, None], np.arange(nb)[None]
    return tiled[r // 128, j // 4, r % 32, r % 128 // 32, j % 4]


def rms_norm(x, weight, residual, eps):
    """(y, h) in float64 of float32 inputs; h = x + residual is rounded to float32, as it is
    defined."""
    h = np.asarray(x, np.float32)
    if residual is not None:
        h = h + np.asarray(residual, np.float32)
    h = h.astype(np.float64)
    root = np.sqrt((h * h).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    return h / root * np.asarray(weight, np.float64), h
