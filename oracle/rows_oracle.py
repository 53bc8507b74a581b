"""Feature rows in 8 or 4 bits restated in float64 numpy from their definition (include/pointslam_hip.h, psl_rows_*): scale =
fp32(max|x| / Q) per group (rounded down where Q times it would not be finite), code = the representable value nearest to x / scale,
ties to even.  The float64 quotient of two 24-bit numbers is never on a tie that the exact one is not on (they differ by at
least 2^-27 of their size), so the codes here are THE codes.  Test infrastructure only."""
import numpy as np

TOP = {"int8": 127.0, "int4": 7.0, "e4m3": 448.0}


def largest_scale(fmt):
    s = np.finfo(np.float32).max / np.float32(TOP[fmt])
    while float(s) * TOP[fmt] >= 2.0 ** 128 - 2.0 ** 103:       # what fp32 rounds to infinity
        s = np.nextafter(s, np.float32(0))
    return s


def nearest_e4m3(q):
    """Three mantissa bits, exponents -6 .. 8, step 2^-9 below 2^-6; ties to the even mantissa."""
    _, e = np.frexp(q)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(q / step) * step


def quantize(x, fmt, group):
    """x [n, heads, dim] (any float type) -> (values of the codes float64 [n, heads, dim], scales float32 [n, heads, dim/group])."""
    x = np.asarray(x, dtype=np.float64)
    n, h, d = x.shape
    g = x.reshape(n, h, d // group, group)
    top = np.abs(g).max(-1)                                     # NaN stays NaN
    with np.errstate(all="ignore"):
        s = np.minimum((top.astype(np.float32) / np.float32(TOP[fmt])).astype(np.float32), largest_scale(fmt))
        s = np.where(np.isfinite(top), s, np.float32(np.nan))
        q = g / s.astype(np.float64)[..., None]
        q = np.where((s > 0)[..., None], q, 0.0)
        q = nearest_e4m3(q) if fmt == "e4m3" else np.round(q)
    return np.clip(q, -TOP[fmt], TOP[fmt]).reshape(n, h, d), s


def values(q, s):
    """What the held rows stand for, in fp32 (one product, rounded once)."""
    n, h, d = q.shape
    with np.errstate(all="ignore"):
        return (q.reshape(n, h, s.shape[-1], -1).astype(np.float32) * s[..., None]).reshape(n, h, d)
