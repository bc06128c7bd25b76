"""The norms in 64 bits (numpy), and how far a 32-bit evaluation may be from them. U32 is float32's unit
roundoff. A sum's error: one rounding for each addition that an element goes through."""
import numpy as np

import scaled_ref as ref

U32 = ref.U32


def row_depth(k):
    """Additions an element of a row's sum goes through: a thread's own (8 of each 512 columns at the
    fewest threads, 8 of each 8192 in long rows), 6 steps of a wave, 16 waves."""
    return 16 + k // 1024 + 6 + 16


def _unit(h, eps):
    h = h.astype(np.float64)
    rms = np.sqrt((h * h).sum(1, keepdims=True) / max(h.shape[1], 1) + eps)
    return h / rms, rms


def unit_error(k):
    """Of n = h / rms, relative: half of the squares' (their own rounding and the sum's), the division by k, eps,
    root and reciprocal, and the product."""
    return (0.5 * (row_depth(k) + 1) + 6) * U32


def norm(h, gain, eps):
    """(y, bound)."""
    n, _ = _unit(h, eps)
    y = n * gain.astype(np.float64)
    return y, np.abs(y) * (unit_error(h.shape[1]) + 2 * U32)


def norm_rows(h, gain, eps):
    """(q, t, bound of t): the int8 rows of h * gain in float32, and their scales over the rms."""
    z = (h.astype(np.float32) * gain.astype(np.float32)).astype(np.float32)
    q, t = ref.quantize(z)
    _, rms = _unit(h, eps)
    t = t.astype(np.float64) / rms[:, 0]
    return q, t, np.abs(t) * (unit_error(h.shape[1]) + 3 * U32)


def norm_grad(d, h, gain, eps, dh=None):
    """(dx, its bound, dgain, its bound)."""
    d, g = d.astype(np.float64), gain.astype(np.float64)
    m, k = d.shape
    n, rms = _unit(h, eps)
    z = d * g
    c = (z * n).sum(1, keepdims=True) / max(k, 1)
    size = np.abs(z * n).sum(1, keepdims=True) / max(k, 1)
    e = unit_error(k)
    dx = (z - n * c) / rms
    # n and 1 / rms are off by e each, c by e, its products and its sum
    bound = (np.abs(z) * (e + 4 * U32) + np.abs(n) * size * (4 * e + (row_depth(k) + 6) * U32)) / rms
    if dh is not None:
        dx = dx + dh.astype(np.float64)
        bound = bound + U32 * np.abs(dx)
    dg = (d * n).sum(0)
    depth = min(m, 1100 + m // 256) + 8     # rows of a workgroup, then the workgroups
    return dx, bound, dg, np.abs(d * n).sum(0) * (e + (depth + 2) * U32)
