"""The scaled operators in 64 bits (numpy), and how far a 32-bit evaluation may be from them.

U32 is float32's unit roundoff; OUT the output type's, and its smallest step near zero."""
import numpy as np

U32 = 2.0**-24
OUT = {"float32": (0.0, 0.0), "float16": (2.0**-11, 2.0**-25), "bfloat16": (2.0**-8, 0.0)}


def quantize(x):
    """(q int8, t float32) of float32 rows, the operations of the definition in float32."""
    x = np.asarray(x, np.float32)
    q = np.zeros(x.shape, np.int8)
    t = np.zeros(x.shape[0], np.float32)
    for i, row in enumerate(x):
        top = np.abs(row).max() if row.size else np.float32(0)
        if not np.isfinite(top):
            t[i] = np.nan
        elif top >= np.float32(2.0**-120):
            t[i] = top * np.float32(1.0 / 127.0)
            q[i] = np.rint(row * (np.float32(127.0) / top)).astype(np.int8)
    return q, t


def products(q, t, w, s):
    acc = q.astype(np.float64) @ w.astype(np.float64)
    return acc * t.astype(np.float64)[:, None] * s.astype(np.float64)


def linear(q, t, w, s, bias=None):
    """(y, bound): the sum's conversion, two products and the bias' addition round once each."""
    y = products(q, t, w, s)
    bound = 4 * U32 * np.abs(y)
    if bias is not None:
        bound = bound + U32 * (np.abs(y) + np.abs(bias))
        y = y + bias
    return y, bound


C, A = np.sqrt(2 / np.pi), 0.044715


def act(g, kind):
    """(act(g), act'(g), |argument of the exponential|)."""
    g = np.clip(g, -1e30, 1e30)
    if kind == "silu":
        z, dz = g, np.ones_like(g)
    else:
        h = np.clip(g, -40, 40)
        z, dz = 2 * C * (h + A * h**3), 2 * C * (1 + 3 * A * h**2)
    e = np.exp(-np.abs(z))
    p = np.where(z >= 0, 1 / (1 + e), e / (1 + e))
    np_ = np.where(z >= 0, e / (1 + e), 1 / (1 + e))
    return g * p, p + np.where(np.abs(z) < 700, g * p * np_ * dz, 0.0), np.abs(z)


def gated(q, t, wg, sg, wu, su, kind):
    """(h, bound). g and u round three times; the logistic function's relative error is the
    absolute one of its argument (six roundings of it, and |dz/dg| of g's) plus a few roundings;
    below 2^-126 nothing is kept."""
    g, u = products(q, t, wg, sg), products(q, t, wu, su)
    a, _, z = act(g, kind)
    h = a * u
    return h, np.abs(h) * (32 + 16 * np.minimum(z, 600)) * U32 + 2.0**-126 * (1 + np.abs(u) + np.abs(g))


def linear_grad(d, w, s, half):
    terms = d.astype(np.float64) * s.astype(np.float64)
    return _grad([(terms, w)], np.abs(terms).max(axis=1, initial=0.0), half, 0.0)


def gated_grad(d, q, t, wg, sg, wu, su, kind, half):
    g, u = products(q, t, wg, sg), products(q, t, wu, su)
    a, slope, z = act(g, kind)
    d = d.astype(np.float64)
    cols = np.maximum(np.abs(wg.astype(np.int64)).sum(0), np.abs(wu.astype(np.int64)).sum(0))
    reach = (cols * np.abs(sg.astype(np.float64) * su)).max(initial=0.0)
    bound = np.abs(d).max(axis=1, initial=0.0) * np.abs(t.astype(np.float64)) * reach * 128 * 1.13
    tg, tu = d * u * slope * sg, d * a * su
    # the slope is a sum of terms up to |act'| + |g p (1 - p) dz|, each as uncertain as in gated
    rough = np.minimum(z, 600) * 16 * U32 + 32 * U32
    more = (np.abs(d * u * sg) * 2.3 * rough) @ np.abs(wg.astype(np.float64)).T
    more += (np.abs(tu) * rough) @ np.abs(wu.astype(np.float64)).T
    return _grad([(tg, wg), (tu, wu)], bound, half, more)


def _grad(parts, row_bound, half, more):
    """(dx, bound) of terms . W^T. Terms are rounded to 11 bits (22 in two halves), or to steps of
    2^-24 of a row whose bound is at least 2^14 there; sums of 32 products, then of those."""
    dx, size, steps, depth = 0.0, 0.0, 0.0, 0
    for terms, w in parts:
        w = w.astype(np.float64)
        dx = dx + terms @ w.T
        size = size + np.abs(terms) @ np.abs(w).T
        steps = steps + np.abs(w).sum(axis=1)
        depth += -(-w.shape[1] // 32)
    unit = 2.0**-11 if half else 2.0**-22
    bound = size * (unit + 4 * U32 + (depth + 32) * 2 * U32)
    return dx, bound + np.outer(row_bound * 2.0**-38, steps) + more


def check(got, want, bound, dtype, what):
    """got (a torch tensor of `dtype`) within the bound and its own rounding of want."""
    unit, least = OUT[str(dtype).replace("torch.", "")]
    if not unit:
        unit = U32
    got = got.detach().cpu().double().numpy().reshape(want.shape)
    top = {"float16": 65504.0, "bfloat16": 3.3895e38, "float32": 3.4028e38}[str(dtype).replace("torch.", "")]
    over = np.abs(want) >= top * (1 - 2.0**-8)
    allowed = bound * (1 + unit) + unit * np.abs(want) + least
    off = np.abs(got - want)
    bad = ~(off <= allowed) & ~over
    assert not bad.any(), "%s: %d of %d outside, worst %g against %g at %s" % (
        what, bad.sum(), bad.size, off[bad].max(), allowed[bad][np.argmax(off[bad])],
        np.unravel_index(np.argmax(np.where(bad, off / allowed, 0)), bad.shape))
