"""Performance cases of the scaled int8 operators: linear layers and gated feed-forward products whose
weights are int8 with a scale for each output channel and whose activations are int8 with a scale for
each token.

`listed()` names the cases, `draw(rng)` gives more of the same ranges. The operators, with W[k, n] int8
and s[n] the channels' scales:

  linear       y = x^ . (W s) + bias: x^ = q t, the rows of x rounded to int8 (q) with one scale (t) each
  gated        h = act(x^ . (Wg sg)) * (x^ . (Wu su)), act silu or gelu (its tanh form)
  linear_grad  dx = (dy s) . W^T, the gradient of `linear` in x^ with the weights frozen
  gated_grad   the gradient of `gated` in x^ from dh and the int8 rows that the forward pass made

A row's scale is its largest magnitude / 127 (0 for a row of zeros) and its values are rounded to the
nearest, ties to even. Activations are normal with a few large channels, as a transformer's are, weights
normal with a deviation of 32 clipped to int8, and the last rows of a batch are padding tokens of zeros.
"""
import math

import torch

own = False        # true: the framework's operators; false: their plain form

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_MACS = 2 * 10**11     # of a drawn case; the largest listed one has 9.6e11
MOST_BYTES = 400 * 2**20   # operands and result of a drawn case


def _case(op, m, k, n, dtype="bf16", bias=False, act="silu", q=False):
    return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "bias": bias, "act": act, "q": q}


def listed():
    return [
        # The smallest call: a few tokens through a small layer, where launches are everything.
        dict(_case("linear", 5, 120, 72, "f32"), name="linear_small"),
        # One sequence's decode step through an up projection.
        dict(_case("linear", 1, 4096, 14336), name="linear_1"),
        # A decode batch of 48 through a down projection: a long row and few channels.
        dict(_case("linear", 48, 14336, 4096, "f16", bias=True), name="linear_48"),
        # Prefill of a ragged 2000-token prompt through a square projection.
        dict(_case("linear", 2000, 4096, 4096, bias=True), name="linear_2000"),
        # The large product of rows that are int8 already, as projections that share an input have them.
        dict(_case("linear", 8192, 8192, 8192, q=True), name="linear_8192"),
        # One sequence's decode step through the gate and up projections.
        dict(_case("gated", 1, 4096, 14336), name="gated_1"),
        # A gated block of odd sizes in float32: no row of anything is aligned.
        dict(_case("gated", 333, 1001, 2731, "f32", act="gelu"), name="gated_odd"),
        # Prefill of 2000 tokens through the gate and up projections.
        dict(_case("gated", 2000, 4096, 14336), name="gated_2000"),
        # The gradient through a small layer of odd sizes.
        dict(_case("linear_grad", 300, 999, 1001, "f32"), name="linear_grad_odd"),
        # The gradient through a square projection for a batch of 4096 tokens.
        dict(_case("linear_grad", 4096, 4096, 4096), name="linear_grad_4096"),
        # The gradient through a gated block of odd sizes.
        dict(_case("gated_grad", 100, 333, 1203, "f16", act="gelu"), name="gated_grad_odd"),
        # The gradient through the gate and up projections for 2048 tokens.
        dict(_case("gated_grad", 2048, 4096, 14336), name="gated_grad_2048"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _to64(v):
    return max(64, (v + 32) // 64 * 64)


def _pairs(case):
    return 2 if case["op"].startswith("gated") else 1


def draw(rng):
    while True:
        op = rng.choices(("linear", "gated", "linear_grad", "gated_grad"), (5, 4, 2, 3))[0]
        # Decode batches (which have no gradient), prefill and training batches.
        if not op.endswith("grad") and rng.random() < 0.4:
            m = _log_int(rng, 1, 64)
        else:
            m = _log_int(rng, 65, 8192)
        k, n = _log_int(rng, 64, 16384), _log_int(rng, 64, 16384)
        if rng.random() < 0.6:
            k, n = _to64(k), _to64(n)
        if 3072 in (m, k, n):
            continue
        c = _case(op, m, k, n, rng.choice(("bf16", "bf16", "f16", "f32")),
                  bias=op == "linear" and rng.random() < 0.3, act=rng.choice(("silu", "gelu")),
                  q=not op.endswith("grad") and rng.random() < 0.25)
        w = work(c)
        if w["flops"] <= 2 * MOST_MACS and w["bytes"] <= MOST_BYTES:
            return c


def _weights(g, k, n):
    w = torch.empty((k, n), device=DEV).normal_(0.0, 32.0, generator=g)
    s = torch.rand(n, device=DEV, generator=g) + 0.5
    return w.round_().clamp_(-127, 127).to(torch.int8), s * (1.0 / (32.0 * math.sqrt(k)))


def _tensors(case, seed):
    """The operands, the same for prepare and exact: x (or q and t), dy, weights, scales, bias."""
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    m, k, n, dtype = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
    live = m - m // 50
    v = {}
    if case["q"] or case["op"] == "gated_grad":
        v["q"] = torch.randint(-127, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
        v["t"] = (torch.rand(m, device=DEV, generator=g) + 0.5) * (4.0 / 127.0)
        v["t"][live:] = 0.0
    elif case["op"] in ("linear", "gated"):
        x = torch.randn((m, k), device=DEV, generator=g)
        x *= torch.where(torch.rand(k, device=DEV, generator=g) < 0.005, 12.0, 1.0)
        x[live:] = 0.0
        v["x"] = x.to(dtype)
    if case["op"].endswith("grad"):
        d = torch.randn((m, n), device=DEV, generator=g) * 1e-3
        d[live:] = 0.0
        v["d"] = d.to(dtype)
    v["w"] = [_weights(g, k, n) for _ in range(_pairs(case))]
    v["bias"] = torch.randn(n, device=DEV, generator=g) * 0.1 if case["bias"] else None
    return v


def prepare(case, seed):
    v = _tensors(case, seed)
    v["op"], v["act"], v["dtype"] = case["op"], case["act"], DTYPES[case["dtype"]]
    if own:
        # A model's weights are laid out once, when it is loaded.
        from veritac_amd.specializations.hip_gemm import scaled
        if len(v["w"]) == 2:
            (wg, sg), (wu, su) = v["w"]
            v["packed"] = scaled.pack_gated(wg, sg, wu, su)
        else:
            v["packed"] = scaled.pack_linear(*v["w"][0], bias=v["bias"])
    return v


def _run_own(v):
    from veritac_amd.specializations.hip_gemm import scaled
    x = scaled.QuantRows(v["q"], v["t"]) if "q" in v else v.get("x")
    if v["op"] == "linear":
        return scaled.linear(x, v["packed"], out_dtype=v["dtype"])
    if v["op"] == "gated":
        return scaled.gated(x, v["packed"], act=v["act"], out_dtype=v["dtype"])
    if v["op"] == "linear_grad":
        return scaled.linear_grad(v["d"], v["packed"])
    return scaled.gated_grad(v["d"], x, v["packed"], act=v["act"])


def _rows(v):
    """x^ as q (whole numbers) and t, in 32 bits."""
    if "q" in v:
        return v["q"].float(), v["t"]
    x = v["x"].float()
    top = x.abs().amax(1)
    some = top > 0
    top127 = torch.full_like(top, 127.0)
    inv = torch.where(some, top127 / torch.where(some, top, top127), 0.0)
    return torch.round(x * inv[:, None]), torch.where(some, top * (1.0 / 127.0), 0.0)


def _product(q, t, w, s):
    return (q @ w.float()) * t[:, None] * s


def _act(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _act_slope(g, act):
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return p * (1.0 + g * (1.0 - p))
    th = torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))
    return 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * 0.7978845608028654 * (1.0 + 0.134145 * g * g)


def run(state):
    if own:
        return _run_own(state)
    v, dtype = state, state["dtype"]
    if v["op"] == "linear":
        y = _product(*_rows(v), *v["w"][0])
        return (y if v["bias"] is None else y + v["bias"]).to(dtype)
    if v["op"] == "linear_grad":
        w, s = v["w"][0]
        return ((v["d"].float() * s) @ w.float().t()).to(dtype)
    q, t = _rows(v)
    (wg, sg), (wu, su) = v["w"]
    g, u = _product(q, t, wg, sg), _product(q, t, wu, su)
    if v["op"] == "gated":
        return (_act(g, v["act"]) * u).to(dtype)
    d = v["d"].float()
    dx = (d * u * _act_slope(g, v["act"]) * sg) @ wg.float().t()
    dx += (d * _act(g, v["act"]) * su) @ wu.float().t()
    return dx.to(dtype)


def work(case):
    m, k, n, e = case["m"], case["k"], case["n"], 4 if case["dtype"] == "f32" else 2
    p = _pairs(case)
    weights = p * n * (k + 4)
    rows = m * (k + 4)                      # int8 and a scale
    x = rows if case["q"] else m * k * e
    if case["op"] in ("linear", "gated"):
        return {"bytes": x + weights + (4 * n if case["bias"] else 0) + m * n * e, "flops": 2.0 * p * m * n * k}
    if case["op"] == "linear_grad":
        return {"bytes": weights + m * (n + k) * e, "flops": 2.0 * m * n * k}
    return {"bytes": rows + weights + m * (n + k) * e, "flops": 8.0 * m * n * k}


def exact(case, seed):
    v = _tensors(case, seed)
    f64 = torch.float64
    if "q" in v:
        xhat = v["q"].to(f64) * v["t"].to(f64).unsqueeze(1)
    elif "x" in v:
        x = v["x"].to(f64)
        step = x.abs().max(dim=1, keepdim=True).values / 127
        xhat = torch.where(step > 0, torch.round(x / step.clamp_min(1e-300)), 0.0) * step
    w = [a.to(f64) * s.to(f64) for a, s in v["w"]]
    if case["op"] == "linear":
        y = torch.mm(xhat, w[0])
        return y if v["bias"] is None else y + v["bias"].to(f64)
    if case["op"] == "linear_grad":
        return torch.mm(v["d"].to(f64), w[0].t().contiguous())
    gate, up = torch.mm(xhat, w[0]), torch.mm(xhat, w[1])
    if case["act"] == "silu":
        cdf = torch.sigmoid(gate)
        slope = cdf + gate * cdf * (1 - cdf)
    else:
        c = math.sqrt(2 / math.pi)
        cdf = torch.sigmoid(2 * c * (gate + 0.044715 * gate**3))     # (1 + tanh z) / 2 = sigmoid(2 z)
        slope = cdf + gate * 2 * cdf * (1 - cdf) * c * (1 + 3 * 0.044715 * gate**2)
    if case["op"] == "gated":
        return gate * cdf * up
    d = v["d"].to(f64)
    return (torch.mm(d * up * slope, w[0].t().contiguous())
            + torch.mm(d * gate * cdf, w[1].t().contiguous()))
