"""Performance cases of the operators around the scaled int8 products: the norm in front of them, low-rank
adapters beside them, and the loss behind the last one.

`listed()` names the cases, `draw(rng)` gives more of the same ranges. The operators, with W[k, n] int8 and
s[n] the channels' scales, x^ the rows of x rounded to int8 (q) with one scale (t) each:

  norm         h = x + r in x's type, y = h / sqrt(mean(h^2) + eps) * gain, as int8 rows (`rows`) or in x's type
  norm_grad    the gradients of `norm` in h and the gain, from dy and the residual's own gradient dh
  adapted      y = x^ . (W s) + c (x . down_a^T) . up_a^T, with the adapter a of each row's own (or none)
  adapted_grad the gradients of `adapted` in x (through the rounding), down and up, W frozen
  loss         log(sum_j exp(l_ij)) - l_i,target_i of each row, l = x^ . (W s), x as floating rows or as the
               int8 rows and scales (dtype i8) that the last norm gives
  loss_grad    the mean of `loss` over the rows that have a target, and its gradient in x, W frozen

A row's scale is its largest magnitude / 127 (0 for a row of zeros) and its values are rounded to the
nearest, ties to even. Activations are normal with a few large channels, as a transformer's are, weights
normal with a deviation of 32 clipped to int8, and the last rows of a batch are padding tokens: zeros, no
adapter, no target.
"""
import math

import torch

own = False        # true: the framework's operators; false: their plain form

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i8": torch.float32}
EPS = 1e-6
SCALING = 0.5
IGNORED = -100
MOST_MACS = 2 * 10**11     # of a drawn case; the largest listed one has 1.1e12
MOST_BYTES = 400 * 2**20   # operands and results of a drawn case


def _norm(op, m, k, dtype="bf16", residual=True, rows=True):
    return {"op": op, "m": m, "k": k, "dtype": dtype, "residual": residual, "rows": rows}


def _adapted(op, m, k, n, rank, adapters, dtype="bf16", segments=True):
    return {"op": op, "m": m, "k": k, "n": n, "rank": rank, "adapters": adapters, "dtype": dtype,
            "segments": segments}


def _loss(op, m, k, n, dtype="bf16"):
    return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype}


def listed():
    return [
        # One sequence's decode step: the residual's addition and the norm in front of a projection.
        dict(_norm("norm", 1, 4096), name="norm_1"),
        # A prefill of 8192 tokens in front of a projection.
        dict(_norm("norm", 8192, 4096), name="norm_8192"),
        # Training with rows of odd length in float32: no row is aligned.
        dict(_norm("norm_grad", 333, 1001, "f32", rows=False), name="norm_grad_odd"),
        # Training on a batch of 4096 tokens.
        dict(_norm("norm_grad", 4096, 4096, rows=False), name="norm_grad_4096"),
        # A decode batch of 48 requests, in no order, of 32 adapters, through an up projection.
        dict(_adapted("adapted", 48, 4096, 14336, 16, 32, segments=False), name="adapted_48"),
        # Prefill of 2000 tokens of requests with 5 adapters of a high rank.
        dict(_adapted("adapted", 2000, 4096, 4096, 64, 5), name="adapted_2000"),
        # Training of three adapters with an odd rank through a layer of odd sizes.
        dict(_adapted("adapted_grad", 300, 999, 1001, 5, 3, "f32"), name="adapted_grad_odd"),
        # Training of one adapter on a batch of 4096 tokens.
        dict(_adapted("adapted_grad", 4096, 4096, 4096, 16, 1), name="adapted_grad_4096"),
        # The smallest loss: a few tokens over a small vocabulary.
        dict(_loss("loss", 5, 120, 1203, "f32"), name="loss_5"),
        # Scoring 2048 tokens, int8 rows behind the last norm, over a large vocabulary.
        dict(_loss("loss", 2048, 4096, 131072, "i8"), name="loss_2048"),
        # A training step's loss over a vocabulary of odd size.
        dict(_loss("loss_grad", 100, 333, 5003, "f16"), name="loss_grad_odd"),
        # A training step's loss of 2048 tokens.
        dict(_loss("loss_grad", 2048, 4096, 65536), name="loss_grad_2048"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _to64(v):
    return max(64, (v + 32) // 64 * 64)


def draw(rng):
    while True:
        op = rng.choice(("norm", "norm_grad", "adapted", "adapted_grad", "loss", "loss_grad"))
        # Decode batches (which have no gradient), prefill and training batches.
        if not op.endswith("grad") and rng.random() < 0.4:
            m = _log_int(rng, 1, 64)
        else:
            m = _log_int(rng, 65, 8192)
        k = _log_int(rng, 64, 16384)
        n = _log_int(rng, 200, 131072) if op.startswith("loss") else _log_int(rng, 64, 16384)
        if rng.random() < 0.6:
            k, n = _to64(k), _to64(n)
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        if op.startswith("norm"):
            c = _norm(op, m, k, dtype, residual=rng.random() < 0.7, rows=op == "norm" and rng.random() < 0.6)
        elif op.startswith("adapted"):
            c = _adapted(op, m, k, n, _log_int(rng, 1, 128), _log_int(rng, 1, 64), dtype,
                         segments=rng.random() < 0.6)
        else:
            c = _loss(op, m, k, n, rng.choice(("i8", "i8", "f32")) if op == "loss" else dtype)
        w = work(c)
        if w["flops"] <= 2 * MOST_MACS and w["bytes"] <= MOST_BYTES:
            return c


def _activations(g, m, k, live, dtype):
    x = torch.randn((m, k), device=DEV, generator=g)
    x *= torch.where(torch.rand(k, device=DEV, generator=g) < 0.005, 12.0, 1.0)
    x[live:] = 0.0
    return x.to(dtype)


def _weights(g, k, n):
    w = torch.empty((k, n), device=DEV).normal_(0.0, 32.0, generator=g)
    s = torch.rand(n, device=DEV, generator=g) + 0.5
    return w.round_().clamp_(-127, 127).to(torch.int8), s * (1.0 / (32.0 * math.sqrt(k)))


def _tensors(case, seed):
    """The operands, the same for prepare and exact."""
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    op, m, k, dtype = case["op"], case["m"], case["k"], DTYPES[case["dtype"]]
    live = m - m // 50
    v = {}
    if op.startswith("norm"):
        v["gain"] = 1.0 + 0.2 * torch.randn(k, device=DEV, generator=g)
        v["x"] = _activations(g, m, k, live, dtype)
        r = (torch.randn((m, k), device=DEV, generator=g) * 0.5).to(dtype) if case["residual"] else None
        if op == "norm_grad":       # x is h, r the residual's own gradient
            d = torch.randn((m, k), device=DEV, generator=g) * 1e-3
            d[live:] = 0.0
            v["d"] = d.to(dtype)
            r = None if r is None else r * 1e-3
        v["r"] = r
        return v
    n = case["n"]
    v["w"], v["s"] = _weights(g, k, n)
    v["x"] = _activations(g, m, k, live, dtype)
    if op.startswith("adapted"):
        L, rank = case["adapters"], case["rank"]
        v["down"] = (torch.randn((L, rank, k), device=DEV, generator=g) / math.sqrt(k)).to(dtype)
        v["up"] = (torch.randn((L, n, rank), device=DEV, generator=g) * (0.3 / math.sqrt(rank))).to(dtype)
        if case["segments"]:        # tokens of a request lie together
            cuts = torch.randint(0, m + 1, (2 * L - 1,), generator=g, device=DEV).sort().values
            which = torch.bucketize(torch.arange(m, device=DEV), cuts, right=True) % L
        else:
            which = torch.randint(0, L, (m,), generator=g, device=DEV)
            which[torch.rand(m, device=DEV, generator=g) < 0.1] = -1
        which[live:] = -1
        v["which"] = which.to(torch.int32)
        if op == "adapted_grad":
            d = torch.randn((m, n), device=DEV, generator=g) * 1e-3
            d[live:] = 0.0
            v["d"] = d.to(dtype)
        return v
    # A model that has learnt something: the target's logit stands out by about 8.
    target = torch.randint(0, n, (m,), generator=g, device=DEV)
    toward = v["w"].t().index_select(0, target).float() * (8.0 / 32.0 / math.sqrt(k))
    v["x"] = torch.where(torch.arange(m, device=DEV)[:, None] < live, v["x"].float() + toward, 0.0).to(dtype)
    target[live:] = IGNORED
    v["target"] = target
    if case["dtype"] == "i8":
        q, t = _quantised(v["x"])
        v["x"] = (q.to(torch.int8), t)
    return v


def prepare(case, seed):
    v = _tensors(case, seed)
    v.update(op=case["op"], dtype=DTYPES[case["dtype"]], rows=case.get("rows"))
    if v["op"].startswith("adapted"):
        v["count"] = case["adapters"]
    if own:
        # A model's weights, and the adapters that are served, are laid out once, when they are loaded.
        from veritac_amd.specializations.hip_gemm import adapters, scaled
        if "w" in v:
            v["packed"] = scaled.pack_linear(v["w"], v["s"])
        if v["op"] == "adapted":
            v["served"] = adapters.pack_adapters(v["down"], v["up"], scaling=SCALING)
    if v["op"] == "loss_grad":
        v["x"].requires_grad_()
    return v


def _run_own(v):
    from veritac_amd.specializations.hip_gemm import adapters, losses, norms, scaled
    op = v["op"]
    if op == "norm":
        if v["rows"]:
            out = norms.norm_rows(v["x"], v["gain"], residual=v["r"], eps=EPS)
            rows = out if v["r"] is None else out[0]
            return rows.dequantize(v["dtype"]) if v["r"] is None else (rows.dequantize(v["dtype"]), out[1])
        return norms.norm(v["x"], v["gain"], residual=v["r"], eps=EPS)
    if op == "norm_grad":
        return norms.norm_grad(v["d"], v["x"], v["gain"], dh=v["r"], eps=EPS)
    if op == "adapted":
        return adapters.adapted(v["x"], v["packed"], v["served"], v["which"])
    if op == "adapted_grad":
        # Trained adapters change between calls: they are given as they are.
        return adapters.adapted_grad(v["d"], v["x"], v["packed"], (v["down"], v["up"], SCALING), v["which"])
    if op == "loss":
        x = scaled.QuantRows(*v["x"]) if isinstance(v["x"], tuple) else v["x"]
        return losses.cross_entropy(x, v["packed"], v["target"], reduction="none")
    loss = losses.cross_entropy(v["x"], v["packed"], v["target"])
    return loss.detach(), torch.autograd.grad(loss, v["x"])[0]


def _quantised(z):
    """The rows of z as whole numbers q and scales t, in 32 bits."""
    top = z.abs().amax(1)
    some = top > 0
    inv = torch.where(some, torch.full_like(top, 127.0) / torch.where(some, top, 1.0), 0.0)
    return torch.round(z * inv[:, None]), torch.where(some, top * (1.0 / 127.0), 0.0)


def _product(v):
    x = v["x"]
    q, t = (x[0].float(), x[1]) if isinstance(x, tuple) else _quantised(x.float())
    return (q @ v["w"].float()) * t[:, None] * v["s"]


def _of_row(v):
    """[m, adapters * rank]: 1 where a column is of the row's adapter."""
    own_of = v["which"][:, None] == torch.arange(v["count"], device=DEV)
    return own_of.float().repeat_interleave(v["down"].shape[1], dim=1)


def _plain_norm(v):
    h = v["x"] if v["r"] is None else (v["x"].float() + v["r"].float()).to(v["dtype"])
    hf = h.float()
    inv = 1.0 / torch.sqrt((hf * hf).mean(1) + EPS)
    z = hf * v["gain"]
    if v["rows"]:
        q, t = _quantised(z)
        y = (q * (t * inv)[:, None]).to(v["dtype"])
    else:
        y = (z * inv[:, None]).to(v["dtype"])
    return y if v["r"] is None else (y, h)


def _plain_norm_grad(v):
    h, d = v["x"].float(), v["d"].float()
    inv = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    z = d * v["gain"]
    dx = inv * (z - h * (inv * inv * (z * h).mean(1, keepdim=True)))
    if v["r"] is not None:
        dx = dx + v["r"].float()
    return dx.to(v["dtype"]), (d * h * inv).sum(0)


def _plain_adapted(v):
    x, mask = v["x"].float(), _of_row(v) * SCALING
    down = v["down"].float().flatten(0, 1)                          # [adapters * rank, k]
    up = v["up"].float().transpose(1, 2).flatten(0, 1)              # [adapters * rank, n]
    u = (x @ down.t()) * mask
    if v["op"] == "adapted":
        return (_product(v) + u @ up).to(v["dtype"])
    d = v["d"].float()
    g = (d @ up.t()) * mask
    dx = (d * v["s"]) @ v["w"].float().t() + g @ down
    d_down = (g.t() @ x).reshape(v["down"].shape)
    d_up = (u.t() @ d).reshape(v["count"], -1, d.shape[1]).transpose(1, 2).contiguous()
    return dx.to(v["dtype"]), d_down.to(v["dtype"]), d_up.to(v["dtype"])


def _plain_loss(v):
    logits, target = _product(v), v["target"]
    has = target >= 0
    at = torch.where(has, target, 0)
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    mine = logits.gather(1, at[:, None])
    loss = torch.where(has, ((top - mine) + torch.log(total))[:, 0], 0.0)
    if v["op"] == "loss":
        return loss
    count = has.sum()
    p = e / total
    p.scatter_add_(1, at[:, None], torch.full_like(mine, -1.0))
    p *= (has / count)[:, None]
    return loss.sum() / count, ((p * v["s"]) @ v["w"].float().t()).to(v["dtype"])


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_grad":
        return _plain_norm_grad(state)
    if op.startswith("adapted"):
        return _plain_adapted(state)
    with torch.no_grad():
        return _plain_loss(state)


def work(case):
    op, m, k, e = case["op"], case["m"], case["k"], {"f32": 4, "i8": 1}.get(case["dtype"], 2)
    if op == "norm":
        y = m * (k + 4) if case["rows"] else m * k * e
        return {"bytes": m * k * e * (3 if case["residual"] else 1) + y + 4 * k, "flops": 6.0 * m * k}
    if op == "norm_grad":
        return {"bytes": m * k * e * (4 if case["residual"] else 3) + 8 * k, "flops": 12.0 * m * k}
    n = case["n"]
    weights = n * (k + 4)
    if op.startswith("adapted"):
        rank = case["rank"]
        used = min(case["adapters"], m) * rank * (k + n) * e
        if op == "adapted":
            return {"bytes": weights + used + m * (k + n) * e + 4 * m, "flops": 2.0 * m * (n * k + rank * (n + k))}
        return {"bytes": weights + 2 * used + m * (2 * k + n) * e + 4 * m,
                "flops": 2.0 * m * (n * k + 3 * rank * (n + k))}
    if op == "loss":
        return {"bytes": weights + m * k * e + 16 * m, "flops": 2.0 * m * n * k}
    return {"bytes": weights + 2 * m * k * e + 8 * m, "flops": 4.0 * m * n * k}


def _exact_rows(z):
    """The rows that int8 rows stand for, in 64 bits."""
    top = z.abs().max(dim=1, keepdim=True).values
    return torch.where(top > 0, torch.round(z * 127 / top.clamp_min(1e-300)), 0.0) * top / 127


def _exact_norm(case, v):
    f64 = torch.float64
    x, gain = v["x"].to(f64), v["gain"].to(f64)
    rms = lambda a: torch.sqrt(a.square().sum(1, keepdim=True) / case["k"] + EPS)  # noqa: E731
    if case["op"] == "norm":
        h = x if v["r"] is None else (x + v["r"].to(f64)).to(v["x"].dtype).to(f64)
        y = h / rms(h) * gain
        y = _exact_rows(y) if case["rows"] else y
        return y if v["r"] is None else (y, h)
    d = v["d"].to(f64)
    unit = x / rms(x)
    z = d * gain
    dx = (z - unit * ((z * unit).sum(1, keepdim=True) / case["k"])) / rms(x)
    return dx if v["r"] is None else dx + v["r"].to(f64), (d * unit).sum(0)


def _exact_adapted(case, v):
    f64 = torch.float64
    x, w = v["x"].to(f64), v["w"].to(f64) * v["s"].to(f64)
    grad = case["op"] == "adapted_grad"
    d = v["d"].to(f64) if grad else None
    first = torch.mm(d, w.t().contiguous()) if grad else torch.mm(_exact_rows(x), w)
    d_down, d_up = torch.zeros(v["down"].shape, dtype=f64, device=DEV), torch.zeros(v["up"].shape, dtype=f64, device=DEV)
    for a in range(case["adapters"]):
        i = torch.nonzero(v["which"] == a)[:, 0]
        down, up = v["down"][a].to(f64), v["up"][a].to(f64)
        u = SCALING * torch.mm(x[i], down.t().contiguous())
        if not grad:
            first[i] += torch.mm(u, up.t().contiguous())
            continue
        t = SCALING * torch.mm(d[i], up)
        first[i] += torch.mm(t, down)
        d_down[a] = torch.mm(t.t().contiguous(), x[i])
        d_up[a] = torch.mm(d[i].t().contiguous(), u)
    return (first, d_down, d_up) if grad else first


def exact(case, seed):
    f64 = torch.float64
    v = _tensors(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(case, v)
    if case["op"].startswith("adapted"):
        return _exact_adapted(case, v)
    has = v["target"] >= 0
    w = v["w"].to(f64) * v["s"].to(f64)
    x = v["x"]
    x = x[0].to(f64) * x[1].to(f64)[:, None] if isinstance(x, tuple) else _exact_rows(x.to(f64))
    log_p = torch.log_softmax(torch.mm(x, w), dim=1)
    at = v["target"].clamp_min(0)[:, None]
    loss = torch.where(has, -log_p.gather(1, at)[:, 0], 0.0)
    if case["op"] == "loss":
        return loss
    p = log_p.exp_()
    p.scatter_add_(1, at, torch.full(at.shape, -1.0, dtype=f64, device=DEV))
    p[~has] = 0.0
    return loss.sum() / has.sum(), torch.mm(p, w.t().contiguous()) / has.sum()
