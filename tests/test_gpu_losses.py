"""Softmax cross entropy over int8 weights and its gradient (needs a gfx950 GPU) against 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import scaled_ref as ref
from loss_ref import CASES, Loss
from test_gpu_scaled import dev, packed, rows, say, up, weights  # noqa: F401
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import losses, norms, scaled

pytestmark = pytest.mark.gpu

KINDS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def operands(m, k, n, dtype, seed=0):
    """Rows that lean towards their targets, so that losses are from next to nothing to large."""
    rng = np.random.default_rng(m * 1009 + k * 31 + n + seed)
    w, s = weights(rng, k, n, -128)
    target = rng.integers(0, n, m)
    x, _ = rows(rng, m, k, torch.float32)
    lean = rng.choice([0.0, 4.0, 30.0], m)[:, None] / (32 * max(k, 1)**0.5)
    x = (x + torch.from_numpy((w[:, target].T * lean).astype(np.float32))).to(dtype)
    if m > 2:
        target[rng.random(m) < 0.2] = -100
        target[0] = n - 1
    bias = rng.normal(0, 0.3, n).astype(np.float32) if (m + n) % 2 else None
    return x, w, s, bias, target


def close(got, want, bound, what):
    ref.check(got, np.asarray(want), np.asarray(bound), got.dtype, what)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n", CASES)
def test_loss_and_gradient(dev, m, k, n, kind):
    dtype = KINDS[kind]
    say("loss", m, k, n, kind)
    x, w, s, bias, target = operands(m, k, n, dtype)
    q, t = ref.quantize(x.float().numpy())
    L = Loss(q, t, w, s, bias, target)
    W, xd, td = packed(dev, w, s, bias), x.to(dev), up(target, dev)
    each = losses.cross_entropy(xd, W, td, reduction="none")
    close(each, L.loss, L.bound, "losses")
    # int8 rows, not padded, and 32-bit targets
    again = losses.cross_entropy(scaled.QuantRows(up(q, dev), up(t, dev)), W, td.int(), reduction="none")
    assert torch.equal(again, each)
    xg = xd.clone().requires_grad_()
    if L.has.any():
        mean = losses.cross_entropy(xg, W, td)
        close(mean.detach(), *L.mean(), "mean")
        dx, = torch.autograd.grad(mean, xg)
        assert dx.dtype == dtype
        close(dx, *L.grad(np.full(m, 1 / L.has.sum()), kind == "bf16"), "dx of the mean")
    g = np.random.default_rng(m).normal(0, 1, m).astype(np.float32)
    g[m // 2] = 0.0
    loss = losses.cross_entropy(xg, W, td, reduction="none")
    dx, = torch.autograd.grad(loss, xg, up(g, dev))
    close(dx, *L.grad(g.astype(np.float64), kind == "bf16"), "dx of each")
    again, = torch.autograd.grad(losses.cross_entropy(xg, W, td, reduction="none"), xg, up(g, dev))
    assert torch.equal(again, dx)


@pytest.mark.parametrize("m", [4, 100, 300])
def test_masked_classes_and_far_logits(dev, m):
    """A bias of -inf, of the type's lowest value, or of +-3e4 leaves the other classes exact."""
    k, n = 256, 500
    x, w, s, _, target = operands(m, k, n, torch.float32)
    q, t = ref.quantize(x.numpy())
    target = np.where(target == -100, 7, target) % 50
    for low, shift in ((-np.inf, 0.0), (-3.4028234e38, 0.0), (-np.inf, 3e4), (-1e30, -3e4)):
        bias = np.full(n, shift, np.float32)
        bias[50:] = low
        L = Loss(q, t, w[:, :50], s[:50], bias[:50], target)
        W = packed(dev, w, s, bias)
        xg = x.to(dev).requires_grad_()
        loss = losses.cross_entropy(xg, W, up(target, dev), reduction="none")
        close(loss.detach(), L.loss, L.bound, "losses")
        dx, = torch.autograd.grad(loss.sum(), xg)
        want, bound = L.grad(np.ones(m), False)
        top = L.reach() * np.abs(s).max()     # the normaliser's, over all classes
        close(dx, want, bound + np.outer(top * 2.0**-38, np.abs(w.astype(np.float64)).sum(1)), "dx")
    # every class at the lowest value: as likely as each other
    bias = np.full(n, -3.4028234e38, np.float32)
    loss = losses.cross_entropy(x.to(dev), packed(dev, w, s, bias), up(target, dev), reduction="none")
    assert (loss - np.log(n)).abs().max() <= 64 * ref.U32 * np.log(n)
    none = losses.cross_entropy(x.to(dev), packed(dev, w, s, np.full(n, -np.inf, np.float32)), up(target, dev), reduction="none")
    assert none.isnan().all()
    # a target that is masked
    bias = np.zeros(n, np.float32)
    bias[target[0]] = -np.inf
    loss = losses.cross_entropy(x.to(dev), packed(dev, w, s, bias), up(target, dev), reduction="none")
    assert loss[0] == np.inf


@pytest.mark.parametrize("m", [5, 90, 300])
def test_rows_without_numbers_or_targets(dev, m):
    k, n = 300, 700
    x, w, s, bias, target = operands(m, k, n, torch.bfloat16)
    target[:] = 3
    target[1], target[2], target[3] = -100, n, -1
    x[4, 5] = float("nan")
    W = packed(dev, w, s, bias)
    xg = x.to(dev).requires_grad_()
    loss = losses.cross_entropy(xg, W, up(target, dev), reduction="none")
    assert loss[1] == 0 and loss[2:5].isnan().all() and loss[0].isfinite() and loss[5:].isfinite().all()
    dx, = torch.autograd.grad(loss.sum(), xg)
    assert not dx[1].any() and dx[2:5].isnan().all() and dx[0].isfinite().all() and dx[5:].isfinite().all()
    other = losses.cross_entropy(xg, W, up(target, dev), reduction="none", ignore_index=-1)
    assert other[3] == 0 and other[1].isnan()
    target[:] = -100
    mean = losses.cross_entropy(xg, W, up(target, dev))
    assert mean.isnan() and not torch.autograd.grad(mean, xg)[0].any()
    assert losses.cross_entropy(xg.detach(), W, up(target, dev), reduction="sum") == 0


def test_shapes_strides_and_sums(dev):
    x, w, s, bias, target = operands(24, 200, 600, torch.float16)
    W, xd, td = packed(dev, w, s, bias), x.to(dev), up(target, dev)
    want = losses.cross_entropy(xd, W, td, reduction="none")
    x3 = torch.zeros(4, 7, 203, device=dev, dtype=torch.float16)[:, :6, 2:202]
    x3.copy_(xd.reshape(4, 6, 200))
    got = losses.cross_entropy(x3, W, td.reshape(4, 6), reduction="none")
    assert got.shape == (4, 6) and torch.equal(got.reshape(-1), want)
    wide = torch.zeros(24, 2, dtype=torch.int64, device=dev)
    wide[:, 1] = td
    assert torch.equal(losses.cross_entropy(xd, W, wide[:, 1], reduction="none"), want)
    total = losses.cross_entropy(xd, W, td, reduction="sum")
    assert total.shape == () and abs(total.item() - want.double().sum().item()) <= 2 * ref.U32 * total.item()
    one = losses.cross_entropy(xd[5], W, td[5], reduction="none")
    assert one.shape == () and torch.equal(one, want[5])
    empty = losses.cross_entropy(xd[:0], W, td[:0], reduction="none")
    assert empty.shape == (0,) and losses.cross_entropy(xd[:0], W, td[:0], reduction="sum") == 0
    xg = xd.clone().requires_grad_()
    loss = losses.cross_entropy(xg, W, td, reduction="sum")
    loss *= 0.25                                    # in place, as accumulated steps do
    a, = torch.autograd.grad(loss, xg)
    b, = torch.autograd.grad(losses.cross_entropy(xg, W, td, reduction="sum") * 0.25, xg)
    assert torch.equal(a, b)


def test_gradient_against_differences(dev):
    """Of the float64 loss along a direction, in rows that the int8 rounding leaves alone."""
    m, k, n = 40, 128, 300
    rng = np.random.default_rng(5)
    w, s = weights(rng, k, n)
    q = rng.integers(-127, 128, (m, k)).astype(np.float32)
    q[:, 0] = 127
    x = torch.from_numpy(q * np.float32(2.0**-6))
    target = rng.integers(0, n, m)
    xg = x.to(dev).requires_grad_()
    dx, = torch.autograd.grad(losses.cross_entropy(xg, packed(dev, w, s), up(target, dev)), xg)
    W64, v = w.astype(np.float64) * s.astype(np.float64), rng.normal(0, 1, (m, k))

    def f(a):
        l = a @ W64
        top = l.max(1, keepdims=True)
        return (top[:, 0] + np.log(np.exp(l - top).sum(1)) - l[np.arange(m), target]).mean()
    a, h = x.double().numpy(), 1e-4
    slope = (f(a + h * v) - f(a - h * v)) / (2 * h)
    got = dx.double().cpu().numpy()
    # h^2 / 6 of third derivatives of a size of |l|^3 ~ 1, and 22-bit terms
    assert abs((got * v).sum() - slope) <= 1e-6 * (np.abs(got * v)).sum() + 1e-8


def test_behind_a_norm_and_captured(dev):
    """norm_rows -> loss as a graph, replayed with other inputs between eager work."""
    m, k, n = 130, 512, 3001
    x, w, s, bias, target = operands(m, k, n, torch.bfloat16)
    W, x, td, gain = packed(dev, w, s, bias), x.to(dev), up(target, dev), torch.ones(k, device=dev)

    def step():
        return losses.cross_entropy(norms.norm_rows(x, gain), W, td), losses.cross_entropy(x[:40], W, td[:40], reduction="none")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for seed in range(4):
        torch.manual_seed(seed)
        x.copy_(torch.randn(m, k))
        td.copy_(torch.randint(0, n, (m,)))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want)


def test_training_step_captured(dev):
    """Forward and backward in one graph, with an eager graph of other leaves alive beside it."""
    m, k, n = 140, 256, 1000
    x, w, s, bias, target = operands(m, k, n, torch.float32)
    W, td = packed(dev, w, s, bias), up(target, dev)
    side = torch.cuda.Stream()
    xs = x.to(dev).requires_grad_()
    eager = losses.cross_entropy(x.to(dev).requires_grad_(), W, td)

    def step():
        return torch.autograd.grad(losses.cross_entropy(xs, W, td), xs)[0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dx = step()
    for seed in range(3):
        with torch.no_grad():
            xs.copy_(torch.from_numpy(np.random.default_rng(seed).normal(0, 1, (m, k))))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, step())
    eager.backward()


def test_refusals(dev):
    x, w, s, bias, target = operands(6, 64, 100, torch.float32)
    W, xd, td = packed(dev, w, s, bias), x.to(dev), up(target, dev)
    G = scaled.pack_gated(up(w, dev), up(s, dev), up(w, dev), up(s, dev))
    for call in (lambda: losses.cross_entropy(xd, G, td), lambda: losses.cross_entropy(xd[:, :63], W, td),
                 lambda: losses.cross_entropy(xd, W, td[:5]), lambda: losses.cross_entropy(xd, W, td.float()),
                 lambda: losses.cross_entropy(xd, W, td.cpu()), lambda: losses.cross_entropy(xd, W, td, reduction="max"),
                 lambda: losses.cross_entropy(xd, W, td, ignore_index=1.0), lambda: losses.cross_entropy(x, W, td),
                 lambda: losses.cross_entropy(xd.clone().requires_grad_(), W, td, stream=5),
                 lambda: losses.cross_entropy(xd, scaled.pack_linear(up(w[:, :0], dev), up(s[:0], dev)), td)):
        with pytest.raises(HipGemmError):
            call()
