"""Norms, their int8 rows and gradients (needs a gfx950 GPU) against their formulas in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import norm_ref
import scaled_ref as ref
from test_gpu_scaled import dev, say, up  # noqa: F401
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import norms, scaled

pytestmark = pytest.mark.gpu

KINDS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# every kernel (threads by the row's length), odd lengths, one row and more rows than workgroups
SIZES = [(1, 1), (3, 7), (1, 128), (5, 511), (70, 513), (1, 1024), (333, 1001), (9, 2048), (2, 2055), (40, 4096),
         (3, 4097), (7, 8192), (3, 8200), (2, 16384), (4, 16390), (3, 40000), (5000, 64), (2100, 600), (1200, 2500)]


def host(rng, m, k, dtype, scale=1.0):
    """Random rows of a type, and their values."""
    x = rng.normal(0, 1, (m, k)) * np.where(rng.random(k) < 0.01, 12, 1) * scale
    t = torch.from_numpy(x).to(dtype)
    return t, t.double().numpy()


def total(x, r, dtype):
    """x + r rounded to the type, as values."""
    return torch.from_numpy(x + r).to(dtype).double().numpy()


def close(got, want, bound, what):
    ref.check(got, want, bound, got.dtype, what)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k", SIZES)
def test_norm(dev, m, k, kind):
    dtype = KINDS[kind]
    say("norm", m, k, kind)
    rng = np.random.default_rng(m * 131 + k)
    x, x64 = host(rng, m, k, dtype)
    r, r64 = host(rng, m, k, dtype, 0.5)
    wide = (m + k) % 2 == 0
    g = torch.from_numpy(1 + 0.3 * rng.normal(0, 1, k)).to(torch.float32 if wide else dtype)
    g64, eps = g.double().numpy(), 1e-5
    x, r, g = x.to(dev), r.to(dev), g.to(dev)
    close(norms.norm(x, g, eps=eps), *norm_ref.norm(x64, g64, eps), "norm")
    y, h = norms.norm(x, g, residual=r, eps=eps)
    h64 = total(x64, r64, dtype)
    assert np.array_equal(h.double().cpu().numpy(), h64)
    close(y, *norm_ref.norm(h64, g64, eps), "norm of the sum")
    for res, v in ((None, x64), (r, h64)):
        rows = norms.norm_rows(x, g, residual=res, eps=eps)
        if res is not None:
            rows, h2 = rows
            assert torch.equal(h2, h)
        q, t, bound = norm_ref.norm_rows(v, g64, eps)
        assert rows.padded and rows.shape == (m, k)
        assert np.array_equal(rows.data[:, :k].cpu().numpy(), q) and not rows.data[:, k:].any()
        close(rows.scale, t, bound, "scales")
        for to in KINDS.values():
            want = (rows.data[:, :k].float() * rows.scale[:, None]).to(to)
            assert torch.equal(rows.dequantize(to), want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k", SIZES)
def test_norm_grad(dev, m, k, kind):
    dtype = KINDS[kind]
    say("norm_grad", m, k, kind)
    rng = np.random.default_rng(m * 17 + k)
    h, h64 = host(rng, m, k, dtype)
    d, d64 = host(rng, m, k, dtype, 1e-2)
    e, e64 = host(rng, m, k, dtype, 1e-2)
    g = torch.from_numpy(1 + 0.3 * rng.normal(0, 1, k)).to(torch.float32 if k % 2 else dtype)
    eps = 1e-6
    for dh, dh64 in ((None, None), (e.to(dev), e64)):
        dx, dg = norms.norm_grad(d.to(dev), h.to(dev), g.to(dev), dh=dh, eps=eps)
        x64, xb, g64, gb = norm_ref.norm_grad(d64, h64, g.double().numpy(), eps, dh64)
        assert dg.dtype == g.dtype
        close(dx, x64, xb, "dx")
        close(dg, g64, gb, "dgain")
        again = norms.norm_grad(d.to(dev), h.to(dev), g.to(dev), dh=dh, eps=eps, gain_grad=False)
        assert again[1] is None and torch.equal(again[0], dx)


@pytest.mark.parametrize("kind,scale,eps", [("f32", 1e25, 1e-6), ("bf16", 3e37, 1e-6), ("f32", 1e-25, 0.0),
                                            ("bf16", 1e-37, 0.0), ("f32", 1e-30, 1e-6), ("bf16", 1e18, 0.0)])
@pytest.mark.parametrize("k", [300, 5000, 20000])
def test_squares_beyond_float32(dev, kind, scale, eps, k):
    """Rows whose squares overflow or vanish keep their norm."""
    dtype = KINDS[kind]
    rng = np.random.default_rng(k)
    h = torch.from_numpy(rng.uniform(0.5, 1.0, (3, k)) * np.where(rng.random((3, k)) < 0.5, -1, 1) * scale).to(dtype)
    g = np.ones(k)
    h64 = h.double().numpy()
    gd = torch.ones(k, device=dev)
    close(norms.norm(h.to(dev), gd, eps=eps), *norm_ref.norm(h64, g, eps), "norm")
    rows = norms.norm_rows(h.to(dev), gd, eps=eps)
    y = norm_ref.norm(h64, g, eps)[0]
    if np.abs(y).max() > 1e-20:     # rows below 2^-120 count as zeros
        step = np.abs(y).max(1, keepdims=True) / 127
        assert (np.abs(rows.dequantize().cpu().numpy() - y) <= 0.501 * step).all()
    d = torch.from_numpy(rng.normal(0, 1, (3, k))).float().to(dtype)
    dx, dg = norms.norm_grad(d.to(dev), h.to(dev), gd, eps=eps)
    x64, xb, g64, gb = norm_ref.norm_grad(d.double().numpy(), h64, g, eps)
    if kind == "f32" and scale < 1 or scale >= 1e18:
        ok = np.abs(x64) > 2.0**-100    # steps near the smallest exponents aside
        assert (np.abs(dx.double().cpu().numpy() - x64) <= xb + np.abs(x64) * (2.0**-8 if kind == "bf16" else U) + 2.0**-120)[ok].all()
    close(dg, g64, gb, "dgain")


U = 2.0**-23


def test_rows_of_zeros_and_without_numbers(dev):
    x = torch.randn(5, 300, device=dev)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    g = torch.ones(300, device=dev)
    y = norms.norm(x, g)
    assert (y[1] == 0).all() and y[2].isnan().all() and y[3, 9].isnan() and y[[0, 4]].isfinite().all()
    r = norms.norm_rows(x, g)
    assert r.scale[1] == 0 and r.scale[2].isnan() and r.scale[3].isnan() and r.scale[[0, 4]].isfinite().all()
    assert not r.data[1:4].any()
    d = torch.randn(5, 300, device=dev)
    dx, _ = norms.norm_grad(d, x, g)
    assert dx[[0, 1, 4]].isfinite().all() and dx[2].isnan().all()


def test_strides_shapes_and_outputs(dev):
    base = torch.randn(6, 4, 333, device=dev, dtype=torch.bfloat16)
    g = torch.rand(300, device=dev) + 0.5
    x = base[:, 1:3, 7:307]             # rows that do not flatten, at odd alignments
    r = base[:, 2:4, 3:303]
    y, h = norms.norm(x, g, residual=r)
    want, hw = norms.norm(x.contiguous(), g, residual=r.contiguous())
    assert y.shape == x.shape and torch.equal(y, want) and torch.equal(h, hw)
    out = torch.full((12, 305), 7.0, device=dev, dtype=torch.bfloat16)
    got = norms.norm(x.reshape(12, 300), g, out=out[:, 2:302])
    assert torch.equal(got, norms.norm(x.reshape(12, 300), g)) and (out[:, :2] == 7).all() and (out[:, 302:] == 7).all()
    one = norms.norm(x[0, 0], g)
    assert one.shape == (300,) and torch.equal(one, norms.norm(x[0, :1], g)[0])
    # the residual replaced by the sum
    for k in (300, 20000):
        x, r = torch.randn(2, k, device=dev), torch.randn(2, k, device=dev)
        gk = torch.rand(k, device=dev)
        want, hw = norms.norm(x, gk, residual=r)
        rows_want, _ = norms.norm_rows(x, gk, residual=r)
        r2 = r.clone()
        got, h = norms.norm(x, gk, residual=r, h_out=r)
        assert h is r and torch.equal(r, hw) and torch.equal(got, want)
        rows, _ = norms.norm_rows(x, gk, residual=r2, h_out=r2)
        assert torch.equal(rows.data, rows_want.data) and torch.equal(r2, hw)


def test_empty(dev):
    g = torch.ones(64, device=dev)
    assert norms.norm(torch.empty(0, 64, device=dev), g).shape == (0, 64)
    assert norms.norm(torch.empty(3, 0, device=dev), g[:0]).shape == (3, 0)
    r = norms.norm_rows(torch.empty(3, 0, device=dev), g[:0])
    assert r.shape == (3, 0) and not r.scale.any()
    dx, dg = norms.norm_grad(torch.empty(0, 64, device=dev), torch.empty(0, 64, device=dev), g)
    assert dx.shape == (0, 64) and not dg.any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_autograd(dev, kind):
    dtype = KINDS[kind]
    torch.manual_seed(3)
    x = torch.randn(4, 6, 200, device=dev).to(dtype).requires_grad_()
    r = torch.randn(4, 6, 200, device=dev).to(dtype).requires_grad_()
    g = (torch.rand(200, device=dev) + 0.5).requires_grad_()
    y, h = norms.norm(x, g, residual=r)
    dy, dh = torch.randn_like(y), torch.randn_like(h)
    dx, dr, dg = torch.autograd.grad((y, h), (x, r, g), (dy, dh))
    want = norms.norm_grad(dy, h.detach(), g.detach(), dh=dh)
    assert torch.equal(dx, want[0]) and torch.equal(dr, want[0]) and torch.equal(dg, want[1])
    y, h = norms.norm(x, g, residual=r)             # each output by itself
    dx, dr, dg = torch.autograd.grad(h, (x, r, g), dh)
    assert torch.equal(dx, dh) and torch.equal(dr, dh) and not dg.any()
    y, h = norms.norm(x, g, residual=r)
    dx, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(dx, norms.norm_grad(torch.ones_like(y), h.detach(), g.detach())[0])
    dx, = torch.autograd.grad(norms.norm(x, g.detach()), x, dy)
    assert torch.equal(dx, norms.norm_grad(dy, x.detach(), g.detach())[0])
    if kind == "f32":
        # against differences of the formula, in 64 bits: steps of 1e-4 in a random direction
        v = torch.randn_like(x)
        f = lambda a: (a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * g.double() * dy.double()).sum()  # noqa: E731
        x64, v64 = x.detach().double(), v.double()
        slope = ((f(x64 + 1e-4 * v64) - f(x64 - 1e-4 * v64)) / 2e-4).item()
        # third derivatives of size about 1 leave 1e-8 of it; 24 x 200 roundings the rest
        assert abs((dx.double() * v64).sum().item() - slope) <= 1e-5 * (dx.double() * v64).abs().sum().item()


def test_graph_and_streams(dev):
    x = torch.randn(37, 1000, device=dev, dtype=torch.bfloat16)
    r = torch.randn_like(x)
    g = torch.rand(1000, device=dev)
    d = torch.randn_like(x)
    side = torch.cuda.Stream()

    def step():
        y, h = norms.norm(x, g, residual=r)
        rows, _ = norms.norm_rows(x, g, residual=r)
        return (y, h, rows.data, rows.scale) + norms.norm_grad(d, h, g)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for seed in range(4):
        torch.manual_seed(seed)
        x.copy_(torch.randn(37, 1000))
        d.copy_(torch.randn(37, 1000))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    y, h = norms.norm(x, g, residual=r, stream=other.cuda_stream)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(y, step()[0]) and torch.equal(h, outs[1])


def test_refusals(dev):
    x, g = torch.randn(4, 64, device=dev), torch.ones(64, device=dev)
    bad = [lambda: norms.norm(x, g[:63]), lambda: norms.norm(x, g.half()), lambda: norms.norm(x.int(), g),
           lambda: norms.norm(x, g, residual=x[:3]), lambda: norms.norm(x, g, residual=x.half()),
           lambda: norms.norm(x, g, eps=-1.0), lambda: norms.norm(x, g, eps="0"), lambda: norms.norm(x, g.cpu()),
           lambda: norms.norm(x, g, out=x), lambda: norms.norm(x, g, h_out=torch.empty_like(x)),
           lambda: norms.norm(x, g, residual=x.clone(), h_out=x), lambda: norms.norm(x.t(), g[:4]),
           lambda: norms.norm_rows(x.clone().requires_grad_(), g), lambda: norms.norm_grad(x, x[:3], g),
           lambda: norms.norm_grad(x.clone().requires_grad_(), x, g),
           lambda: norms.norm(x.clone().requires_grad_(), g, out=torch.empty_like(x)),
           lambda: norms.norm(torch.randn(1, 64, device=dev).expand(4, 64), g)]
    for call in bad:
        with pytest.raises(HipGemmError):
            call()
