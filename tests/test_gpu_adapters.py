"""Low-rank adapters beside int8 linear layers and their gradients (needs a gfx950 GPU) against 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import scaled_ref as ref
from adapter_ref import CASES, Adapted
from test_gpu_scaled import dev, packed, rows, say, up as to, weights  # noqa: F401
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import adapters, scaled

pytestmark = pytest.mark.gpu

KINDS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# two halves of u: bfloat16 rounds by 2^-8, and what is left by 2^-8 again
UNIT = {"f32": 0.0, "f16": 2.0**-22, "bf16": 2.0**-16}


class Case:
    def __init__(self, m, k, n, rank, count, kind, dev, order="mixed"):
        rng = np.random.default_rng(m * 131 + k * 17 + n + rank)
        dtype = self.dtype = KINDS[kind]
        self.kind = kind
        x, x32 = rows(rng, m, k, dtype)
        w, s = weights(rng, k, n, -128)
        bias = rng.normal(0, 0.3, n).astype(np.float32) if (m + n) % 2 else None
        down = torch.from_numpy(rng.normal(0, 1 / max(k, 1)**0.5, (count, rank, k))).to(dtype)
        up = torch.from_numpy(rng.normal(0, 0.3 / rank**0.5, (count, n, rank))).to(dtype)
        which = rng.integers(-1, count, m) if order == "mixed" else np.sort(rng.integers(-1, count, m))
        self.q, self.t = ref.quantize(x32)
        self.scaling = 0.75
        args = (w, s, bias, down.double().numpy(), up.double().numpy(), self.scaling, which, UNIT[kind])
        self.ref = Adapted(x32, self.q, self.t, *args)
        self.ref8 = Adapted(self.q.astype(np.float64) * self.t[:, None].astype(np.float64), self.q, self.t, *args)
        d = torch.from_numpy(rng.normal(0, 1e-2, (m, n))).to(dtype)
        self.d64 = d.double().numpy()
        self.x, self.d, self.down, self.up = x.to(dev), d.to(dev), down.to(dev), up.to(dev)
        self.W, self.which = packed(dev, w, s, bias), to(which.astype(np.int32), dev)
        self.triple = self.down, self.up, self.scaling


def close(got, want, what):
    ref.check(got, *want, got.dtype, what)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n,rank,count", CASES)
def test_adapted_and_its_gradients(dev, m, k, n, rank, count, kind):
    say("adapted", m, k, n, rank, count, kind)
    c = Case(m, k, n, rank, count, kind, dev, "sorted" if (m + rank) % 2 else "mixed")
    A = adapters.pack_adapters(c.down, c.up, scaling=c.scaling)
    y = adapters.adapted(c.x, c.W, A, c.which)
    assert y.dtype == c.dtype
    close(y, c.ref.forward(), "y")
    assert torch.equal(adapters.adapted(c.x, c.W, c.triple, c.which), y)
    r = scaled.QuantRows(to(c.q, dev), to(c.t, dev))
    close(adapters.adapted(r, c.W, A, c.which), c.ref8.forward(), "y of int8 rows")
    got = adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)
    for g, want, name in zip(got, c.ref.grad(c.d64, kind == "bf16"), ("dx", "ddown", "dup")):
        assert g.dtype == c.dtype
        close(g, want, name)
    for a, b in zip(got, adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 40, 100, 300])
def test_no_index_and_no_adapter(dev, m, kind):
    c = Case(m, 256, 512, 16, 1, kind, dev)
    all0 = torch.zeros(m, dtype=torch.int32, device=dev)
    none = torch.full((m,), -7, dtype=torch.int32, device=dev)
    y = adapters.adapted(c.x, c.W, c.triple)
    assert torch.equal(y, adapters.adapted(c.x, c.W, c.triple, all0))
    one = adapters.adapted(c.x, c.W, (c.down[0], c.up[0], c.scaling))
    assert torch.equal(one, y)
    assert torch.equal(adapters.adapted(c.x, c.W, c.triple, none), scaled.linear(c.x, c.W))
    for a, b in zip(adapters.adapted_grad(c.d, c.x, c.W, c.triple), adapters.adapted_grad(c.d, c.x, c.W, c.triple, all0)):
        assert torch.equal(a, b)
    dx, dd, du = adapters.adapted_grad(c.d, c.x, c.W, c.triple, none)
    assert not dd.any() and not du.any() and torch.equal(dx, scaled.linear_grad(c.d, c.W))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [6, 40, 90, 300])
def test_a_row_is_not_touched_by_others(dev, m, kind):
    """Adapters that hold NaN or infinity, indices beyond the last and rows without numbers stay with their rows."""
    k, n = 512, 640
    c = Case(m, k, n, 16, 4, kind, dev)
    which = torch.arange(m, device=dev, dtype=torch.int32) % 4
    good = adapters.adapted(c.x, c.W, c.triple, which)
    dgood = adapters.adapted_grad(c.d, c.x, c.W, c.triple, which)
    down, up = c.down.clone(), c.up.clone()
    down[1] = float("nan")
    up[2] = float("inf")
    x = c.x.clone()
    x[4, 3] = float("nan")
    which[3] = 4
    which[5] = 2**31 - 1
    y = adapters.adapted(x, c.W, (down, up, c.scaling), which)
    bad = (which == 1) | (which == 2) | (which >= 4)
    bad[4] = True
    assert y[which == 1].isnan().all() and not y[which == 2].isfinite().any() and y[which >= 4].isnan().all() and y[4].isnan().all()
    assert torch.equal(y[~bad], good[~bad])
    dx, dd, du = adapters.adapted_grad(c.d, c.x, c.W, (down, up, c.scaling), which)
    ok = (which == 0) | (which == 3)
    assert torch.equal(dx[ok], dgood[0][ok]) and dx[which >= 4].isnan().all()
    assert dd[[0, 3]].isfinite().all() and du[[0, 3]].isfinite().all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,rank", [(65, 1, 3), (70, 7, 16), (129, 130, 20), (100, 999, 64), (333, 4100, 64), (66, 14336, 128),
                                      (3100, 520, 64), (1600, 264, 128)])
def test_rounded_beside_u(dev, m, k, rank, kind):
    """The rows that u's kernel rounds are linear's: with adapters that add nothing, the outputs are the same."""
    say("rounded beside u", m, k, rank, kind)
    g = torch.Generator().manual_seed(m + k)
    dtype, n, count = KINDS[kind], 40, 3
    x = torch.randn(m, k + 3, generator=g).mul(torch.rand(m, 1, generator=g) * 4).to(dtype)
    x[1], x[2, 0], x[3, k - 1], x[4] = 0, float("nan"), float("-inf"), torch.finfo(dtype).tiny / 4
    x[5, : k - 1] = 0
    rng = np.random.default_rng(k)
    W = packed(dev, *weights(rng, k, n, -128), None)
    down = torch.randn(count, rank, k, generator=g).to(dtype).to(dev)
    up = torch.zeros(count, n, rank, dtype=dtype, device=dev)
    which = torch.randint(-1, count, (m,), generator=g, dtype=torch.int32)
    which[16:32] = -1
    for at in (0, 1, 3):
        rows = x.to(dev)[:, at:at + k]
        want = scaled.linear(rows, W)
        for w in (which.to(dev), None):
            torch.testing.assert_close(adapters.adapted(rows, W, (down, up), w), want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("m", [30, 200])
def test_u_beyond_float16(dev, m):
    """float16 adapters whose u leaves float16's range, at either end."""
    c = Case(m, 256, 320, 20, 2, "f16", dev)
    for f in (3e4, 2.0**-13):
        down, up = (c.down.float() * f).half(), (c.up.float() / f).half()
        x = c.x.float().clamp(-1, 1).half()
        q, t = ref.quantize(x.float().cpu().numpy())
        q0, t0, w, s, bias = c.ref.base
        R = Adapted(x.double().cpu().numpy(), q, t, w, s, bias, down.double().cpu().numpy(), up.double().cpu().numpy(), 8.0,
                    c.ref.which, UNIT["f16"])
        close(adapters.adapted(x, c.W, (down, up, 8.0), c.which), R.forward(), "y at %g" % f)
        for g, want, name in zip(adapters.adapted_grad(c.d, x, c.W, (down, up, 8.0), c.which), R.grad(c.d64, False),
                                 ("dx", "ddown", "dup")):
            close(g, want, name)


def test_strides_shapes_and_outputs(dev):
    c = Case(24, 200, 304, 8, 3, "bf16", dev)
    want = adapters.adapted(c.x, c.W, c.triple, c.which)
    x3 = torch.zeros(4, 7, 203, device=dev, dtype=torch.bfloat16)[:, :6, 2:202]
    x3.copy_(c.x.reshape(4, 6, 200))
    got = adapters.adapted(x3, c.W, c.triple, c.which.reshape(4, 6))
    assert got.shape == (4, 6, 304) and torch.equal(got.reshape(24, 304), want)
    out = torch.full((24, 311), 7.0, device=dev, dtype=torch.bfloat16)
    assert torch.equal(adapters.adapted(c.x, c.W, c.triple, c.which, out=out[:, 3:307]), want)
    assert (out[:, :3] == 7).all() and (out[:, 307:] == 7).all()
    two = torch.stack((c.which, c.which), 1)[:, 0]
    assert torch.equal(adapters.adapted(c.x, c.W, (c.down.transpose(1, 2).contiguous().transpose(1, 2), c.up, c.scaling), two), want)
    one = adapters.adapted(c.x[7], c.W, c.triple, c.which[7])
    assert one.shape == (304,)
    close(one.reshape(1, -1), [a[7:8] for a in c.ref.forward()], "a row by itself")
    assert adapters.adapted(c.x[:0], c.W, c.triple, c.which[:0]).shape == (0, 304)
    dx, dd, du = adapters.adapted_grad(c.d[:0], c.x[:0], c.W, c.triple, c.which[:0])
    assert dx.shape == (0, 200) and not dd.any() and not du.any()
    W0 = scaled.pack_linear(torch.zeros(200, 0, dtype=torch.int8, device=dev), torch.zeros(0, device=dev))
    assert adapters.adapted(c.x, W0, (c.down, c.up[:, :0]), c.which).shape == (24, 0)
    dx, dd, du = adapters.adapted_grad(c.d[:, :0], c.x, W0, (c.down, c.up[:, :0]), c.which)
    assert not dx.any() and not dd.any() and du.shape == (3, 0, 8)
    d3 = torch.zeros(4, 7, 304, device=dev, dtype=torch.bfloat16)[:, :6]
    d3.copy_(c.d.reshape(4, 6, 304))
    for a, b in zip(adapters.adapted_grad(d3, x3, c.W, c.triple, c.which.reshape(4, 6)),
                    adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)):
        assert torch.equal(a.reshape(b.shape), b)


@pytest.mark.parametrize("kind", KINDS)
def test_autograd(dev, kind):
    c = Case(90, 128, 200, 6, 3, kind, dev)
    x, down, up = (t.clone().requires_grad_() for t in (c.x, c.down, c.up))
    y = adapters.adapted(x, c.W, (down, up, c.scaling), c.which)
    want = adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)
    for a, b in zip(torch.autograd.grad(y, (x, down, up), c.d), want):
        assert torch.equal(a, b)
    y = adapters.adapted(c.x, c.W, (down, up, c.scaling), c.which)
    for a, b in zip(torch.autograd.grad(y, (down, up), c.d), want[1:]):
        assert torch.equal(a, b)
    y = adapters.adapted(x, c.W, (c.down[0], c.up[0]))
    assert torch.equal(torch.autograd.grad(y, x, c.d)[0], adapters.adapted_grad(c.d, c.x, c.W, (c.down[0], c.up[0]))[0])
    with torch.no_grad():
        down += 1       # after the forward pass that saved it
        y = adapters.adapted(c.x, c.W, (down, up, c.scaling), c.which)
        assert torch.equal(y, adapters.adapted(c.x, c.W, (down.detach().clone(), up.detach(), c.scaling), c.which))
    y = adapters.adapted(x, c.W, (down, up, c.scaling), c.which)
    with torch.no_grad():
        up += 1
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, c.d)


def test_gradient_against_differences(dev):
    """Of the float64 formula along directions, in float32."""
    c = Case(50, 96, 130, 4, 2, "f32", dev)
    rng = np.random.default_rng(3)
    R = c.ref
    vx, vd, vu = (rng.normal(0, 1, a.shape) for a in (R.x, R.down, R.up))
    W64 = R.w * R.s

    def f(e):
        x, down, up = R.x + e * vx, R.down + e * vd, R.up + e * vu
        y = x @ W64     # straight through the rounding
        for a in range(2):
            i = R.rows(a)
            y[i] += R.c * (x[i] @ down[a].T) @ up[a].T
        return (y * c.d64).sum()
    got = adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)
    terms = [(g.double().cpu().numpy() * v) for g, v in zip(got, (vx, vd, vu))]
    slope = (f(1e-4) - f(-1e-4)) / 2e-4
    # f is cubic: h^2 of its third derivative, and 32-bit gradients
    assert abs(sum(t.sum() for t in terms) - slope) <= 1e-5 * sum(np.abs(t).sum() for t in terms)


def test_captured_and_on_streams(dev):
    """Two decode batches captured on streams of their own, replayed in turn with other rows and indices."""
    steps = []
    for m, k, n in ((12, 4096, 700), (100, 512, 1000)):
        c = Case(m, k, n, 16, 5, "bf16", dev)
        A = adapters.pack_adapters(c.down, c.up, scaling=c.scaling)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            adapters.adapted(c.x, c.W, A, c.which)
            adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = adapters.adapted(c.x, c.W, A, c.which)
            grads = adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)
        steps.append((c, A, graph, (y, *grads)))
    for seed in range(3):
        torch.manual_seed(seed)
        for c, A, graph, outs in steps:
            c.x.copy_(torch.randn(c.x.shape))
            c.which.copy_(torch.randint(-1, 5, c.which.shape))
            graph.replay()
        torch.cuda.synchronize()
        for c, A, graph, outs in steps:
            want = (adapters.adapted(c.x, c.W, A, c.which), *adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which))
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
    c, A, _, _ = steps[0]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    y = adapters.adapted(c.x, c.W, c.triple, c.which, stream=other.cuda_stream)
    grads = adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which, stream=other.cuda_stream)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(y, adapters.adapted(c.x, c.W, A, c.which))
    for a, b in zip(grads, adapters.adapted_grad(c.d, c.x, c.W, c.triple, c.which)):
        assert torch.equal(a, b)


def test_refusals(dev):
    c = Case(6, 64, 96, 4, 2, "bf16", dev)
    A = adapters.pack_adapters(c.down, c.up)
    r = scaled.quantize_rows(c.x)
    w64 = c.which.long()
    bad = [lambda: adapters.adapted(c.x.half(), c.W, A, c.which), lambda: adapters.adapted(c.x, c.W, A, w64),
           lambda: adapters.adapted(c.x, c.W, A, c.which[:5]), lambda: adapters.adapted(c.x, c.W, A, c.which.cpu()),
           lambda: adapters.adapted(c.x, c.W, c.down, c.which), lambda: adapters.adapted(c.x[:, :63], c.W, A, c.which),
           lambda: adapters.adapted(c.x, c.W, (c.down, c.up[:, :95]), c.which),
           lambda: adapters.adapted(c.x, c.W, (c.down, c.up[..., :3]), c.which),
           lambda: adapters.adapted(c.x, c.W, (c.down, c.up.half()), c.which),
           lambda: adapters.adapted(c.x, c.W, (c.down[:0], c.up[:0]), c.which),
           lambda: adapters.adapted(c.x, c.W, (c.down, c.up, float("nan")), c.which),
           lambda: adapters.adapted(c.x.clone().requires_grad_(), c.W, A, c.which),
           lambda: adapters.adapted(r, c.W, (c.down.clone().requires_grad_(), c.up), c.which),
           lambda: adapters.adapted(c.x, c.W, A, c.which, out=torch.empty(6, 96, device=dev)),
           lambda: adapters.adapted(c.x, c.W, A, c.which, out=c.x),
           lambda: adapters.pack_adapters(c.down.clone().requires_grad_(), c.up),
           lambda: adapters.pack_adapters(torch.zeros(2, 129, 64, device=dev), torch.zeros(2, 96, 129, device=dev)),
           lambda: adapters.adapted_grad(c.d, c.x[:5], c.W, c.triple, c.which),
           lambda: adapters.adapted_grad(c.d, c.x, c.W, A, c.which),
           lambda: adapters.adapted_grad(c.d.float(), c.x, c.W, c.triple, c.which),
           lambda: adapters.adapted_grad(c.d.clone().requires_grad_(), c.x, c.W, c.triple, c.which)]
    for i, call in enumerate(bad):
        with pytest.raises(HipGemmError):
            call()
            print("call", i)
