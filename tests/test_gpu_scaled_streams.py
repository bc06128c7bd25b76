"""Scaled calls with stream=: what a call copies and fills on its way is in order with its kernels, also
while torch's current stream has work of its own queued up."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import dev, say, up, weights  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu


class Busy:
    """Some 30 ms of work on torch's current stream, and a stream beside it that starts where that one
    stands now."""

    def __init__(self, dev):
        self.a = torch.randn(4096, 4096, device=dev)
        self.b = torch.empty_like(self.a)
        self.side = torch.cuda.Stream(dev)

    def __enter__(self):
        torch.cuda.synchronize()
        for _ in range(20):
            torch.mm(self.a, self.a, out=self.b)
        return self.side.cuda_stream

    def __exit__(self, *exc):
        torch.cuda.synchronize()


def test_packing_beside_a_busy_stream(dev):
    rng = np.random.default_rng(1)
    (w, s), (w2, s2) = weights(rng, 300, 200), weights(rng, 300, 200)
    w, s, w2, s2, bias = (up(v, dev) for v in (w, s, w2, s2, rng.normal(0, 1, 200).astype(np.float32)))
    want = [scaled.pack_linear(w, s, bias), scaled.pack_gated(w, s, w2, s2)]
    busy = Busy(dev)
    for _ in range(3):
        say("pack on a side stream")
        with busy as side:
            got = [scaled.pack_linear(w, s, bias, stream=side), scaled.pack_gated(w, s, w2, s2, stream=side)]
        for a, b in zip(got, want):
            assert torch.equal(a.data, b.data) and torch.equal(a.meta, b.meta)


def test_quantising_weights_beside_a_busy_stream(dev):
    w = torch.randn(700, 300, device=dev)
    want = scaled.quantize_weight(w)
    busy = Busy(dev)
    for _ in range(3):
        say("quantize_weight on a side stream")
        with busy as side:
            got = scaled.quantize_weight(w, stream=side)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rows_that_are_copied_beside_a_busy_stream(dev):
    """Rows of three dimensions whose leading two do not flatten."""
    rng = np.random.default_rng(2)
    w, s = weights(rng, 256, 192)
    L = scaled.pack_linear(up(w, dev), up(s, dev))
    G = scaled.pack_gated(up(w, dev), up(s, dev), up(w, dev), up(s, dev))
    x = torch.randn(40, 30, 256, device=dev).transpose(0, 1)
    d = torch.randn(40, 30, 192, device=dev).transpose(0, 1)
    r = scaled.quantize_rows(x)
    calls = [lambda **kw: scaled.quantize_rows(x, **kw).data, lambda **kw: scaled.linear(x, L, **kw),
             lambda **kw: scaled.gated(x, G, **kw), lambda **kw: scaled.linear_grad(d, L, **kw),
             lambda **kw: scaled.gated_grad(d, r, G, **kw)]
    want = [f() for f in calls]
    busy = Busy(dev)
    say("copied rows on a side stream")
    for _ in range(2):
        with busy as side:
            got = [f(stream=side) for f in calls]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # and their memory is not handed out while the side stream may still read it
    with busy as side:
        got = [f(stream=side) for f in calls for _ in range(3)]
        spoil = [torch.full((40 * 30 * 256,), float("nan"), device=dev) for _ in range(8)]
    assert all(torch.equal(a, b) for a, b in zip(got, [v for v in want for _ in range(3)])) and len(spoil) == 8
