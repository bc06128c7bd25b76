"""Norms of rows at the smallest float32 values (needs a gfx950 GPU), where squares vanish and a mean of few of them
leaves float32's range even after they were scaled, against 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import norm_ref
import scaled_ref as ref
from test_gpu_norms import close
from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import norms

pytestmark = pytest.mark.gpu

LEAST = 2.0**-149       # of float32


def smallest(m, k, kind):
    """Rows of whole multiples of the least value: one alone, few, or many small ones."""
    rng = np.random.default_rng(k)
    h = np.zeros((m, k))
    if kind == "one":
        h[np.arange(m), rng.integers(0, k, m)] = LEAST * np.arange(1, m + 1)
    elif kind == "few":
        for i in range(m):
            h[i, rng.integers(0, k, 3)] = LEAST * rng.integers(-50, 51, 3)
        h[:, 0] = LEAST * 7
    else:
        h[:] = LEAST * rng.integers(-2000, 2001, (m, k))
    return h


@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-30, 1e-22])
@pytest.mark.parametrize("kind", ["one", "few", "many"])
@pytest.mark.parametrize("k", [1, 300, 4096, 5000, 16384, 20000])
def test_the_smallest_rows(dev, k, kind, eps):
    """eps on both sides of 2^-80 (8.3e-25) and below 2^-60."""
    say("smallest rows", k, kind, eps)
    eps = float(np.float32(eps))
    h64 = smallest(5, k, kind)
    h, gain = torch.from_numpy(h64).float().to(dev), torch.ones(k, device=dev)
    y, bound = norm_ref.norm(h64, np.ones(k), eps)
    # outputs among the denormals themselves are rounded to steps of the least value
    close(norms.norm(h, gain, eps=eps), y, bound + LEAST, "norm")
    if eps < 1e-40:
        # z in the row's own scale is the row: whole multiples of the least value over the largest
        rows = norms.norm_rows(h, gain, eps=eps)
        step = np.abs(y).max(1, keepdims=True) / 127
        assert (np.abs(rows.dequantize().double().cpu().numpy() - y) <= 0.501 * step).all()
    rng = np.random.default_rng(k + 1)
    d64 = rng.normal(0, 1, (5, k)).astype(np.float32).astype(np.float64) * 2.0**-70
    dx, dg = norms.norm_grad(torch.from_numpy(d64).float().to(dev), h, gain, eps=eps)
    x64, xb, g64, gb = norm_ref.norm_grad(d64, h64, np.ones(k), eps)
    ref.check(dx, x64, xb + LEAST, dx.dtype, "dx")
    # products of d and a denormal n: steps of the least value, one a row and one a sum
    ref.check(dg, g64, gb + 16 * LEAST, dg.dtype, "dgain")
