"""Gradients of many long rows (needs a gfx950 GPU) against 64 bits, and of more than their statistics have workgroups."""
import pytest

torch = pytest.importorskip("torch")

import norm_ref
from test_gpu_norms import close
from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import norms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k", [(1500, 8200), (700, 20000)])
def test_gradients_of_many_long_rows(dev, m, k):
    say("many long rows", m, k)
    g = torch.Generator().manual_seed(m)
    h, d, e = (torch.randn(m, k, generator=g).bfloat16() for _ in range(3))
    gain = 1 + 0.3 * torch.randn(k, generator=g)
    dx, dg = norms.norm_grad(d.to(dev), h.to(dev), gain.to(dev), dh=e.to(dev))
    x64, xb, g64, gb = norm_ref.norm_grad(d.double().numpy(), h.double().numpy(), gain.double().numpy(), 1e-6, e.double().numpy())
    close(dx, x64, xb, "dx")
    close(dg, g64, gb, "dgain")


def test_more_long_rows_than_workgroups(dev):
    """2^20 workgroups: the rows behind them, and the first, are those of a call of their own (17 GB an operand)."""
    say("2^20 long rows")
    m, k, part = (1 << 20) + 70, 8200, 300
    h = torch.empty(m, k, dtype=torch.bfloat16, device=dev).normal_()
    gain = torch.rand(k, device=dev) + 0.5
    dx, _ = norms.norm_grad(h, h, gain, gain_grad=False)
    for s in (slice(0, part), slice(m - part, m)):
        assert torch.equal(dx[s], norms.norm_grad(h[s], h[s], gain, gain_grad=False)[0])
    assert dx[m - part:].any()
