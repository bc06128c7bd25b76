"""Gradients of more long rows than their statistics have workgroups (needs a gfx950 GPU), against 64 bits."""
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
