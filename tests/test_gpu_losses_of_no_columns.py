"""The loss of many rows without columns (needs a gfx950 GPU): their logits are the biases."""
import pytest

torch = pytest.importorskip("torch")

import scaled_ref as ref
from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import losses, scaled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(65536, 5), (140001, 70)])
def test_rows_without_columns(dev, m, n):
    say("no columns", m, n)
    bias = torch.randn(n, device=dev)
    W = scaled.pack_linear(torch.zeros(0, n, dtype=torch.int8, device=dev), torch.ones(n, device=dev), bias)
    target = torch.arange(m, device=dev) % (n + 1)
    target[target == n] = -100
    x = torch.zeros(m, 0, device=dev, requires_grad=True)
    loss = losses.cross_entropy(x, W, target, reduction="none")
    b = bias.double()
    want = torch.where(target >= 0, torch.logsumexp(b, 0) - b[target.clamp_min(0)], 0.0)
    # exponentials of |l - m| <= 8, the sum's and the logarithm's roundings, two subtractions
    assert (loss.double() - want).abs().max() <= 64 * ref.U32
    assert torch.autograd.grad(loss.sum(), x)[0].shape == (m, 0)
    mean = losses.cross_entropy(x.detach(), W, target)
    assert abs(mean.item() - (want.sum() / (target >= 0).sum()).item()) <= 64 * ref.U32
