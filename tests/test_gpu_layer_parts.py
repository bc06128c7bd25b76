"""Calls whose workspaces take their rows in parts (needs a gfx950 GPU): equal, bit for bit, to calls of the parts'
rows, which run on the same kernels."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import adapters, losses, scaled

pytestmark = pytest.mark.gpu


def layer(dev, k, n):
    g = torch.Generator(device=dev)
    g.manual_seed(k + n)
    w = torch.randint(-100, 101, (k, n), dtype=torch.int8, device=dev, generator=g)
    return scaled.pack_linear(w, torch.rand(n, device=dev, generator=g) / (60 * k**0.5))


# terms of 2 or 4 bytes for each of 131072 classes: at most 2047 or 1023 rows of 512 MiB
@pytest.mark.parametrize("dtype,m,part", [(torch.bfloat16, 3000, 1536), (torch.float32, 1500, 768)])
def test_gradients_of_a_large_vocabulary(dev, dtype, m, part):
    say("parts of a loss' gradient", dtype, m)
    k, n = 64, 131072
    W = layer(dev, k, n)
    x = torch.randn(m, k, device=dev, dtype=dtype).requires_grad_()
    target = torch.randint(0, n, (m,), device=dev)
    target[::7] = -100
    g = torch.rand(m, device=dev)
    dx, = torch.autograd.grad(losses.cross_entropy(x, W, target, reduction="none"), x, g)
    for r in range(0, m, part):
        s = slice(r, r + part)
        xs = x.detach()[s].clone().requires_grad_()
        want, = torch.autograd.grad(losses.cross_entropy(xs, W, target[s], reduction="none"), xs, g[s])
        assert torch.equal(dx[s], want)


def test_logits_of_a_few_rows_of_a_very_large_vocabulary(dev):
    """64 rows of 4 million logits are a gigabyte: 33 rows at a time."""
    say("parts of logits")
    m, k, n = 64, 64, 4000000
    W = layer(dev, k, n)
    x, target = torch.randn(m, k, device=dev), torch.randint(0, n, (m,), device=dev)
    loss = losses.cross_entropy(x, W, target, reduction="none")
    for i in (0, 31, 32, 33, 34, 63):
        l = scaled.linear(x[i:i + 1], W).double()
        want = torch.logsumexp(l, 1) - l[:, target[i]]
        # the logits' own roundings, and a sum of 4e6 in steps of 4096
        assert abs(loss[i].item() - want.item()) <= 2e-6 * want.item(), i


def test_adapters_gradients(dev):
    """float32 terms of 60032 columns: 2048 rows of 512 MiB; down's and up's gradients are over all rows."""
    say("parts of adapters' gradients")
    m, k, n, rank = 5000, 64, 60000, 4
    W = layer(dev, k, n)
    x, d = torch.randn(m, k, device=dev), torch.randn(m, n, device=dev)
    down, up = torch.randn(3, rank, k, device=dev), torch.randn(3, n, rank, device=dev)
    which = torch.arange(m, device=dev, dtype=torch.int32) // 7 % 4 - 1
    dx, dd, du = adapters.adapted_grad(d, x, W, (down, up), which)
    part = 1792        # three parts of whole 256-row tiles
    dds, dus = torch.zeros_like(dd, dtype=torch.float64), torch.zeros_like(du, dtype=torch.float64)
    for r in range(0, m, part):
        s = slice(r, r + part)
        a, b, c = adapters.adapted_grad(d[s], x[s], W, (down, up), which[s])
        assert torch.equal(dx[s], a)
        dds, dus = dds + b, dus + c
    for got, want in ((dd, dds), (du, dus)):
        # sums of 5000 rows in another order: 2^-24 for each of some 100 additions
        assert (got - want).abs().max() <= 100 * 2.0**-24 * want.abs().max() * 8
