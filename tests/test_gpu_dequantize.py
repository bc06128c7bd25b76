"""The values of int8 rows (needs a gfx950 GPU) where a kernel of their own does not reach: scales that ask for
gradients, rows that share memory, and more rows than a launch has."""
import pytest

torch = pytest.importorskip("torch")
import torch.autograd.forward_ad as forward_ad

from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu

TYPES = [None, torch.float32, torch.float16, torch.bfloat16]


def rows(dev, m, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    data = torch.randint(-127, 128, (m, k), dtype=torch.int8, generator=g)
    return data.to(dev), torch.rand(m, generator=g).to(dev)


def plain(data, scale, k, dtype):
    return (data[:, :k].float() * scale[:, None]).to(torch.float32 if dtype is None else dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_the_scales(dev, dtype):
    data, scale = rows(dev, 6, 40)
    scale.requires_grad_()
    r = scaled.QuantRows(data, scale, k=37)
    y = r.dequantize(dtype)
    assert y.requires_grad and torch.equal(y, plain(data, scale, 37, dtype))
    dy = torch.randn(6, 37, device=dev).to(y.dtype)
    got, = torch.autograd.grad(y, scale, dy)
    want, = torch.autograd.grad(plain(data, scale, 37, dtype), scale, dy)
    assert torch.equal(got, want) and got.any()
    with torch.no_grad():
        assert torch.equal(r.dequantize(dtype), y) and not r.dequantize(dtype).requires_grad
    p = scaled.QuantRows(data, torch.nn.Parameter(scale.detach(), requires_grad=False), k=37)
    assert torch.equal(p.dequantize(dtype), y)


@pytest.mark.parametrize("dtype", TYPES)
def test_tangents_of_the_scales(dev, dtype):
    data, scale = rows(dev, 5, 16)
    with forward_ad.dual_level():
        tangent = torch.rand(5, device=dev)
        y = scaled.QuantRows(data, forward_ad.make_dual(scale, tangent)).dequantize(dtype)
        value, t = forward_ad.unpack_dual(y)
        assert torch.equal(value, plain(data, scale, 16, dtype)) and torch.equal(t, plain(data, tangent, 16, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_share_memory(dev, dtype):
    data, scale = rows(dev, 1, 300)
    s = torch.rand(9, device=dev)
    for shared in (data.expand(9, 300), data[0].as_strided((9, 200), (7, 1)), data[0].as_strided((9, 5), (2, 1))):
        r = scaled.QuantRows(shared, s)
        assert torch.equal(r.dequantize(dtype), plain(shared, s, shared.shape[1], dtype))


def test_more_rows_than_a_launch_has(dev):
    say("2^24 rows")
    for m, k in (((1 << 24) - 1, 1), (1 << 24, 1), ((1 << 24) + 3, 5)):
        data = torch.randint(-127, 128, (m, k), dtype=torch.int8, device=dev)
        scale = torch.rand(m, device=dev)
        for dtype in (torch.float32, torch.bfloat16):
            assert torch.equal(scaled.QuantRows(data, scale).dequantize(dtype), plain(data, scale, k, dtype))
