"""Scaled operators over rows without values (K = 0): the bias or zeros, for every kind of rows."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import dev, packed, packed_pair  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 3, 70])
def test_int8_rows_without_values(dev, m):
    s, bias = np.ones(48, np.float32), np.arange(48, dtype=np.float32)
    none = np.zeros((0, 48), np.int8)
    L, G = packed(dev, none, s, bias), packed_pair(dev, none, s, none, s)
    x = torch.empty(m, 0, device=dev)
    raw = scaled.QuantRows(torch.empty(m, 0, dtype=torch.int8, device=dev), torch.ones(m, device=dev))
    for r in (scaled.quantize_rows(x), raw):
        y = scaled.linear(r, L, out_dtype=torch.float32)
        assert torch.equal(y, torch.arange(48, device=dev).float().expand(m, 48))
        assert not scaled.gated(r, G, out_dtype=torch.float32).any()
        assert scaled.gated_grad(torch.ones(m, 48, device=dev), r, G).shape == (m, 0)


def test_autograd_over_rows_without_values(dev):
    s, none = np.ones(48, np.float32), np.zeros((0, 48), np.int8)
    L, G = packed(dev, none, s), packed_pair(dev, none, s, none, s)
    for shape in ((3, 0), (2, 3, 0), (0,)):
        for f in (lambda v: scaled.linear(v, L), lambda v: scaled.gated(v, G)):
            x = torch.empty(shape, device=dev, requires_grad=True)
            y = f(x)
            assert y.shape == (*shape[:-1], 48) and not y.any()
            y.sum().backward()
            assert x.grad.shape == shape
