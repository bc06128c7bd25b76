"""Gradients of rows of one type through outputs of another: they have the rows' bits and range."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import DTYPES, IDS, dev, packed, packed_pair, weights  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("out_dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_the_gradient_has_the_rows_type(dev, dtype, out_dtype, op):
    rng = np.random.default_rng(4)
    (w, s), (w2, s2) = weights(rng, 96, 130), weights(rng, 96, 130)
    s, s2 = s * np.float32(20), s2 * np.float32(20)
    x = torch.randn(9, 96, device=dev, dtype=dtype)
    # the last rows' gradients leave float16's range, dy itself (at most 12000 x 4) does not
    d = torch.randn(9, 130, device=dev).clamp(-4, 4) * torch.tensor([1.0] * 7 + [1e4, 1.2e4], device=dev)[:, None]
    d = d.to(out_dtype)
    leaf = x.clone().requires_grad_(True)
    wide = torch.promote_types(dtype, out_dtype)
    if op == "linear":
        W = packed(dev, w, s)
        scaled.linear(leaf, W, out_dtype=out_dtype).backward(d)
        want = scaled.linear_grad(d.to(wide), W)
    else:
        W = packed_pair(dev, w, s, w2, s2)
        scaled.gated(leaf, W, out_dtype=out_dtype).backward(d)
        want = scaled.gated_grad(d.to(wide), scaled.quantize_rows(x), W)
    assert leaf.grad.dtype == dtype and torch.equal(leaf.grad, want.to(dtype))
    if dtype != torch.float16:
        assert torch.isfinite(leaf.grad).all()
        assert leaf.grad.abs().max() > 65504
