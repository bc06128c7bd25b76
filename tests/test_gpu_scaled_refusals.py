"""Every mismatch of a scaled call is a HipGemmError, and nothing else."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import dev, packed, packed_pair, up, weights  # noqa: F401
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu


def test_mismatches_raise_hip_gemm_error(dev):
    rng = np.random.default_rng(1)
    w, s = weights(rng, 96, 40)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w, s)
    wd, sd = up(w, dev), up(s, dev)
    x, d = torch.zeros(3, 96, device=dev), torch.zeros(3, 40, device=dev)
    r = scaled.quantize_rows(x)
    leaf = torch.zeros(3, 96, device=dev, requires_grad=True)
    strided = torch.zeros(3, 80, device=dev)[:, ::2]
    calls = [
        (lambda: scaled.linear(x[:, :95], W), "95 columns"), (lambda: scaled.linear(x, G), "pack_linear"),
        (lambda: scaled.gated(x, W), "pack_gated"), (lambda: scaled.linear(x, None), "pack_linear"),
        (lambda: scaled.linear(x.cpu(), W), "no CPU path"), (lambda: scaled.linear(x.double(), W), "float32"),
        (lambda: scaled.linear([1.0], W), "torch tensor"), (lambda: scaled.linear(np.zeros((3, 96)), W), "torch tensor"),
        (lambda: scaled.linear(np.zeros((3, 96)), W, stream=0), "torch tensor"),
        (lambda: scaled.linear(x, W, out_dtype=torch.int32), "type must be"),
        (lambda: scaled.linear(x, W, out_dtype="float32"), "type must be"),
        (lambda: scaled.linear(r, W), "need out_dtype"),
        (lambda: scaled.linear(x.t().contiguous().t(), W), "unit stride"),
        (lambda: scaled.linear(x[:1].expand(3, 96), W), "overlapping rows"),
        (lambda: scaled.linear(x, W, out=torch.zeros(3, 41, device=dev)), "out must be"),
        (lambda: scaled.linear(x, W, out=strided), "unit stride"),
        (lambda: scaled.linear(x, W, out=torch.zeros(1, 40, device=dev).expand(3, 40)), "do not overlap"),
        (lambda: scaled.linear(x, W, out=torch.zeros(3, 40, device=dev), out_dtype=torch.float16), "out must be"),
        (lambda: scaled.linear(x, W, out=torch.zeros(3, 40)), "out must be"),
        (lambda: scaled.linear(x, W, out=[0.0] * 120), "out must be"), (lambda: scaled.gated(r, G, out=7), "out must be"),
        (lambda: scaled.linear_grad(d, W, out="x"), "out must be"),
        (lambda: scaled.gated_grad(d, r, G, out=np.zeros((3, 96))), "out must be"),
        (lambda: scaled.linear(x, W, out=x.view(-1)[:120].view(3, 40)), "overlaps"),
        (lambda: scaled.linear_grad(d[:, :39], W), "39 columns"), (lambda: scaled.gated_grad(d[:2], r, G), "dh is 2 x 40"),
        (lambda: scaled.gated_grad(d, x, G), "QuantRows"), (lambda: scaled.gated(x, G, act="relu"), "act must be"),
        (lambda: scaled.gated(x, G, act=["silu"]), "act must be"),
        (lambda: scaled.linear(leaf, W, out=d), "neither out nor stream"),
        (lambda: scaled.pack_linear(wd, sd[:39]), "scale of w"), (lambda: scaled.pack_linear(wd, sd, sd.double()), "bias"),
        (lambda: scaled.pack_linear(wd, sd.cpu()), "scale of w is on"), (lambda: scaled.pack_linear(wd.t(), sd), "unit stride"),
        (lambda: scaled.pack_linear(wd[:1].expand(96, 40), sd), "pitch"),
        (lambda: scaled.pack_gated(wd, sd, wd[:95], sd), "w_up has shape"),
        (lambda: scaled.pack_linear(None, sd), "int8"), (lambda: scaled.quantize_weight(7), "floating"),
        (lambda: scaled.quantize_weight(wd), "float32"), (lambda: scaled.quantize_rows(None), "torch tensor")]
    for call, what in calls:
        with pytest.raises(HipGemmError, match=what):
            call()
    assert torch.equal(scaled.linear(x, W), torch.zeros(3, 40, device=dev))
