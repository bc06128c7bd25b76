"""Inputs whose gradients the scaled operators would leave out are refused, without a GPU."""
import pytest

torch = pytest.importorskip("torch")
import torch.autograd.forward_ad as forward_ad

from veritac_amd import _lib
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import scaled


def weight(pair):
    size, floats = _lib.scaled_size(100, 60, pair)
    return scaled.ScaledWeight(torch.zeros(size, dtype=torch.int8), torch.zeros(floats), 100, 60, pair)


def rows():
    return scaled.QuantRows(torch.zeros(3, 100, dtype=torch.int8), torch.ones(3))


CALLS = {"quantize_rows": (100, scaled.quantize_rows),
         "linear": (100, lambda v: scaled.linear(v, weight(False))),
         "gated": (100, lambda v: scaled.gated(v, weight(True))),
         "linear_grad": (60, lambda v: scaled.linear_grad(v, weight(False))),
         "gated_grad": (60, lambda v: scaled.gated_grad(v, rows(), weight(True)))}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    width, call = CALLS[name]
    with forward_ad.dual_level():
        v = forward_ad.make_dual(torch.zeros(3, width), torch.ones(3, width))
        with pytest.raises(HipGemmError, match="forward-mode"):
            call(v)
        with pytest.raises(HipGemmError, match="no CPU path"):      # a level without a tangent is an ordinary call
            call(torch.zeros(3, width))


@pytest.mark.parametrize("name", ["quantize_rows", "linear_grad", "gated_grad"])
def test_gradients_are_not_left_out(name):
    width, call = CALLS[name]
    v = torch.zeros(3, width, requires_grad=True)
    for leaf in (v, v * 2):
        with pytest.raises(HipGemmError, match="%s passes no gradient" % name):
            call(leaf)
        with pytest.raises(HipGemmError, match="no CPU path"):
            call(leaf.detach())
        with torch.no_grad(), pytest.raises(HipGemmError, match="no CPU path"):
            call(leaf)
