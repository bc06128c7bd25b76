"""What feed-forward blocks and adapters refuse, without a GPU: wrong arguments are HipGemmErrors before anything runs."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from veritac_amd import _lib
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import feed_forward, scaled

D, N = 64, 96


def weight(k, n, pair):
    size, floats = _lib.scaled_size(k, n, pair)
    return scaled.ScaledWeight(torch.zeros(size, dtype=torch.int8), torch.zeros(floats), k, n, pair)


def block(**kw):
    return feed_forward.FeedForward(weight(D, N, True), weight(N, D, False), **kw)


ROWS = {"int8 rows": lambda: scaled.QuantRows(torch.zeros(3, D, dtype=torch.int8), torch.ones(3)), "none": lambda: None,
        "list": lambda: [1.0] * D, "array": lambda: np.zeros((3, D), np.float32), "integers": lambda: torch.zeros(3, D, dtype=torch.int32)}


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("rows", ROWS)
def test_a_block_refuses_rows_that_are_no_floating_tensor(rows, normed):
    with pytest.raises(HipGemmError):
        block(**(dict(norm=torch.ones(D)) if normed else {}))(ROWS[rows]())
