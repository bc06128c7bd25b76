"""What feed-forward blocks and adapters refuse, without a GPU: wrong arguments are HipGemmErrors before anything runs."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from veritac_amd import _lib
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import adapters, feed_forward, scaled

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


def test_missing_rows_are_refused_where_nothing_is_put_out():
    """u and h are made from the rows also without columns of the outputs or of dx."""
    lib, a = _lib.load_library(), [(1 + i) << 30 for i in range(12)]
    f32, i8 = _lib.TYPE_F32, _lib.TYPE_I8

    def adapted(x, kind, t):
        return lib.vt_adapted_linear(x, kind, 64, t, 4, 64, a[1], a[2], 0, a[3], 8, 2, 1.0, a[4], a[5], a[6], f32, 1, None)

    def grad(dy):
        return lib.vt_adapted_grad(dy, f32, 32, None, 1, 4, 0, a[1], a[2], 32, None, a[3], 8, 2, 1.0, a[4], a[5], a[6], a[7], 1, None, a[8], None)
    for rc in (adapted(None, f32, None), adapted(a[0], i8, None), adapted(None, i8, a[7]), grad(None)):
        assert rc == _lib.VT_EINVAL, (rc, _lib.last_error())


def test_outputs_are_not_left_out():
    lib, a = _lib.load_library(), [(1 + i) << 30 for i in range(12)]
    rc = lib.vt_adapted_linear(a[0], _lib.TYPE_F32, 64, None, 4, 64, a[1], a[2], 32, a[3], 8, 2, 1.0, a[4], a[5], None, _lib.TYPE_F32, 32, None)
    assert rc == _lib.VT_EINVAL, (rc, _lib.last_error())


FITS = dict(dtype=torch.float16, count=2, rank=4, k=64, n=96, scaling=0.5)


def held(**kw):
    size = _lib.adapter_size(64, 96, 4, 2, _lib.TYPE_F16)
    return adapters.Adapters(torch.zeros(size, dtype=torch.uint8), **{**FITS, **kw})


@pytest.mark.parametrize("kw", [dict(count="2"), dict(count=2.0), dict(count=None), dict(rank=4.0), dict(rank=True), dict(k="64"), dict(n=None),
                                dict(n=1 << 70), dict(n=(1 << 64) + 96), dict(k=-64), dict(rank=0), dict(count=0), dict(dtype=torch.int8), dict(dtype="f16")], ids=str)
def test_adapters_are_of_whole_sizes(kw):
    assert held().count == 2
    with pytest.raises(HipGemmError):
        held(**kw)


@pytest.mark.parametrize("scaling", [1e39, -1e39, 10**400, float("inf"), float("nan"), "1", True, None],
                         ids=["above", "below", "huge", "inf", "nan", "text", "truth", "none"])
def test_scalings_are_float32_numbers(scaling):
    assert held(scaling=-3e38).scaling == -3e38
    with pytest.raises(HipGemmError):
        held(scaling=scaling)
    with pytest.raises(HipGemmError):
        feed_forward.FeedForward(weight(D, N, True), weight(N, D, False), adapters=(torch.zeros(2, 4, N), torch.zeros(2, D, 4), scaling))
