"""QuantRows and ScaledWeight hold what the kernels may read and write: sizes that the tensors do not
have are refused where the object is made, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from veritac_amd import _lib
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import scaled


def rows(m=100, width=128, **kw):
    return scaled.QuantRows(torch.zeros(m, width, dtype=torch.int8), torch.ones(m), **kw)


@pytest.mark.parametrize("kw,what", [
    (dict(shape=(2, 128)), "100 rows"),                  # fewer rows than there are: outputs too small
    (dict(shape=(101, 128)), "100 rows"), (dict(shape=(5, 10, 128)), "100 rows"), (dict(shape=(100, 64)), "100 rows"),
    (dict(shape=()), "100 rows"), (dict(shape=(-10, -10, 128)), "100 rows"), (dict(shape=(100.0, 128)), "100 rows"),
    (dict(k=129), "width"), (dict(k=-1), "width"), (dict(k=64.0), "width"), (dict(k=True), "width"),
    (dict(k=64, shape=(100, 128)), "100 rows"),
], ids=str)
def test_rows_of_other_sizes_are_refused(kw, what):
    with pytest.raises(HipGemmError, match=what):
        rows(**kw)


def test_padded_rows_hold_their_padding():
    for k in (1, 100, 128, 1000, 1024, 1025):
        pitch = _lib.quant_pitch(k)
        assert rows(3, pitch, k=k, padded=True).k == k
        with pytest.raises(HipGemmError, match="padded rows"):
            rows(3, pitch - 1, k=min(k, pitch - 1), padded=True)
    with pytest.raises(HipGemmError, match="padded rows"):      # columns of a wider matrix: the last row ends with it
        scaled.QuantRows(torch.zeros(5, 128, dtype=torch.int8)[:, 16:], torch.ones(5), padded=True)


def test_rows_of_any_leading_shape():
    assert rows(6, 128, k=100).shape == (6, 100)
    r = rows(6, 128, k=100, shape=[1, 2, 3, 100])
    assert r.shape == (1, 2, 3, 100) and r.dequantize().shape == (1, 2, 3, 100)
    assert rows(1, 128, shape=(128,)).dequantize().shape == (128,)
    assert rows(0, 128, shape=(0, 7, 128)).dequantize().shape == (0, 7, 128)
    assert rows(3, 0).shape == (3, 0)
    assert rows(3, 0, padded=True).k == 0


def weight(k=100, n=60, pair=False, data=None, meta=None):
    size, floats = _lib.scaled_size(100, 60, pair)
    return scaled.ScaledWeight(torch.zeros(size, dtype=torch.int8) if data is None else data,
                               torch.zeros(floats) if meta is None else meta, k, n, pair)


def test_packed_weights_have_their_size():
    size, floats = _lib.scaled_size(100, 60, False)
    assert weight().n == 60 and weight(pair=True).pair
    for call, what in ((lambda: weight(k=200), "data"), (lambda: weight(n=65), "data"),
                       (lambda: weight(data=torch.zeros(size - 1, dtype=torch.int8)), "data"),
                       (lambda: weight(data=torch.zeros(size)), "data"),
                       (lambda: weight(data=torch.zeros(2 * size, dtype=torch.int8)[::2]), "data"),
                       (lambda: weight(data=[0] * size), "data"),
                       (lambda: weight(meta=torch.zeros(floats - 1)), "meta"),
                       (lambda: weight(meta=torch.zeros(floats, dtype=torch.float64)), "meta"),
                       (lambda: weight(meta=torch.zeros(2 * floats)[::2]), "meta"),
                       (lambda: weight(k=-1), "K")):
        with pytest.raises(HipGemmError, match=what):
            call()
