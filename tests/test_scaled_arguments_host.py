"""QuantRows hold what the kernels may read and write: sizes that the tensors do not
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

