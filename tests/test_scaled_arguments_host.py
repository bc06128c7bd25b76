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


def test_packing_needs_operands_apart_and_aligned():
    lib, p = _lib.load_library(), 1 << 20
    K, N = 64, 32
    ok = dict(W0=p, W1=None, ld0=N, ld1=0, s0=2 * p, s1=None, bias=3 * p, Bp=4 * p, meta=5 * p)
    pair = dict(ok, W1=6 * p, ld1=N, s1=7 * p, bias=None)
    at = {"W0": K * N - 4, "W1": K * N - 4, "s0": 4 * N - 4, "s1": 4 * N - 4, "bias": 4 * N - 4}      # last elements

    def call(a):
        return lib.vt_scaled_pack(a["W0"], a["W1"], a["ld0"], a["ld1"], a["s0"], a["s1"], a["bias"], K, N, a["Bp"], a["meta"],
                                  None)
    for base, names in ((ok, ("W0", "s0", "bias", "Bp")), (pair, ("W0", "W1", "s0", "s1", "Bp"))):
        for name in names:
            assert call(dict(base, **{name: base["meta"] - (at.get(name, 128 * 64 - 16) // 16 * 16)})) == _lib.VT_EINVAL, name
            if name[0] in "sb":
                assert call(dict(base, **{name: base[name] + 2})) == _lib.VT_EINVAL, name
                assert call(dict(base, **{name: base["Bp"]})) == _lib.VT_EINVAL, name
    assert lib.vt_scaled_linear(p, _lib.TYPE_I8, 64, 2 * p + 1, 4, 64, 3 * p, 4 * p, 32, 5 * p, _lib.TYPE_F32, 32,
                                None) == _lib.VT_EINVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="no call here reaches a device")
def test_packing_takes_operands_side_by_side():
    lib, p = _lib.load_library(), 1 << 20
    assert lib.vt_scaled_pack(p, None, 32, 0, p + 64 * 32, None, p + 64 * 32 + 128, 64, 32, 2 * p, 2 * p + 128 * 64,
                              None) == _lib.VT_ENODEV
