"""Scaled int8 operators without a GPU: sizes and layouts the library reports, every refusal of the C
entries before a device call, and the Python layer's checks."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from veritac_amd import _lib
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import feed_forward, scaled

F32, F16, BF16, I8, I8P = _lib.TYPE_F32, _lib.TYPE_F16, _lib.TYPE_BF16, _lib.TYPE_I8, _lib.TYPE_I8_PADDED


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def test_pitches_and_sizes(lib):
    for k in (0, 1, 127, 128, 129, 1000, 1023):
        assert _lib.quant_pitch(k) == -(-k // 128) * 128
    for k in (1024, 1025, 4096, 131071):
        assert _lib.quant_pitch(k) == -(-k // 256) * 256
    for k, n in ((1, 1), (100, 64), (1001, 65), (4096, 14336)):
        kp = _lib.quant_pitch(k)
        one, two = -(-n // 64) * 64, 2 * (-(-n // 32) * 32)
        assert _lib.scaled_size(k, n, False) == (kp * one, 2 * one + 16)
        assert _lib.scaled_size(k, n, True) == (kp * two, 2 * two + 16)


@pytest.mark.parametrize("k,n", [(-1, 1), (1, -1), (131072, 1), (1, 65535 * 64 + 1)])
def test_sizes_that_no_weight_has(lib, k, n):
    with pytest.raises(HipGemmError):
        _lib.scaled_size(k, n, False)


def test_int32_sums_bound_k(lib):
    """131071 products of -128 and -128 stay below 2^31, 131072 do not."""
    assert 131071 * 16384 < 2**31 <= 131072 * 16384
    assert _lib.scaled_size(131071, 16, False)[0] > 0
    assert lib.vt_scaled_linear(16, F32, 131072, None, 1, 131072, 16, 16, 16, 1 << 40, F32, 16, None) == _lib.VT_EINVAL
    assert "131071" in _lib.last_error()


BASE = 1 << 20     # addresses that no check reads


def linear(lib, **kw):
    a = dict(X=BASE, xt=F32, ldx=64, T=None, M=4, K=64, B=BASE * 2, meta=BASE * 3, N=32, Y=BASE * 4, yt=F32, ldy=32)
    a.update(kw)
    return lib.vt_scaled_linear(a["X"], a["xt"], a["ldx"], a["T"], a["M"], a["K"], a["B"], a["meta"], a["N"], a["Y"],
                                a["yt"], a["ldy"], None)


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(K=-1), dict(N=-1), dict(M=1 << 30), dict(xt=0), dict(xt=9), dict(yt=I8), dict(X=None), dict(B=None),
    dict(meta=None), dict(Y=None), dict(ldx=63), dict(ldy=31), dict(ldx=1 << 41), dict(X=BASE + 2), dict(Y=BASE * 4 + 1),
    dict(B=BASE * 2 + 4), dict(meta=BASE * 3 + 4), dict(Y=BASE), dict(Y=BASE * 2), dict(Y=BASE * 3),
    dict(xt=I8, ldx=64),                                         # int8 rows without scales
    dict(xt=I8, ldx=64, T=BASE * 4),                             # scales that the output overwrites
    dict(xt=I8P, ldx=64, T=BASE * 5),                            # padded rows are 128 bytes
    dict(xt=I8P, ldx=136, T=BASE * 5), dict(xt=I8P, ldx=128, T=BASE * 5, X=BASE + 8),
], ids=str)
def test_native_refusals(lib, kw):
    assert linear(lib, **kw) == _lib.VT_EINVAL, kw
    assert "vt_scaled_linear" in _lib.last_error()


FAR = 1 << 44      # addresses this far apart


def many_rows(lib, m):
    return [linear(lib, M=m, X=FAR, Y=2 * FAR), lib.vt_quant_rows(FAR, F32, 64, 2 * FAR, 128, 3 * FAR, m, 64, None)]


def test_more_rows_than_a_launch_takes(lib):
    # a workgroup per row of up to 256 threads: 2^24 rows would be 2^32 threads
    assert many_rows(lib, 1 << 24) == [_lib.VT_EINVAL] * 2


def test_empty_calls_need_no_device(lib):
    assert linear(lib, M=0, X=None, Y=None) == _lib.VT_OK
    assert linear(lib, N=0, Y=None, B=None) == _lib.VT_OK
    assert lib.vt_quant_rows(None, F32, 0, None, 0, None, 0, 0, None) == _lib.VT_OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="no call here reaches a device")
def test_valid_calls_end_without_a_device(lib):
    for kw in ({}, dict(xt=BF16, yt=F16), dict(xt=I8, T=BASE * 5), dict(xt=I8P, ldx=128, T=BASE * 5), dict(K=0, X=None, B=None),
               dict(X=BASE + 4), dict(Y=BASE * 4 + 4, ldy=33)):
        assert linear(lib, **kw) == _lib.VT_ENODEV, kw
    assert many_rows(lib, (1 << 24) - 1) == [_lib.VT_ENODEV] * 2


def test_other_entries_refuse(lib):
    p = BASE
    q = lib.vt_quant_rows
    assert q(p, F32, 64, p * 2, 128, p * 3, -1, 64, None) == _lib.VT_EINVAL
    assert q(p, I8, 64, p * 2, 128, p * 3, 1, 64, None) == _lib.VT_EINVAL
    assert q(p, F32, 63, p * 2, 128, p * 3, 1, 64, None) == _lib.VT_EINVAL
    assert q(p, F32, 64, p * 2, 127, p * 3, 1, 64, None) == _lib.VT_EINVAL
    assert q(p, F32, 64, p * 2 + 8, 128, p * 3, 1, 64, None) == _lib.VT_EINVAL
    assert q(p, F32, 64, p, 128, p * 3, 1, 64, None) == _lib.VT_EINVAL           # in place
    pack = lib.vt_scaled_pack
    assert pack(p, None, 16, 0, p * 2, None, None, 64, 32, p * 3, p * 4, None) == _lib.VT_EINVAL        # pitch
    assert pack(p, None, 32, 0, None, None, None, 64, 32, p * 3, p * 4, None) == _lib.VT_EINVAL         # scales
    assert pack(p, p * 5, 32, 32, p * 2, p * 2, p * 2, 64, 32, p * 3, p * 4, None) == _lib.VT_EINVAL    # bias of a pair
    assert pack(p, None, 32, 0, p * 2, p * 2, None, 64, 32, p * 3, p * 4, None) == _lib.VT_EINVAL       # half a pair
    assert pack(p, None, 32, 0, p * 2, None, None, 64, 32, p, p * 4, None) == _lib.VT_EINVAL            # overlap
    g = lib.vt_scaled_gated
    assert g(p, F32, 64, None, 4, 64, p * 2, p * 3, 32, 2, p * 4, F32, 32, None) == _lib.VT_EINVAL
    assert "activation" in _lib.last_error()
    lg = lib.vt_scaled_linear_grad
    assert lg(p, I8, 32, 4, 64, p * 2, p * 3, 32, p * 4, 64, None) == _lib.VT_EINVAL
    assert lg(p, F32, 31, 4, 64, p * 2, p * 3, 32, p * 4, 64, None) == _lib.VT_EINVAL
    assert lg(p, F32, 32, 4, 64, p * 2, p * 3, 32, p * 4, 63, None) == _lib.VT_EINVAL
    assert lg(p, F32, 32, 4, 64, p * 2, p * 3, 32, p, 64, None) == _lib.VT_EINVAL
    gg = lib.vt_scaled_gated_grad
    ok = [p, F32, 32, p * 5, I8, 64, p * 6, 4, 64, p * 2, p * 3, 32, 0, p * 4, 64, None]
    for at, bad in ((1, I8), (4, F32), (5, 63), (6, None), (12, 7), (13, p * 5), (13, p * 6)):
        args = list(ok)
        args[at] = bad
        assert gg(*args) == _lib.VT_EINVAL, (at, bad)


def cpu_weight(pair=False):
    return scaled.ScaledWeight(torch.zeros(128 * 64, dtype=torch.int8), torch.zeros(2 * 64 + 16), 100, 32 if pair else 60, pair)


def test_python_refusals():
    w, s = torch.zeros(100, 60, dtype=torch.int8), torch.ones(60)
    for call in (lambda: scaled.pack_linear(w, s), lambda: scaled.pack_gated(w, s, w, s),
                 lambda: scaled.quantize_rows(torch.zeros(3, 100)), lambda: scaled.quantize_weight(torch.zeros(100, 60)),
                 lambda: scaled.linear(torch.zeros(3, 100), cpu_weight()),
                 lambda: scaled.linear_grad(torch.zeros(3, 60), cpu_weight())):
        with pytest.raises(HipGemmError, match="no CPU path"):
            call()
    for call, what in ((lambda: scaled.pack_linear(w.float(), s), "int8"),
                       (lambda: scaled.pack_linear(w[0], s), "int8"),
                       (lambda: scaled.quantize_rows(torch.zeros(3, 100, dtype=torch.float64)), "float32"),
                       (lambda: scaled.quantize_rows([1.0]), "torch tensor"),
                       (lambda: scaled.quantize_weight(torch.zeros(3)), "k, n"),
                       (lambda: scaled.gated(torch.zeros(3, 100), cpu_weight(True), act="relu"), "act must be"),
                       (lambda: scaled.gated_grad(torch.zeros(3, 32), None, cpu_weight(True), act="tanh"), "act must be"),
                       (lambda: scaled.QuantRows(w.float(), s), "int8"),
                       (lambda: scaled.QuantRows(w, torch.ones(60)), "scale"),
                       (lambda: scaled.QuantRows(w, torch.ones(100, dtype=torch.float64)), "scale"),
                       (lambda: scaled.QuantRows(w.t(), torch.ones(60)), "unit stride"),
                       (lambda: scaled.linear(scaled.QuantRows(w, torch.ones(100)), cpu_weight(), out_dtype=torch.float32),
                        "no CPU path")):
        with pytest.raises(HipGemmError, match=what):
            call()


def test_quant_rows_stand_for_their_values():
    q = torch.from_numpy(np.array([[127, -127], [0, 64]], np.int8))
    r = scaled.QuantRows(q, torch.tensor([0.5, 2.0]))
    assert r.shape == (2, 2) and not r.padded
    assert torch.equal(r.dequantize(), torch.tensor([[63.5, -63.5], [0.0, 128.0]]))


def test_feed_forward_checks_its_weights():
    G, D = cpu_weight(True), cpu_weight()
    with pytest.raises(HipGemmError, match="pack_gated"):
        feed_forward.FeedForward(D, D)
    with pytest.raises(HipGemmError, match="pack_linear"):
        feed_forward.FeedForward(G, G)
    with pytest.raises(HipGemmError, match="down takes"):
        feed_forward.FeedForward(G, D)
    fit = scaled.ScaledWeight(D.data, D.meta, G.n, 60, False)
    with pytest.raises(HipGemmError, match="act must be"):
        feed_forward.FeedForward(G, fit, act="relu")
    assert feed_forward.FeedForward(G, fit).act == "silu"


def test_the_header_says_what_python_uses():
    text = open(_lib.PKG_DIR + "/../include/vt_hip_gemm.h").read()
    for name, value in (("TYPE_F32", F32), ("TYPE_F16", F16), ("TYPE_BF16", BF16), ("TYPE_I8", I8), ("TYPE_I8_PADDED", I8P),
                        ("ACT_SILU", _lib.ACT_IDS["silu"]), ("ACT_GELU", _lib.ACT_IDS["gelu"])):
        assert "#define VT_%s %d" % (name, value) in text
    assert ctypes.sizeof(ctypes.c_void_p) == 8
