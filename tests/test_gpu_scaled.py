"""Scaled int8 operators on the GPU against their definitions in 64 bits (tests/scaled_ref.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import scaled_ref as ref
from veritac_amd import _lib
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    assert _lib.load_library().vt_device_count() >= 1, "GPU visible but not gfx950"
    return torch.device("cuda", 0)


def say(*a):
    print(*a, flush=True)


def weights(rng, k, n, least=-127):
    w = np.clip(np.rint(rng.normal(0, 32, (k, n))), least, 127).astype(np.int8)
    s = ((rng.random(n) + 0.5) / (32 * max(k, 1)**0.5)).astype(np.float32)
    return w, s


def rows(rng, m, k, dtype):
    """Activations of `dtype` with a few large columns, a row of zeros, and their float32 values."""
    x = rng.normal(0, 1, (m, k)) * np.where(rng.random(k) < 0.02, 12.0, 1.0)
    if m > 3:
        x[m // 2] = 0.0
    x = torch.from_numpy(x.astype(np.float32)).to(dtype)
    return x, x.float().numpy()


def up(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def packed(dev, w, s, bias=None):
    return scaled.pack_linear(up(w, dev), up(s, dev), None if bias is None else up(bias, dev))


def packed_pair(dev, wg, sg, wu, su):
    return scaled.pack_gated(up(wg, dev), up(sg, dev), up(wu, dev), up(su, dev))


# --- rows to int8 -----------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k", [(1, 1), (2, 15), (3, 16), (5, 63), (4, 64), (7, 65), (3, 1000), (2, 1024), (3, 1025),
                                 (2, 4096), (2, 4097), (3, 8191), (2, 16384), (2, 16400), (2, 40001)])
def test_quantize_rows_equals_the_definition(dev, m, k, dtype):
    rng = np.random.default_rng(m * 100003 + k)
    x, x32 = rows(rng, m, k, dtype)
    say("quantize", m, k, dtype)
    r = scaled.quantize_rows(x.to(dev))
    q, t = ref.quantize(x32)
    assert np.array_equal(r.scale.cpu().numpy(), t)
    got = r.data.cpu().numpy()
    assert np.array_equal(got[:, :k], q)
    assert not got[:, k:].any()
    assert np.array_equal(r.dequantize().cpu().numpy(), q.astype(np.float32) * t[:, None])


def test_quantize_rows_of_ties_extremes_and_non_finite_values(dev):
    x = np.zeros((12, 70), np.float32)
    x[0, :6] = [127, 0.5, 1.5, 2.5, -0.5, -1.5]          # ties to even
    x[1, 3] = 3.4e38
    x[2, 5] = 2.0**-120                                  # the least row that is not zeros
    x[3, 5] = np.nextafter(np.float32(2.0**-120), np.float32(0))
    x[4, :3] = [1e-45, -1e-40, 1e-39]
    x[5, :2] = [np.inf, 1.0]
    x[6, :2] = [-np.inf, np.nan]
    x[7, 69] = np.nan
    x[8, :2] = [-0.0, 0.0]
    x[9] = -5.0
    x[10, 0], x[10, 1:] = 1.0, 1.0 / 254
    x[11, :2] = [-3.4028235e38, 3.4028235e38]
    r = scaled.quantize_rows(up(x, dev))
    q, t = ref.quantize(x)
    assert np.array_equal(r.scale.cpu().numpy(), t, equal_nan=True)
    assert np.array_equal(r.data.cpu().numpy()[:, :70], q)
    assert np.isnan(t[5:8]).all() and t[3] == 0 and t[4] == 0 and t[2] > 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_quantize_rows_of_any_pitch_and_alignment(dev, dtype):
    rng = np.random.default_rng(5)
    x, x32 = rows(rng, 6, 300, dtype)
    for shift, pitch in ((0, 304), (1, 301), (3, 320), (0, 300)):
        flat = torch.full((6 * pitch + shift + 8,), float("nan"), dtype=dtype, device=dev)
        view = flat[shift:shift + 6 * pitch].view(6, pitch)[:, :300]
        view.copy_(x)
        r = scaled.quantize_rows(view)
        q, t = ref.quantize(x32)
        assert np.array_equal(r.scale.cpu().numpy(), t) and np.array_equal(r.data.cpu().numpy()[:, :300], q)


def test_quantize_weight_rounds_each_channel(dev):
    w = torch.randn(70, 33, device=dev)
    q, s = scaled.quantize_weight(w)
    qr, tr = ref.quantize(w.cpu().numpy().T)
    assert np.array_equal(q.cpu().numpy(), qr.T) and np.array_equal(s.cpu().numpy(), tr)


# --- forward ----------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 16, 16), (2, 64, 64), (5, 120, 72), (3, 63, 65), (16, 300, 31), (17, 256, 33), (33, 130, 200),
          (48, 1024, 96), (64, 1000, 130), (65, 333, 203), (100, 1023, 97), (130, 1024, 300), (257, 1025, 511),
          (300, 2048, 1000), (512, 1024, 2048), (1, 4096, 1000), (4, 5000, 260), (1000, 320, 1300), (700, 4096, 520),
          # few rows: rounded by the product itself or not, K in slices that finish in it or not
          (1, 16384, 40), (3, 5000, 20), (16, 2048, 48), (9, 1700, 1000), (16, 1024, 500), (2, 131071, 17)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(dev, m, k, n, dtype):
    rng = np.random.default_rng(m * 7919 + k * 31 + n)
    x, x32 = rows(rng, m, k, dtype)
    w, s = weights(rng, k, n)
    bias = rng.normal(0, 0.3, n).astype(np.float32) if n % 2 else None
    say("linear", m, k, n, dtype)
    y = scaled.linear(x.to(dev), packed(dev, w, s, bias))
    assert y.dtype == dtype and y.shape == (m, n)
    want, bound = ref.linear(*ref.quantize(x32), w, s, bias)
    ref.check(y, want, bound, dtype, "linear")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_gated(dev, m, k, n, dtype, act):
    rng = np.random.default_rng(m * 104729 + k * 31 + n)
    x, x32 = rows(rng, m, k, dtype)
    (wg, sg), (wu, su) = weights(rng, k, n), weights(rng, k, n)
    say("gated", m, k, n, dtype, act)
    h = scaled.gated(x.to(dev), packed_pair(dev, wg, sg, wu, su), act=act)
    assert h.dtype == dtype and h.shape == (m, n)
    want, bound = ref.gated(*ref.quantize(x32), wg, sg, wu, su, act)
    ref.check(h, want, bound, dtype, "gated " + act)


# (m, k, packed columns): enough tiles of 256 x 256 or 256 x 128 for the persistent kernels, ragged ends
LARGE = [(4000, 1000, 3904), (2000, 4000, 4032), (260, 1500, 17000), (2100, 200, 8000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,cols", LARGE)
def test_linear_on_whole_chip_tiles(dev, m, k, cols, dtype):
    rng = np.random.default_rng(m + k)
    x, x32 = rows(rng, m, k, dtype)
    n = cols - 4
    w, s = weights(rng, k, n)
    bias = rng.normal(0, 0.3, n).astype(np.float32)
    say("linear", m, k, n, dtype)
    y = scaled.linear(x.to(dev), packed(dev, w, s, bias))
    ref.check(y, *ref.linear(*ref.quantize(x32), w, s, bias), dtype, "linear")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,cols", LARGE)
def test_gated_on_whole_chip_tiles(dev, m, k, cols, dtype, act):
    rng = np.random.default_rng(m + k)
    x, x32 = rows(rng, m, k, dtype)
    n = cols // 2 - 5
    (wg, sg), (wu, su) = weights(rng, k, n), weights(rng, k, n)
    say("gated", m, k, n, dtype, act)
    h = scaled.gated(x.to(dev), packed_pair(dev, wg, sg, wu, su), act=act)
    ref.check(h, *ref.gated(*ref.quantize(x32), wg, sg, wu, su, act), dtype, "gated")


@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (20, 100, 70), (70, 1024, 256), (300, 1300, 520)])
def test_int8_rows_with_every_value(dev, m, k, n):
    """Rows that are int8 already: -128 among them, any pitch, scales that are zero or negative."""
    rng = np.random.default_rng(m + k + n)
    q = rng.integers(-128, 128, (m, k), dtype=np.int8)
    t = rng.normal(0, 0.1, m).astype(np.float32)
    t[m // 2] = 0.0
    w, s = weights(rng, k, n, -128)
    s[n // 2] = -s[n // 2]
    w2, s2 = weights(rng, k, n, -128)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w2, s2)
    for shift, pitch in ((0, k), (1, k + 3), (16, -(-k // 16) * 16 + 16)):
        flat = torch.full((m * pitch + 64,), 77, dtype=torch.int8, device=dev)
        view = flat[shift:shift + m * pitch].view(m, pitch)[:, :k]
        view.copy_(torch.from_numpy(q))
        r = scaled.QuantRows(view, up(t, dev))
        want, bound = ref.linear(q, t, w, s)
        ref.check(scaled.linear(r, W, out_dtype=torch.float32), want, bound, torch.float32, "linear")
        want, bound = ref.gated(q, t, w, s, w2, s2, "silu")
        ref.check(scaled.gated(r, G, out_dtype=torch.bfloat16), want, bound, torch.bfloat16, "gated")


def test_the_longest_sums_stay_exact(dev):
    """131071 products of -128 and -128: the largest sum that int32 holds."""
    k = 131071
    q, w = np.full((3, k), -128, np.int8), np.full((k, 5), -128, np.int8)
    q[1], w[:, 2] = 127, 127
    t, s = np.ones(3, np.float32), np.ones(5, np.float32)
    y = scaled.linear(scaled.QuantRows(up(q, dev), up(t, dev)), packed(dev, w, s), out_dtype=torch.float32)
    assert np.array_equal(y.cpu().numpy(), (q.astype(np.float64) @ w.astype(np.float64)).astype(np.float32))


def test_rows_rounded_once_serve_several_products(dev):
    rng = np.random.default_rng(3)
    x, x32 = rows(rng, 37, 520, torch.bfloat16)
    r = scaled.quantize_rows(x.to(dev))
    for n in (16, 99):
        w, s = weights(rng, 520, n)
        W = packed(dev, w, s)
        assert torch.equal(scaled.linear(r, W, out_dtype=torch.bfloat16), scaled.linear(x.to(dev), W))


@pytest.mark.parametrize("m,n", [(1, 70), (5, 256), (300, 264), (70, 515)])
def test_outputs_of_any_pitch_leave_the_rest_alone(dev, m, n):
    rng = np.random.default_rng(n)
    x, x32 = rows(rng, m, 256, torch.bfloat16)
    w, s = weights(rng, 256, n)
    w2, s2 = weights(rng, 256, n)
    for shift, pitch in ((0, n + 8), (1, n + 1), (3, n + 5)):
        for op in ("linear", "gated"):
            flat = torch.full((m * pitch + 8,), 7.0, dtype=torch.bfloat16, device=dev)
            out = flat[shift:shift + m * pitch].view(m, pitch)[:, :n]
            if op == "linear":
                assert scaled.linear(x.to(dev), packed(dev, w, s), out=out) is out
                want, bound = ref.linear(*ref.quantize(x32), w, s)
            else:
                assert scaled.gated(x.to(dev), packed_pair(dev, w, s, w2, s2), out=out) is out
                want, bound = ref.gated(*ref.quantize(x32), w, s, w2, s2, "silu")
            ref.check(out.contiguous(), want, bound, torch.bfloat16, op)
            out.fill_(7.0)
            assert (flat == 7.0).all()


def test_rows_that_hold_nan_or_infinity_give_nan_and_spoil_no_other(dev):
    rng = np.random.default_rng(11)
    for m in (6, 70, 300):
        x, x32 = rows(rng, m, 200, torch.float32)
        w, s = weights(rng, 200, 65)
        w2, s2 = weights(rng, 200, 65)
        bad = x.clone()
        bad[1, 7], bad[3, 0], bad[m - 1, 199] = float("nan"), float("inf"), float("-inf")
        rows_bad = [1, 3, m - 1]
        keep = [i for i in range(m) if i not in rows_bad]
        for f in (lambda v: scaled.linear(v.to(dev), packed(dev, w, s)),
                  lambda v: scaled.gated(v.to(dev), packed_pair(dev, w, s, w2, s2), act="gelu")):
            y, good = f(bad), f(x)
            assert torch.isnan(y[rows_bad]).all() and torch.equal(y[keep], good[keep])


def test_large_gates_saturate_without_nan(dev):
    q = np.array([[127, 0], [-127, 0], [1, 0], [0, 127]], np.int8)
    w = np.array([[127, 1], [1, 127]], np.int8)
    for t0 in (1.0, 1e4, 1e15):
        t = np.full(4, t0, np.float32)
        s = np.array([1.0, 0.5], np.float32)
        G = packed_pair(dev, w, s, w, s)
        for act in ("silu", "gelu"):
            h = scaled.gated(scaled.QuantRows(up(q, dev), up(t, dev)), G, act=act, out_dtype=torch.float32)
            want, bound = ref.gated(q, t, w, s, w, s, act)
            ref.check(h, want, bound, torch.float32, act)
            d = np.ones((4, 2), np.float32)
            dx = scaled.gated_grad(up(d, dev), scaled.QuantRows(up(q, dev), up(t, dev)), G, act=act)
            want, bound = ref.gated_grad(d, q, t, w, s, w, s, act, False)
            ref.check(dx, want, bound, torch.float32, act + " gradient")


def test_empty_sizes(dev):
    w, s = weights(np.random.default_rng(0), 64, 48)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w, s)
    for lead in ((0,), (2, 0)):
        assert scaled.linear(torch.empty(*lead, 64, device=dev), W).shape == (*lead, 48)
        assert scaled.gated(torch.empty(*lead, 64, device=dev), G).shape == (*lead, 48)
        assert scaled.linear_grad(torch.empty(*lead, 48, device=dev), W).shape == (*lead, 64)
    none = packed(dev, np.zeros((0, 48), np.int8), s, np.arange(48, dtype=np.float32))
    y = scaled.linear(torch.empty(3, 0, device=dev), none)          # an empty sum and the bias
    assert torch.equal(y, torch.arange(48, device=dev).float().expand(3, 48))
    pair = packed_pair(dev, np.zeros((0, 48), np.int8), s, np.zeros((0, 48), np.int8), s)
    assert not scaled.gated(torch.empty(3, 0, device=dev), pair).any()
    assert scaled.linear_grad(torch.ones(3, 48, device=dev), none).shape == (3, 0)
    thin = packed(dev, np.zeros((64, 0), np.int8), np.zeros(0, np.float32))
    assert scaled.linear(torch.ones(3, 64, device=dev), thin).shape == (3, 0)
    assert not scaled.linear_grad(torch.ones(3, 0, device=dev), thin).any()
    thin2 = packed_pair(dev, *[np.zeros((64, 0), np.int8), np.zeros(0, np.float32)] * 2)
    r = scaled.quantize_rows(torch.ones(3, 64, device=dev))
    assert not scaled.gated_grad(torch.ones(3, 0, device=dev), r, thin2).any()


def test_rows_of_more_dimensions(dev):
    rng = np.random.default_rng(2)
    w, s = weights(rng, 64, 40)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w, s)
    x = torch.randn(2, 3, 5, 64, device=dev, dtype=torch.bfloat16)
    assert torch.equal(scaled.linear(x, W), scaled.linear(x.view(30, 64), W).view(2, 3, 5, 40))
    assert torch.equal(scaled.gated(x[0, 0, 0], G), scaled.gated(x[0, 0, :1], G)[0])
    r = scaled.quantize_rows(x)
    assert r.shape == (2, 3, 5, 64) and scaled.linear(r, W, out_dtype=x.dtype).shape == (2, 3, 5, 40)
    d = torch.randn(2, 3, 5, 40, device=dev, dtype=torch.bfloat16)
    assert scaled.linear_grad(d, W).shape == (2, 3, 5, 64)
    assert scaled.gated_grad(d, r, G).shape == (2, 3, 5, 64)


# --- gradients --------------------------------------------------------------

GRAD_SHAPES = [(1, 1, 1), (2, 64, 64), (5, 120, 72), (3, 63, 65), (33, 130, 200), (65, 333, 203), (130, 1024, 300),
               (129, 1025, 129), (300, 500, 1000), (257, 2048, 640), (520, 256, 1500)]


def gradients(rng, m, n, dtype):
    d = torch.from_numpy((rng.normal(0, 1, (m, n)) * 1e-3).astype(np.float32)).to(dtype)
    if m > 3:
        d[m // 2] = 0.0
    return d, d.float().numpy()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", GRAD_SHAPES)
def test_linear_grad(dev, m, k, n, dtype):
    rng = np.random.default_rng(m * 13 + k * 31 + n)
    d, d32 = gradients(rng, m, n, dtype)
    w, s = weights(rng, k, n, -128)
    say("linear_grad", m, k, n, dtype)
    dx = scaled.linear_grad(d.to(dev), packed(dev, w, s))
    assert dx.dtype == dtype and dx.shape == (m, k)
    want, bound = ref.linear_grad(d32, w, s, dtype != torch.float32)
    ref.check(dx, want, bound, dtype, "linear_grad")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", GRAD_SHAPES)
def test_gated_grad(dev, m, k, n, dtype, act):
    rng = np.random.default_rng(m * 17 + k * 31 + n)
    d, d32 = gradients(rng, m, n, dtype)
    x, x32 = rows(rng, m, k, dtype)
    (wg, sg), (wu, su) = weights(rng, k, n, -128), weights(rng, k, n)
    G = packed_pair(dev, wg, sg, wu, su)
    say("gated_grad", m, k, n, dtype, act)
    r = scaled.quantize_rows(x.to(dev))
    dx = scaled.gated_grad(d.to(dev), r, G, act=act)
    q, t = ref.quantize(x32)
    want, bound = ref.gated_grad(d32, q, t, wg, sg, wu, su, act, dtype != torch.float32)
    ref.check(dx, want, bound, dtype, "gated_grad " + act)
    # rows that are not padded give the same
    raw = scaled.QuantRows(up(q, dev), up(t, dev))
    assert torch.equal(dx, scaled.gated_grad(d.to(dev), raw, G, act=act))


# tiles of 128 x 256 and 256 x 256 of the whole chip; one slice, few and many
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(2100, 2048, 20), (1990, 2300, 150), (4000, 4000, 140), (1025, 3900, 700)])
def test_gradients_on_whole_chip_tiles(dev, m, k, n, dtype):
    rng = np.random.default_rng(m + k + n)
    d, d32 = gradients(rng, m, n, dtype)
    w, s = weights(rng, k, n, -128)
    say("linear_grad", m, k, n, dtype)
    dx = scaled.linear_grad(d.to(dev), packed(dev, w, s))
    ref.check(dx, *ref.linear_grad(d32, w, s, dtype != torch.float32), dtype, "linear_grad")
    w2, s2 = weights(rng, k, n)
    x, x32 = rows(rng, m, k, dtype)
    q, t = ref.quantize(x32)
    say("gated_grad", m, k, n, dtype)
    dx = scaled.gated_grad(d.to(dev), scaled.quantize_rows(x.to(dev)), packed_pair(dev, w, s, w2, s2))
    ref.check(dx, *ref.gated_grad(d32, q, t, w, s, w2, s2, "silu", dtype != torch.float32), dtype, "gated_grad")


# contractions split over workgroups on those tiles, in parts of unequal length
@pytest.mark.parametrize("m,k,n,dtype", [(2050, 1000, 3000, torch.float32), (2050, 500, 4000, torch.float32),
                                         (2050, 2000, 4000, torch.float32), (1100, 1025, 8000, torch.bfloat16),
                                         (2050, 2000, 8000, torch.float16)])
def test_split_contractions_on_large_tiles(dev, m, k, n, dtype):
    rng = np.random.default_rng(m + k + n)
    d, d32 = gradients(rng, m, n, dtype)
    w, s = weights(rng, k, n, -128)
    say("linear_grad", m, k, n, dtype)
    W = packed(dev, w, s)
    dx = scaled.linear_grad(d.to(dev), W)
    ref.check(dx, *ref.linear_grad(d32, w, s, dtype != torch.float32), dtype, "linear_grad")
    assert torch.equal(dx, scaled.linear_grad(d.to(dev), W))      # the sums' order is fixed


@pytest.mark.parametrize("dtype,act", [(torch.float32, "gelu"), (torch.bfloat16, "silu")], ids=["f32-gelu", "bf16-silu"])
@pytest.mark.parametrize("m,k,n", [(4000, 1000, 1947), (2000, 4000, 2011)])
def test_gated_grad_terms_on_whole_chip_tiles(dev, m, k, n, dtype, act):
    rng = np.random.default_rng(m + k + n)
    d, d32 = gradients(rng, m, n, dtype)
    (wg, sg), (wu, su) = weights(rng, k, n, -128), weights(rng, k, n)
    x, x32 = rows(rng, m, k, dtype)
    q, t = ref.quantize(x32)
    say("gated_grad", m, k, n, dtype, act)
    dx = scaled.gated_grad(d.to(dev), scaled.quantize_rows(x.to(dev)), packed_pair(dev, wg, sg, wu, su), act=act)
    ref.check(dx, *ref.gated_grad(d32, q, t, wg, sg, wu, su, act, dtype != torch.float32), dtype, "gated_grad")


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_grad_equals_differences(dev, act):
    """Central differences of the 64-bit definition along random directions of x^."""
    rng = np.random.default_rng(8)
    m, k, n = 6, 150, 90
    d, d32 = gradients(rng, m, n, torch.float32)
    x, x32 = rows(rng, m, k, torch.float32)
    (wg, sg), (wu, su) = weights(rng, k, n), weights(rng, k, n)
    q, t = ref.quantize(x32)
    dx = scaled.gated_grad(d.to(dev), scaled.quantize_rows(x.to(dev)), packed_pair(dev, wg, sg, wu, su),
                           act=act).cpu().double().numpy()
    xhat = q.astype(np.float64) * t[:, None]

    def loss(v):
        g = v @ wg.astype(np.float64) * sg
        u = v @ wu.astype(np.float64) * su
        return (d32 * ref.act(g, act)[0] * u).sum(axis=1)

    for _ in range(5):
        v = rng.normal(0, 1, (m, k))
        h = 1e-5
        slope = (loss(xhat + h * v) - loss(xhat - h * v)) / (2 * h)
        # differences are good to h^2 of the third derivative and 2^-52 / h of the loss; the
        # gradient to 2^-20 of its terms' size
        size = (np.abs(dx) * np.abs(v)).sum(axis=1) + 1e-12
        assert (np.abs(slope - (dx * v).sum(axis=1)) <= 1e-5 * size).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_autograd_gives_those_gradients(dev, dtype):
    rng = np.random.default_rng(21)
    x = torch.randn(3, 7, 96, device=dev, dtype=dtype)
    (wg, sg), (wu, su), (wd, sd) = weights(rng, 96, 130), weights(rng, 96, 130), weights(rng, 130, 50)
    G, D = packed_pair(dev, wg, sg, wu, su), packed(dev, wd, sd)
    leaf = x.clone().requires_grad_(True)
    h = scaled.gated(leaf, G, act="gelu")
    y = scaled.linear(h, D)
    with torch.no_grad():
        h0 = scaled.gated(x, G, act="gelu")
        assert torch.equal(h, h0) and torch.equal(y, scaled.linear(h0, D))
    d = torch.randn_like(y)
    (y * d).sum().backward()
    dh = scaled.linear_grad(d, D)
    want = scaled.gated_grad(dh, scaled.quantize_rows(x), G, act="gelu")
    assert torch.equal(leaf.grad, want) and leaf.grad.dtype == dtype
    # a broadcast gradient (of a sum) and a transposed one
    leaf.grad = None
    scaled.linear(leaf, packed(dev, wg, sg)).sum().backward()
    ones = torch.ones(3, 7, 130, device=dev, dtype=dtype)
    assert torch.equal(leaf.grad, scaled.linear_grad(ones, packed(dev, wg, sg)))
    with torch.no_grad():
        assert not scaled.linear(leaf, packed(dev, wg, sg)).requires_grad


def test_gradients_of_rows_that_hold_nan_or_infinity(dev):
    rng = np.random.default_rng(12)
    w, s = weights(rng, 100, 70)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w, s)
    x, _ = rows(rng, 9, 100, torch.float32)
    r = scaled.quantize_rows(x.to(dev))
    d, _ = gradients(rng, 9, 70, torch.float32)
    bad = d.clone()
    bad[2, 3], bad[5, 69] = float("nan"), float("inf")
    keep = [0, 1, 3, 4, 6, 7, 8]
    for f in (lambda v: scaled.linear_grad(v.to(dev), W), lambda v: scaled.gated_grad(v.to(dev), r, G)):
        y, good = f(bad), f(d)
        assert torch.isnan(y[[2, 5]]).all() and torch.equal(y[keep], good[keep])


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e6, 1e25])
def test_gradients_of_any_magnitude(dev, scale):
    """The rows' power of two keeps float16 terms in range whatever the loss is scaled by."""
    rng = np.random.default_rng(14)
    m, k, n = 20, 90, 110
    w, s = weights(rng, k, n)
    w2, s2 = weights(rng, k, n)
    x, x32 = rows(rng, m, k, torch.float32)
    q, t = ref.quantize(x32)
    d = (rng.normal(0, 1, (m, n)) * scale * 10.0**rng.uniform(-3, 3, (m, 1))).astype(np.float32)
    dx = scaled.linear_grad(up(d, dev), packed(dev, w, s))
    ref.check(dx, *ref.linear_grad(d, w, s, False), torch.float32, "linear_grad")
    dx = scaled.gated_grad(up(d, dev), scaled.quantize_rows(x.to(dev)), packed_pair(dev, w, s, w2, s2))
    ref.check(dx, *ref.gated_grad(d, q, t, w, s, w2, s2, "silu", False), torch.float32, "gated_grad")


# --- streams, graphs, offsets ---------------------------------------------------

def test_calls_on_another_stream(dev):
    rng = np.random.default_rng(31)
    w, s = weights(rng, 512, 384)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w, s)
    xs = [torch.randn(m, 512, device=dev, dtype=torch.bfloat16) for m in (1, 40, 400)]
    want = [(scaled.linear(x, W), scaled.gated(x, G), scaled.linear_grad(scaled.linear(x, W), W)) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [(scaled.linear(x, W), scaled.gated(x, G), scaled.linear_grad(scaled.linear(x, W), W)) for x in xs]
    raw = [scaled.gated(x, G, stream=side.cuda_stream) for x in xs]
    side.synchronize()
    for a, b, c in zip(want, got, raw):
        assert all(torch.equal(u, v) for u, v in zip(a, b)) and torch.equal(a[1], c)


@pytest.mark.parametrize("m", [1, 8, 48, 300])
def test_a_captured_block_replays(dev, m):
    """Gate, up and down of a block in one HIP graph, replayed on new inputs between eager work."""
    rng = np.random.default_rng(m)
    (wg, sg), (wu, su), (wd, sd) = weights(rng, 1024, 1500), weights(rng, 1024, 1500), weights(rng, 1500, 1024)
    G, D = packed_pair(dev, wg, sg, wu, su), packed(dev, wd, sd)
    x = torch.randn(m, 1024, device=dev, dtype=torch.bfloat16)
    h, y = torch.empty(m, 1500, device=dev, dtype=x.dtype), torch.empty(m, 1024, device=dev, dtype=x.dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        scaled.linear(scaled.gated(x, G, out=h), D, out=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        scaled.linear(scaled.gated(x, G, out=h), D, out=y)
    for i in range(4):
        x.copy_(torch.randn(m, 1024, device=dev))
        want = scaled.linear(scaled.gated(x, G), D)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i


def test_equal_calls_give_equal_bits(dev):
    rng = np.random.default_rng(44)
    w, s = weights(rng, 4096, 600)
    w2, s2 = weights(rng, 4096, 600)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w2, s2)
    for m in (1, 16, 64, 200):
        x = torch.randn(m, 4096, device=dev)
        d = torch.randn(m, 600, device=dev)
        r = scaled.quantize_rows(x)
        runs = [(scaled.linear(x, W), scaled.gated(x, G), scaled.linear_grad(d, W), scaled.gated_grad(d, r, G))
                for _ in range(3)]
        for a in runs[1:]:
            assert all(torch.equal(u, v) for u, v in zip(a, runs[0]))


def test_offsets_past_32_bits(dev):
    """Rows 2^23 elements apart: the last ones lie past 2^32 bytes of x, y and the gradients."""
    rng = np.random.default_rng(9)
    m, k, n, pitch = 300, 256, 192, 1 << 23
    w, s = weights(rng, k, n)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w, s)
    big = torch.empty(m * pitch, dtype=torch.bfloat16, device=dev)
    x = big.view(m, pitch)[:, :k]
    y = big.view(m, pitch)[:, 4096:4096 + n]
    x.copy_(torch.randn(m, k, device=dev))
    xc = x.contiguous()
    assert torch.equal(scaled.linear(x, W), scaled.linear(xc, W))
    r = scaled.quantize_rows(xc)
    for want, f in ((scaled.linear(xc, W), lambda: scaled.linear(xc, W, out=y)),
                    (scaled.gated(xc, G), lambda: scaled.gated(r, G, out=y))):
        f()
        assert torch.equal(y.contiguous(), want)
    dc = y.contiguous()
    z = torch.empty(m * pitch, dtype=torch.bfloat16, device=dev).view(m, pitch)[:, :k]
    scaled.linear_grad(y, W, out=z)
    assert torch.equal(z.contiguous(), scaled.linear_grad(dc, W))
    scaled.gated_grad(y, r, G, out=z)
    assert torch.equal(z.contiguous(), scaled.gated_grad(dc, r, G))


# --- refusals and the example -----------------------------------------------------

def test_mismatches_are_refused(dev):
    rng = np.random.default_rng(1)
    w, s = weights(rng, 96, 40)
    W, G = packed(dev, w, s), packed_pair(dev, w, s, w, s)
    x, d = torch.zeros(3, 96, device=dev), torch.zeros(3, 40, device=dev)
    r = scaled.quantize_rows(x)
    leaf = torch.zeros(3, 96, device=dev, requires_grad=True)
    for call, what in ((lambda: scaled.linear(x[:, :95], W), "95 columns"),
                       (lambda: scaled.linear(x, G), "pack_linear"), (lambda: scaled.gated(x, W), "pack_gated"),
                       (lambda: scaled.linear(x.cpu(), W), "no CPU path"),
                       (lambda: scaled.linear(x.double(), W), "float32"),
                       (lambda: scaled.linear(x, W, out_dtype=torch.int32), "type must be"),
                       (lambda: scaled.linear(r, W), "need out_dtype"),
                       (lambda: scaled.linear(x.t().contiguous().t(), W), "unit stride"),
                       (lambda: scaled.linear(x[:1].expand(3, 96), W), "overlapping rows"),
                       (lambda: scaled.linear(x, W, out=torch.zeros(3, 41, device=dev)), "out must be"),
                       (lambda: scaled.linear(x, W, out=torch.zeros(3, 40, device=dev), out_dtype=torch.float16), "out must be"),
                       (lambda: scaled.linear(x, W, out=torch.zeros(3, 40)), "out must be"),
                       (lambda: scaled.linear(x, W, out=x.view(-1)[:120].view(3, 40)), "overlaps"),
                       (lambda: scaled.linear_grad(d[:, :39], W), "39 columns"),
                       (lambda: scaled.gated_grad(d[:2], r, G), "dh is 2 x 40"),
                       (lambda: scaled.gated_grad(d, x, G), "QuantRows"),
                       (lambda: scaled.linear(leaf, W, out=d), "neither out nor stream"),
                       (lambda: scaled.pack_linear(up(w, dev), up(s, dev)[:39]), "scale of w"),
                       (lambda: scaled.pack_linear(up(w, dev), up(s, dev), up(s, dev).double()), "bias"),
                       (lambda: scaled.pack_gated(up(w, dev), up(s, dev), up(w[:95], dev), up(s, dev)), "w_up has shape")):
        with pytest.raises(Exception, match=what):
            call()
    assert torch.equal(scaled.linear(x, W), torch.zeros(3, 40, device=dev))     # and nothing is left broken


def test_a_feed_forward_block_in_use(dev):
    """The example: int8 rounding leaves the block within a few percent of float32 (each of the
    three roundings of operands to 127 steps of their largest is about 1 % of their size), and an
    adapter trains through it."""
    from veritac_amd.specializations.hip_gemm import feed_forward
    got = feed_forward.main()
    assert got["prefill"] < 0.06 and got["decode"] < 0.06
    assert got["loss_last"] < 0.2 * got["loss_first"]


def test_captured_blocks_replay_beside_eager_calls(dev):
    from veritac_amd.specializations.hip_gemm import feed_forward
    w = [torch.randn(a, b, device=dev) / a**0.5 for a, b in ((512, 1400), (512, 1400), (1400, 512))]
    block = feed_forward.FeedForward.from_float(*w, act="gelu")
    step = block.capture(torch.zeros(5, 512, device=dev, dtype=torch.float16))
    for i in range(4):
        x = torch.randn(5, 512, device=dev, dtype=torch.float16)
        want = block(x)
        step.x.copy_(x)
        step.replay()
        assert torch.equal(step.y, want), i
