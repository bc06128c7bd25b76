"""Bits that the scaled operators keep, on the GPU against their definitions in 64 bits: bounds a few
roundings wide, which an intermediate value of fewer bits leaves."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import scaled_ref as ref
from test_gpu_scaled import dev, gradients, packed, packed_pair, rows, say, up, weights  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu

# --- float16 gradients: terms of 22 bits ----------------------------------------
# scaled_ref's bound for terms in two halves; with one half (11 bits) an element whose terms
# cancel is off by more than its own rounding.


@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (33, 130, 200), (129, 1025, 129), (300, 500, 1000), (2100, 2048, 700)])
def test_float16_linear_gradients_keep_their_bits(dev, m, k, n):
    rng = np.random.default_rng(m + 3 * k + n)
    d, d32 = gradients(rng, m, n, torch.float16)
    w, s = weights(rng, k, n, -128)
    say("linear_grad f16", m, k, n)
    dx = scaled.linear_grad(d.to(dev), packed(dev, w, s))
    ref.check(dx, *ref.linear_grad(d32, w, s, False), torch.float16, "linear_grad")


# the last two: terms from the persistent kernels' tiles
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(2, 64, 64), (65, 333, 203), (130, 1024, 300), (520, 256, 1500), (4000, 1000, 1947),
                                   (2000, 4000, 2011)])
def test_float16_gated_gradients_keep_their_bits(dev, m, k, n, act):
    rng = np.random.default_rng(m + 5 * k + n)
    d, d32 = gradients(rng, m, n, torch.float16)
    x, x32 = rows(rng, m, k, torch.float16)
    (wg, sg), (wu, su) = weights(rng, k, n, -128), weights(rng, k, n)
    q, t = ref.quantize(x32)
    say("gated_grad f16", m, k, n, act)
    dx = scaled.gated_grad(d.to(dev), scaled.quantize_rows(x.to(dev)), packed_pair(dev, wg, sg, wu, su), act=act)
    ref.check(dx, *ref.gated_grad(d32, q, t, wg, sg, wu, su, act, False), torch.float16, "gated_grad " + act)

# --- float32 gated products: the activation's error --------------------------------
# Root mean square of the relative error where |g| <= 1, in units of float32's rounding U: a rounding
# counts 1 / sqrt(3), exp2 and rcp (1 ulp) 2 / sqrt(3). g takes 3 roundings, enters h with a
# sensitivity of up to 1 + |z'(g)| |g| / 2 (silu 1.5 to 1.75, gelu 2) and the exponent's argument with
# 1.2 (silu) or 4 (gelu) more; the logistic function, both products and u take exp2, rcp and 8
# roundings. In quadrature 2.8 U (silu) and 3.2 U (gelu).


@pytest.mark.parametrize("act,limit", [("silu", 3.0), ("gelu", 3.5)])
@pytest.mark.parametrize("m,k,n", [(8, 256, 4000), (300, 256, 520), (2000, 1024, 2048)])
def test_float32_gated_products_keep_their_bits(dev, m, k, n, act, limit):
    rng = np.random.default_rng(m + k + n)
    q = rng.integers(-127, 128, (m, k), dtype=np.int8)
    t = (rng.random(m) + 0.5).astype(np.float32) / 127
    (wg, sg), (wu, su) = weights(rng, k, n), weights(rng, k, n)
    say("gated f32", m, k, n, act)
    h = scaled.gated(scaled.QuantRows(up(q, dev), up(t, dev)), packed_pair(dev, wg, sg, wu, su), act=act,
                     out_dtype=torch.float32)
    want, _ = ref.gated(q, t, wg, sg, wu, su, act)
    near = (np.abs(ref.products(q, t, wg, sg)) <= 1) & (np.abs(want) > 1e-30)
    assert near.mean() > 0.3
    off = (h.cpu().double().numpy()[near] - want[near]) / want[near]
    assert np.sqrt((off**2).mean()) <= limit * ref.U32


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_products_of_very_negative_gates(dev, act):
    """Down to 2^-126 a small act(g) keeps its bits: g from -1 to -150 for silu, to -12 for gelu."""
    g = np.arange(1, 128, dtype=np.float32) * np.float32(1.18 if act == "silu" else 0.09)
    q = -np.arange(1, 128, dtype=np.int8)[:, None]
    w = np.ones((1, 8), np.int8)
    s = np.full(8, g[0], np.float32)
    one = np.ones(8, np.float32)
    t = np.ones(127, np.float32)
    want, bound = ref.gated(q, t, w, s, w, one, act)
    for pad in (0, 200):        # few rows, and tiles
        qp = np.concatenate([q, np.zeros((pad, 1), np.int8)])
        tp = np.ones(127 + pad, np.float32)
        h = scaled.gated(scaled.QuantRows(up(qp, dev), up(tp, dev)), packed_pair(dev, w, s, w, one), act=act,
                         out_dtype=torch.float32)
        ref.check(h[:127].contiguous(), want, bound, torch.float32, act)
