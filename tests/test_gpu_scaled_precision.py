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
