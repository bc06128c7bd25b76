"""Calls that take their rows in parts: each row's result is the one it has in a call of few rows."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import scaled_ref as ref
from test_gpu_scaled import dev, packed, packed_pair, say, up, weights  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu

PICK = lambda m, part: sorted({0, 1, part - 1, part, part + 1, m // 2, m - 2, m - 1})      # rows at the parts' ends


def test_forward_in_parts(dev):
    rng = np.random.default_rng(1)
    m, k, n = 40000, 16384, 32          # 655 MB of int8 rows: two parts of 20224 and 19776
    w, s = weights(rng, k, n)
    w2, s2 = weights(rng, k, n)
    x = torch.randn(m, k, device=dev, dtype=torch.bfloat16)
    at = PICK(m, 20224)
    q, t = ref.quantize(x[at].float().cpu().numpy())
    say("linear in parts")
    ref.check(scaled.linear(x, packed(dev, w, s))[at], *ref.linear(q, t, w, s), torch.bfloat16, "linear")
    say("gated in parts")
    ref.check(scaled.gated(x, packed_pair(dev, w, s, w2, s2))[at], *ref.gated(q, t, w, s, w2, s2, "silu"), torch.bfloat16,
              "gated")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_in_parts(dev, dtype):
    rng = np.random.default_rng(2)
    m, k, n = (30000, 96, 8192) if dtype == torch.float32 else (60000, 96, 8192)     # 983 MB of terms
    part = (m // 2 + 255) // 256 * 256
    w, s = weights(rng, k, n)
    d = (torch.randn(m, n, device=dev) * 1e-3).to(dtype)
    at = PICK(m, part)
    d32 = d[at].float().cpu().numpy()
    half = dtype == torch.bfloat16
    say("linear_grad in parts", dtype)
    ref.check(scaled.linear_grad(d, packed(dev, w, s))[at], *ref.linear_grad(d32, w, s, half), dtype, "linear_grad")
    n //= 2
    w, s, (w2, s2) = w[:, :n].copy(), s[:n].copy(), weights(rng, k, n)
    d, d32 = d[:, :n], d32[:, :n]
    q = rng.integers(-127, 128, (m, k), dtype=np.int8)
    t = ((rng.random(m) + 0.5) * 0.02).astype(np.float32)
    say("gated_grad in parts", dtype)
    dx = scaled.gated_grad(d, scaled.QuantRows(up(q, dev), up(t, dev)), packed_pair(dev, w, s, w2, s2))
    ref.check(dx[at], *ref.gated_grad(d32, q[at], t[at], w, s, w2, s2, "silu", half), dtype, "gated_grad")
