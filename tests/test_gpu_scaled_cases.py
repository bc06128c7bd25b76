"""Every kernel of the scaled operators on the GPU (scaled_cases.py) against the definitions in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import scaled_ref as ref
from scaled_cases import CASES
from test_gpu_scaled import dev, gradients, packed, packed_pair, rows, say, up, weights  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu

KINDS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("op,m,k,n,kind,x_kind", CASES, ids=lambda v: str(v))
def test_case(dev, op, m, k, n, kind, x_kind):
    dtype = KINDS[kind]
    rng = np.random.default_rng(m * 7919 + k * 31 + n)
    act = "gelu" if (m + n) % 2 else "silu"
    say(op, m, k, n, kind, x_kind, act)
    x = None
    if op != "linear_grad":
        if x_kind == "i8":
            q = rng.integers(-128, 128, (m, k), dtype=np.int8)
            t = ((rng.random(m) + 0.5) * 0.02).astype(np.float32)
            x = scaled.QuantRows(up(q, dev), up(t, dev))
        else:
            xs, x32 = rows(rng, m, k, dtype)
            q, t = ref.quantize(x32)
            x = xs.to(dev) if op != "gated_grad" else scaled.quantize_rows(xs.to(dev))
    w, s = weights(rng, k, n, -128)
    if op == "linear":
        bias = rng.normal(0, 0.3, n).astype(np.float32) if n % 2 else None
        got = scaled.linear(x, packed(dev, w, s, bias), out_dtype=dtype)
        want = ref.linear(q, t, w, s, bias)
    elif op == "linear_grad":
        d, d32 = gradients(rng, m, n, dtype)
        got = scaled.linear_grad(d.to(dev), packed(dev, w, s))
        want = ref.linear_grad(d32, w, s, dtype == torch.bfloat16)
    else:
        w2, s2 = weights(rng, k, n)
        G = packed_pair(dev, w, s, w2, s2)
        if op == "gated":
            got = scaled.gated(x, G, act=act, out_dtype=dtype)
            want = ref.gated(q, t, w, s, w2, s2, act)
        else:
            d, d32 = gradients(rng, m, n, dtype)
            got = scaled.gated_grad(d.to(dev), x, G, act=act)
            want = ref.gated_grad(d32, q, t, w, s, w2, s2, act, dtype == torch.bfloat16)
    ref.check(got, *want, dtype, op)
