"""Which stream everything that a norm, an adapter or a loss enqueues is on, without a GPU (the fixture and what it
stands for: test_scaled_streams_host.py)."""
import contextlib

import pytest

torch = pytest.importorskip("torch")

from test_scaled_streams_host import MAIN, SIDE, log  # noqa: F401
from veritac_amd import _lib
from veritac_amd.specializations.hip_gemm import adapters, losses, norms, scaled

M, K, N = 6, 64, 48


@pytest.fixture
def here(log, monkeypatch):  # noqa: F811
    for module in (norms, losses, adapters):
        monkeypatch.setattr(module, "_current_stream", lambda d: log.current)
        monkeypatch.setattr(module, "_on", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(scaled, "_on", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "adapter_size", lambda *a: 64)
    return log


def far(cols):
    """Rows that do not flatten, so that a call copies them."""
    return torch.ones(2, 3, cols).transpose(0, 1)


def head():
    return scaled.ScaledWeight(torch.zeros(128 * 64, dtype=torch.int8), torch.zeros(2 * 64 + 16), K, N, False)


DOWN, UP = torch.ones(2, 4, K), torch.ones(2, N, 4).transpose(1, 2).contiguous().transpose(1, 2)
CALLS = {
    "norm": lambda **kw: norms.norm(far(K), torch.ones(K), **kw),
    "norm of a sum": lambda **kw: norms.norm(far(K), torch.ones(K), residual=far(K), **kw),
    "norm_rows": lambda **kw: norms.norm_rows(far(K), torch.ones(K), residual=far(K), **kw),
    "norm_grad": lambda **kw: norms.norm_grad(far(K), far(K), torch.ones(K), dh=far(K), **kw),
    "cross_entropy": lambda **kw: losses.cross_entropy(far(K), head(), torch.zeros(2, 3, dtype=torch.int64).transpose(0, 1), **kw),
    "losses": lambda **kw: losses.cross_entropy(far(K), head(), torch.zeros(3, 2, dtype=torch.int32), reduction="none", **kw),
    "pack_adapters": lambda **kw: adapters.pack_adapters(DOWN, UP, **kw),
    "adapted": lambda **kw: adapters.adapted(far(K), head(), (DOWN, UP), torch.zeros(2, 3, dtype=torch.int32).transpose(0, 1), **kw),
    "adapted_grad": lambda **kw: adapters.adapted_grad(far(N), far(K), head(), (DOWN, UP, 2.0), None, **kw),
}


def pointers(result):
    if isinstance(result, adapters.Adapters):
        return {result.data.data_ptr()}
    if isinstance(result, tuple):
        return {p for r in result for p in pointers(r)}
    if isinstance(result, scaled.QuantRows):
        return {result.data.data_ptr(), result.scale.data_ptr()}
    return {result.data_ptr()}


@pytest.mark.parametrize("name", CALLS)
def test_all_work_of_a_call_is_on_its_stream(here, name):
    for stream, want in ((None, MAIN), (MAIN, MAIN), (SIDE, SIDE)):
        del here.work[:], here.recorded[:]
        result = CALLS[name](**({} if stream is None else {"stream": stream}))
        # the operands are made within the call's expression, on the caller's stream
        seen = [w for w in here.work if w[0] not in ("ones", "zeros", "fill_", "zero_")]
        assert any(w[0].startswith("vt_") for w in seen) and {w[1] for w in seen} == {want}, (stream, seen)
        assert here.current == MAIN
        assert {p for p, s in here.recorded if s == MAIN} == (pointers(result) if want == SIDE else set())


def test_given_outputs_are_the_caller_s(here):
    x, r = torch.ones(M, K), torch.ones(M, K)
    out, h = torch.empty(M, K), torch.empty(M, K)
    got = norms.norm(x, torch.ones(K), residual=r, out=out, h_out=h, stream=SIDE)
    assert got[0] is out and got[1] is h and not here.recorded
    y = torch.empty(M, N)
    assert adapters.adapted(x, head(), (DOWN, UP), out=y, stream=SIDE) is y and not here.recorded
