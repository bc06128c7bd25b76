"""Which stream everything a scaled call enqueues is on, without a GPU: CPU tensors that say they are on
one, a native library that only logs, and a dispatch mode that logs torch's own work. A call's copies,
fills and kernels have to be on one stream, since nobody else can order them, and what it returns has to
be known to the allocator on the stream that its caller goes on with."""
import contextlib

import pytest

torch = pytest.importorskip("torch")
from torch.utils._python_dispatch import TorchDispatchMode

from veritac_amd import _lib
from veritac_amd.specializations.hip_gemm import backend, scaled

MAIN, SIDE = 1111, 2222
NO_WORK = ("empty", "new_empty", "empty_strided", "detach", "alias", "view", "_unsafe_view", "t", "transpose", "permute",
           "slice", "select", "unsqueeze", "as_strided", "expand", "_reshape_alias")


class Stream:
    def __init__(self, handle, device=None):
        self.cuda_stream = handle


class Log(TorchDispatchMode):
    """Torch's operators that write memory, the native calls, and record_stream, with their streams."""

    def __init__(self):
        super().__init__()
        self.current, self.work, self.recorded = MAIN, [], []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        name = func.overloadpacket.__name__
        if name not in NO_WORK:
            self.work.append((name, self.current))
        return func(*args, **(kwargs or {}))


class Native:
    def __init__(self, log):
        self.log, self.real = log, _lib.load_library()

    def __getattr__(self, name):
        if name in ("vt_quant_pitch", "vt_scaled_size"):
            return getattr(self.real, name)

        def call(*args):
            self.log.work.append((name, args[-1]))
            return 0
        return call


@pytest.fixture
def log(monkeypatch):
    log = Log()
    native = Native(log)

    @contextlib.contextmanager
    def on(stream):
        before, log.current = log.current, stream.cuda_stream
        yield
        log.current = before

    def here(make):
        return lambda *a, device=None, **kw: make(*a, **kw)

    monkeypatch.setattr(torch, "empty", here(torch.empty))
    monkeypatch.setattr(torch, "zeros", here(torch.zeros))
    monkeypatch.setattr(torch.Tensor, "device", property(lambda t: torch.device("cuda", 0)), raising=False)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True), raising=False)
    monkeypatch.setattr(torch.Tensor, "record_stream",
                        lambda t, s: log.recorded.append((t.data_ptr(), s.cuda_stream)), raising=False)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Stream(log.current))
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(scaled, "_current_stream", lambda d: log.current)
    monkeypatch.setattr(backend, "_current_stream", lambda d: log.current)
    monkeypatch.setattr(_lib, "load_library", lambda: native)
    with log:
        yield log


K, N = 64, 48


def operands():
    w, s = torch.ones(K, N, dtype=torch.int8), torch.ones(N)
    linear = scaled.ScaledWeight(torch.zeros(128 * 64, dtype=torch.int8), torch.zeros(2 * 64 + 16), K, N, False)
    pair = scaled.ScaledWeight(torch.zeros(128 * 128, dtype=torch.int8), torch.zeros(2 * 128 + 16), K, N, True)
    rows = scaled.QuantRows(torch.zeros(6, 128, dtype=torch.int8), torch.ones(6), k=K, padded=True)
    x, d = torch.ones(2, 3, K).transpose(0, 1), torch.ones(2, 3, N).transpose(0, 1)     # rows that do not flatten
    return w, s, linear, pair, rows, x, d


CALLS = {
    "pack_linear": lambda w, s, L, G, r, x, d, **kw: scaled.pack_linear(w, s, **kw),
    "pack_linear bias": lambda w, s, L, G, r, x, d, **kw: scaled.pack_linear(w, s, s, **kw),
    "pack_gated": lambda w, s, L, G, r, x, d, **kw: scaled.pack_gated(w, s, w, s, **kw),
    "quantize_weight": lambda w, s, L, G, r, x, d, **kw: scaled.quantize_weight(torch.ones(K, N), **kw),
    "quantize_rows": lambda w, s, L, G, r, x, d, **kw: scaled.quantize_rows(x, **kw),
    "linear": lambda w, s, L, G, r, x, d, **kw: scaled.linear(x, L, **kw),
    "linear of int8 rows": lambda w, s, L, G, r, x, d, **kw: scaled.linear(r, L, out_dtype=torch.float32, **kw),
    "gated": lambda w, s, L, G, r, x, d, **kw: scaled.gated(x, G, **kw),
    "linear_grad": lambda w, s, L, G, r, x, d, **kw: scaled.linear_grad(d, L, **kw),
    "gated_grad": lambda w, s, L, G, r, x, d, **kw: scaled.gated_grad(d, r, G, **kw),
}


def pointers(result):
    if isinstance(result, scaled.QuantRows):
        result = result.data, result.scale
    if isinstance(result, scaled.ScaledWeight):
        result = result.data, result.meta
    return {t.data_ptr() for t in (result if isinstance(result, tuple) else (result,))}


@pytest.mark.parametrize("name", CALLS)
def test_all_work_of_a_call_is_on_its_stream(log, name):
    ops = operands()
    for stream, want in ((None, MAIN), (MAIN, MAIN), (SIDE, SIDE)):
        del log.work[:], log.recorded[:]
        result = CALLS[name](*ops, **({} if stream is None else {"stream": stream}))
        seen = [w for w in log.work if w[0] != "ones"]
        assert any(w[0].startswith("vt_") for w in seen) and {w[1] for w in seen} == {want}, (stream, seen)
        assert log.current == MAIN
        # memory of the side stream's, used on the caller's from here on
        assert {p for p, s in log.recorded if s == MAIN} == (pointers(result) if want == SIDE else set())


def test_a_given_output_is_the_caller_s(log):
    w, s, L, G, r, x, d = operands()
    out = torch.empty(3, 2, N)
    del log.work[:]
    assert scaled.linear(x, L, out=out, stream=SIDE) is out and not log.recorded
    assert {w[1] for w in log.work} == {SIDE}
