"""Which device a call launches on, without a GPU (the fixture and what it stands for: test_scaled_streams_host.py):
the library launches on the current one, so every native call is made with its operands' device current."""
import contextlib

import pytest

torch = pytest.importorskip("torch")

from test_layer_operators_streams_host import CALLS as LAYER, K, N, far, head, here  # noqa: F401
from test_scaled_streams_host import CALLS as SCALED, log, operands  # noqa: F401
from veritac_amd import _lib
from veritac_amd.specializations.hip_gemm import adapters, losses, norms, scaled


class Native:
    """A native library whose calls are counted, and those with another device current than the operands' listed."""

    def __init__(self, under, current):
        self.under, self.current, self.calls, self.astray = under, current, 0, []

    def __getattr__(self, name):
        real = getattr(self.under, name)
        if name in ("vt_quant_pitch", "vt_scaled_size"):    # no device's
            return real

        def call(*args):
            self.calls += 1
            if self.current[-1] != 0:
                self.astray.append(name)
            return real(*args)
        return call


ON = scaled._on


@pytest.fixture
def native(here, monkeypatch):  # noqa: F811
    """Operands are on device 0, and device 1 is current."""
    current = [1]

    @contextlib.contextmanager
    def device(d):
        current.append(torch.device(d).index)
        yield
        current.pop()
    native = Native(_lib.load_library(), current)
    for module in (scaled, norms, losses, adapters):
        monkeypatch.setattr(module, "_on", ON)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[-1], raising=False)
    monkeypatch.setattr(scaled, "_current_device", None, raising=False)
    monkeypatch.setattr(_lib, "load_library", lambda: native)
    yield native
    assert current == [1]


TRAINED = {
    "linear": lambda x: scaled.linear(x, head()), "norm": lambda x: norms.norm(x, torch.ones(K), residual=x)[0],
    "gated": lambda x: scaled.gated(x, operands()[3]), "adapted": lambda x: adapters.adapted(x, head(), (torch.ones(2, 4, K), torch.ones(2, N, 4))),
    "loss": lambda x: losses.cross_entropy(x, head(), torch.zeros(3, 2, dtype=torch.int64)),
}


@pytest.mark.parametrize("name", SCALED)
def test_scaled_calls(native, name):
    SCALED[name](*operands())
    assert native.calls and not native.astray


@pytest.mark.parametrize("name", LAYER)
def test_layer_calls(native, name):
    LAYER[name]()
    assert native.calls and not native.astray


@pytest.mark.parametrize("name", TRAINED)
def test_trained_calls(native, name):
    x = far(K).contiguous().requires_grad_()
    torch.autograd.grad(TRAINED[name](x).sum(), x)
    assert native.calls >= 2 and not native.astray
