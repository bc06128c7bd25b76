"""Low-rank adapters of many requests beside an int8 linear layer
(include/vt_hip_gemm.h gives the formulas).

    W = scaled.pack_linear(w, s)                            # the shared projection, int8 [k, n]
    A = adapters.pack_adapters(down, up, scaling=0.5)       # down [L, r, k], up [L, n, r]: once, to serve
    y = adapters.adapted(x, W, A, which)                    # row i with adapter which[i], -1 for none

    y = adapters.adapted(x, W, (down, up, 0.5), which)      # to train: as they are now
    y.backward(dy)                                          # differentiable in x, down and up

y = scaled.linear(x, W) + scaling * (x down_a^T) up_a^T, with x as it is given in
the second product (before its rounding to int8, unless it is QuantRows), and
rounded once. `which` is int32 of x's leading shape, or None: every row has
adapter 0. A negative index is no adapter; an index of L or more gives its row
NaN. Adapters, outputs, floating rows and gradients have one type; QuantRows
take adapters of any. A single adapter may be given as down [r, k], up [n, r].

Otherwise the conventions are scaled's: work on torch's current stream or on
`stream`, every mismatch a HipGemmError before anything is launched, a call made
once on a stream can be captured there.
"""
from __future__ import annotations

from ... import _lib
from ..._lib import HipGemmError
from . import scaled
from .scaled import _current_stream, _gpu, _is_int, _on, _pitch, _rows, _torch, _types

MAX_RANK = 128


class Adapters:
    """Adapters laid out for `adapted` (pack_adapters): `count` of a rank for k
    inputs and n outputs, of one floating type, times `scaling`."""

    __slots__ = ("data", "dtype", "count", "rank", "k", "n", "scaling")

    def __init__(self, data, dtype, count, rank, k, n, scaling):
        torch = _torch()
        if dtype not in _types():
            raise HipGemmError("adapters must be float32, float16 or bfloat16 (got %s)" % (dtype,))
        for name, v in (("count", count), ("rank", rank), ("k", k), ("n", n)):
            if not _is_int(v) or not 0 <= v < 1 << 31:      # as far as any size of the library's goes
                raise HipGemmError("%s must be a whole number of 0 .. 2^31 - 1 (got %r)" % (name, v))
        size = _lib.adapter_size(k, n, rank, count, _types()[dtype])
        if not isinstance(data, torch.Tensor) or data.dtype != torch.uint8 or data.shape != (size,) \
                or not data.is_contiguous():
            raise HipGemmError("data must be a contiguous uint8 tensor of %d bytes" % size)
        self.data, self.dtype, self.count, self.rank, self.k, self.n = data, dtype, count, rank, k, n
        self.scaling = _scaling(scaling)

    @property
    def device(self):
        return self.data.device

    def _tensors(self):
        return (self.data,)

    def __repr__(self):
        return "Adapters(%d of rank %d, k=%d, n=%d, %s, device=%s)" % (
            self.count, self.rank, self.k, self.n, self.dtype, self.device)


def _scaling(scaling):
    if isinstance(scaling, bool) or not isinstance(scaling, (int, float)) or not abs(scaling) <= 3.4028234e38:
        raise HipGemmError("scaling must be a number of float32's range (got %.60r)" % (scaling,))
    return float(scaling)


def _pair(down, up):
    """down [L, r, k] and up [L, n, r], checked; a single adapter gets its L."""
    torch = _torch()
    for name, t in (("down", down), ("up", up)):
        if not isinstance(t, torch.Tensor) or t.dtype not in _types() or t.dim() not in (2, 3):
            raise HipGemmError("%s must be a float32, float16 or bfloat16 tensor of 2 or 3 dimensions" % name)
        _gpu(name, t)
    if up.dtype != down.dtype or up.device != down.device or up.dim() != down.dim():
        raise HipGemmError("down is %s %s on %s, up %s %s on %s" % (down.dtype, tuple(down.shape), down.device,
                                                                   up.dtype, tuple(up.shape), up.device))
    if down.dim() == 2:
        down, up = down.unsqueeze(0), up.unsqueeze(0)
    if down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2]:
        raise HipGemmError("down must be [L, r, k] and up [L, n, r] (got %s and %s)" % (tuple(down.shape), tuple(up.shape)))
    if down.shape[0] < 1 or not 1 <= down.shape[1] <= MAX_RANK:
        raise HipGemmError("needs at least one adapter, of a rank of 1 to %d (got %s)" % (MAX_RANK, tuple(down.shape)))
    return down, up


def _layout(down, up, forward, back):
    """The layouts of checked adapters that each direction reads, or None."""
    torch = _torch()
    (count, rank, k), n = down.shape, up.shape[1]
    kind = _types()[down.dtype]
    down, up = down.contiguous(), up.contiguous()
    size = _lib.adapter_size(k, n, rank, count, kind)
    f, b = (torch.empty(size, dtype=torch.uint8, device=down.device) if w else None for w in (forward, back))
    with _on(down.device):
        _lib.check(_lib.load_library().vt_adapter_pack(
            down.data_ptr(), up.data_ptr(), kind, k, n, rank, count, _ptr(f), _ptr(b), _current_stream(down.device)),
            "vt_adapter_pack")
    return f, b


def _ptr(t):
    return None if t is None else t.data_ptr()


def _pack(down, up, scaling):
    down, up = _pair(down.detach(), up.detach())
    return Adapters(_layout(down, up, True, False)[0], down.dtype, down.shape[0], down.shape[1], down.shape[2], up.shape[1], scaling)


def pack_adapters(down, up, *, scaling=1.0, stream=None):
    """Adapters down [L, r, k] and up [L, n, r], laid out once for `adapted`. Not
    differentiable: train with (down, up, scaling) itself."""
    for t in (down, up):
        scaled._constant("pack_adapters", t, "give adapted (down, up, scaling)")
    _pair(down, up)
    scaling = _scaling(scaling)
    return scaled._enqueued(down, stream, lambda: _pack(down, up, scaling))


def _triple(adapters):
    """(down, up, scaling) of adapters that are not packed."""
    if not isinstance(adapters, (tuple, list)) or len(adapters) not in (2, 3):
        raise HipGemmError("adapters must come from pack_adapters, or be (down, up) or (down, up, scaling)")
    _pair(adapters[0], adapters[1])
    return adapters[0], adapters[1], _scaling(adapters[2]) if len(adapters) == 3 else 1.0


def _which(which, lead, device):
    torch = _torch()
    if which is None:
        return None
    if not isinstance(which, torch.Tensor) or which.dtype != torch.int32 or which.shape != tuple(lead) \
            or which.device != device:
        raise HipGemmError("which must be int32 %s on %s" % (tuple(lead), device))
    return which if which.dim() == 1 and which.is_contiguous() else which.reshape(-1).contiguous()


def _fits(A, W, device):
    scaled._check_weight(W, False, device, A.k)
    if A.n != W.n:
        raise HipGemmError("adapters give %d columns, the weights %d" % (A.n, W.n))
    if A.device != device:
        raise HipGemmError("adapters are on %s, rows on %s" % (A.device, device))


def _u(m, rank, device):
    pitch = 16 if rank <= 16 else (rank + 31) // 32 * 32
    return _torch().empty((m, pitch), dtype=_torch().float32, device=device)


def _forward(x, W, A, which, out):
    """(y, u)."""
    if isinstance(x, scaled.QuantRows):
        data, k, lead = x.data, x.k, tuple(x.shape[:-1])
        _gpu("x", data)
        kind, scale = (_lib.TYPE_I8_PADDED if x.padded else _lib.TYPE_I8), x.scale.data_ptr()
    else:
        data, lead = _rows("x", x)
        k, kind, scale = data.shape[1], _types()[x.dtype], None
        if x.dtype != A.dtype:
            raise HipGemmError("adapters are %s, rows %s" % (A.dtype, x.dtype))
    device = data.device
    _fits(A, W, device)
    if k != A.k:
        raise HipGemmError("rows have %d columns, the adapters take %d" % (k, A.k))
    w = _which(which, lead, device)
    m = data.shape[0]
    o2, ret, allocated = scaled._output("output", out, m, W.n, lead, A.dtype, device, data)
    ldy = max(W.n, 1) if allocated or o2.dim() != 2 or m < 2 or not W.n else o2.stride(-2)
    u = _u(m, A.rank, device)
    with _on(device):
        _lib.check(_lib.load_library().vt_adapted_linear(
            data.data_ptr(), kind, _pitch(data), scale, m, k, W.data.data_ptr(), W.meta.data_ptr(), W.n,
            A.data.data_ptr(), A.rank, A.count, A.scaling, None if w is None else w.data_ptr(), u.data_ptr(),
            o2.data_ptr(), _types()[A.dtype], ldy, _current_stream(device)), "vt_adapted_linear")
    return ret, u


def adapted(x, W, adapters, which=None, *, out=None, stream=None):
    """scaled.linear(x, W) plus each row's adapter's part (the module's formula).

    adapters: pack_adapters' result, or (down, up) or (down, up, scaling), which
    are laid out within the call and which it is differentiable in.
    """
    if isinstance(adapters, Adapters):
        scaled._constant("adapted with packed adapters", x, "give (down, up, scaling)")
        down = up = None
        scaling = adapters.scaling
    else:
        wants = scaled._wants_grad(x)
        down, up, scaling = _triple(adapters)
        if any([wants] + [scaled._wants_grad(t) for t in (down, up)]):      # each, for its refusal
            if out is not None or stream is not None:
                raise HipGemmError("a differentiable call takes neither out nor stream")
            if isinstance(x, scaled.QuantRows):
                raise HipGemmError("gradients need floating rows")
            return _function().apply(x, down, up, W, scaling, which)

    def call():
        return _forward(x, W, adapters if down is None else _pack(down, up, scaling), which, out)[0]
    return scaled._enqueued(x.data if isinstance(x, scaled.QuantRows) else x, stream, call, out is None)


def _adapted_grad(dy, x, W, down, up, scaling, which, u, wanted):
    """The gradients in x, down and up that are wanted, as `wanted` says."""
    torch = _torch()
    shapes = down.shape, up.shape
    down, up = _pair(down, up)
    (count, rank, k), n = down.shape, up.shape[1]
    d, lead = _rows("dy", dy)
    device, m = d.device, d.shape[0]
    x2 = None
    if x is not None:
        x2, x_lead = _rows("x", x)
        if x2.device != device or x.dtype != dy.dtype or tuple(x_lead) != tuple(lead):
            raise HipGemmError("x is %s %s on %s, dy %s %s on %s" % (x.dtype, tuple(x.shape), x.device, dy.dtype,
                                                                   tuple(dy.shape), device))
        if x2.shape[1] != k:
            raise HipGemmError("x has %d columns, the adapters take %d" % (x2.shape[1], k))
    if down.dtype != dy.dtype or down.device != device:
        raise HipGemmError("adapters are %s on %s, dy %s on %s" % (down.dtype, down.device, dy.dtype, device))
    scaled._check_weight(W, False, device, k)
    if d.shape[1] != W.n or n != W.n:
        raise HipGemmError("dy has %d columns, the adapters give %d and the weights %d" % (d.shape[1], n, W.n))
    w = _which(which, lead, device)
    kind = _types()[dy.dtype]
    with _on(device):
        again = wanted[2] and u is None     # u as the forward pass makes it
        forward, back = _layout(down, up, again, True)
        u = _u(m, rank, device) if again else u
        h = _u(m, rank, device)
        dx = torch.empty((*lead, k), dtype=dy.dtype, device=device) if wanted[0] else None
        dd = torch.empty(shapes[0], dtype=dy.dtype, device=device) if wanted[1] else None
        du = torch.empty(shapes[1], dtype=dy.dtype, device=device) if wanted[2] else None
        _lib.check(_lib.load_library().vt_adapted_grad(
            d.data_ptr(), kind, _pitch(d), _ptr(x2), 0 if x2 is None else _pitch(x2), m, k, W.data.data_ptr(),
            W.meta.data_ptr(), n, _ptr(forward), back.data_ptr(), rank, count, scaling, _ptr(w), _ptr(u), h.data_ptr(),
            _ptr(dx), max(k, 1), _ptr(dd), _ptr(du), _current_stream(device)), "vt_adapted_grad")
    return dx, dd, du


def adapted_grad(dy, x, W, adapters, which=None, *, stream=None):
    """(dx, ddown, dup): the gradients of `adapted` in x (its int8 product's
    straight through the rounding), down and up, for adapters (down, up) or (down,
    up, scaling) and the x of the forward pass."""
    tensors = adapters[:2] if isinstance(adapters, (tuple, list)) else ()
    for t in (dy, x, *tensors):
        scaled._constant("adapted_grad", t, "there is no second derivative")
    down, up, scaling = _triple(adapters)
    return scaled._enqueued(dy, stream, lambda: _adapted_grad(dy, x, W, down, up, scaling, which, None, (True,) * 3))


_function_class = None


def _function():
    """The autograd function, made on first use: importing this module does not
    import torch."""
    global _function_class
    if _function_class is None:
        torch = _torch()

        class Adapted(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, down, up, W, scaling, which):
                y, u = _forward(x, W, _pack(down, up, scaling), which, None)
                ctx.W, ctx.scaling = W, scaling
                ctx.save_for_backward(x, down, up, which, u)
                return y

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dy):
                x, down, up, which, u = ctx.saved_tensors
                wanted = ctx.needs_input_grad[:3]
                return (*_adapted_grad(scaled._incoming(dy, x.dtype), x if wanted[1] else None, ctx.W, down, up,
                                       ctx.scaling, which, u, wanted), None, None, None)

        _function_class = Adapted
    return _function_class
