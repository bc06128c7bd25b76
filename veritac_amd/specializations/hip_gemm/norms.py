"""Root-mean-square norms in front of the scaled products, with the residual's
addition before them and int8 rows with scales behind (include/vt_hip_gemm.h
gives the formulas).

    y = norms.norm(x, gain)                          # y of x's type
    y, h = norms.norm(x, gain, residual=r)           # h = x + r, y = h / rms(h) * gain
    rows, h = norms.norm_rows(x, gain, residual=r)   # y as scaled.QuantRows, for the products
    dx, dgain = norms.norm_grad(dy, h, gain, dh=dh)  # dx is the gradient of x and of r

h is rounded to x's type and y is the norm of that h. norm is differentiable in
x, the residual and the gain; norm_rows and norm_grad are not, and refuse inputs
whose gradients they would leave out. gain [k] is float32 or of x's type.
Otherwise the conventions are scaled's: rows [..., k] of any pitch and
alignment with unit stride in the last dimension, work on torch's current stream
or on `stream`, every mismatch a HipGemmError before anything is launched.
"""
from __future__ import annotations

from ... import _lib
from ..._lib import HipGemmError
from . import scaled
from .scaled import _current_stream, _on, _pitch, _rows, _torch, _types


def _gain(gain, k, x):
    torch = _torch()
    if not isinstance(gain, torch.Tensor) or gain.dtype not in (torch.float32, x.dtype) or gain.shape != (k,) \
            or (k > 1 and gain.stride(0) != 1):
        raise HipGemmError("gain must be a contiguous tensor [%d], float32 or of the rows' type" % k)
    if gain.device != x.device:
        raise HipGemmError("gain is on %s, rows on %s" % (gain.device, x.device))


def _eps(eps):
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0 <= eps < 3e38:
        raise HipGemmError("eps must be a number of at least 0 (got %r)" % (eps,))
    return float(eps)


def _like(name, t, x, lead):
    """Another operand of x's shape, type and device, as a matrix of rows."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or t.dtype != x.dtype or t.shape != x.shape or t.device != x.device:
        raise HipGemmError("%s must be %s %s on %s, as the rows are" % (name, x.dtype, tuple(x.shape), x.device))
    return _rows(name, t)[0]


def _matrix(name, given, like, lead, k):
    """(matrix to write, tensor to return) of an output of the rows' type."""
    if given is None and len(lead) == 1:
        o2 = like.new_empty((like.shape[0], k))
        return o2, o2
    o2, ret, _ = scaled._output(name, given, like.shape[0], k, lead, like.dtype, like.device, like)
    return (o2 if o2.dim() == 2 else o2.reshape(like.shape[0], k)), ret


def _forward(x, gain, residual, eps, rows, out, h_out):
    torch = _torch()
    x2, lead = _rows("x", x)
    m, k = x2.shape
    _gain(gain, k, x2)
    eps = _eps(eps)
    r2 = None if residual is None else _like("residual", residual, x, lead)
    if residual is None and h_out is not None:
        raise HipGemmError("h_out is the sum of x and a residual")
    h2 = h = None
    if r2 is not None:
        h2, h = _matrix("h", h_out, x2, lead, k)
    if rows:
        pitch = _lib.quant_pitch(k)
        y2 = x2.new_empty((m, pitch), dtype=torch.int8)
        scale = x2.new_empty(m, dtype=torch.float32)
        y = scaled.QuantRows._made(y2, scale, k, (*lead, k))
    else:
        scale = None
        y2, y = _matrix("output", out, x2, lead, k)
    with _on(x2.device):
        _lib.check(_lib.load_library().vt_norm(
            x2.data_ptr(), _pitch(x2), None if r2 is None else r2.data_ptr(), 0 if r2 is None else _pitch(r2),
            _types()[x2.dtype], gain.data_ptr(), _types()[gain.dtype], eps, None if h2 is None else h2.data_ptr(),
            0 if h2 is None else _pitch(h2), y2.data_ptr(), _pitch(y2), None if scale is None else scale.data_ptr(),
            m, k, _current_stream(x2.device)), "vt_norm")
    return y if h is None else (y, h)


def norm(x, gain, *, residual=None, eps=1e-6, out=None, h_out=None, stream=None):
    """x / rms(x) * gain, or with a residual (y, h) of h = x + residual.

    Differentiable in x, residual and gain, then without out, h_out and stream.
    h_out may be the residual itself, which is then replaced by h.
    """
    wants = [scaled._wants_grad(t) for t in (x, gain, residual)]    # each, for its refusal
    if any(wants):
        if out is not None or h_out is not None or stream is not None:
            raise HipGemmError("a differentiable call takes neither out, h_out nor stream")
        y, h = _function().apply(x, gain, residual, eps)
        return y if residual is None else (y, h)
    if stream is None:
        return _forward(x, gain, residual, eps, False, out, h_out)
    given = (() if out is None else (out,)) + (() if h_out is None else (h_out,))
    return scaled._enqueued(x, stream, lambda: _forward(x, gain, residual, eps, False, out, h_out), held=given)


def norm_rows(x, gain, *, residual=None, eps=1e-6, h_out=None, stream=None):
    """norm's y as QuantRows, rounded from its 32-bit values, or with a residual
    (rows, h). Not differentiable: train through norm."""
    for t in (x, gain, residual):
        scaled._constant("norm_rows", t, "train through norm, whose rows linear and gated round for themselves")
    if stream is None:
        return _forward(x, gain, residual, eps, True, None, h_out)
    given = () if h_out is None else (h_out,)
    return scaled._enqueued(x, stream, lambda: _forward(x, gain, residual, eps, True, None, h_out), held=given)


def norm_grad(dy, h, gain, *, dh=None, eps=1e-6, gain_grad=True, stream=None):
    """(dx, dgain) from dy, the h that was normed (x where there was no residual)
    and the gradient dh that reaches h from elsewhere. dx has h's type, dgain
    gain's; dgain is None with gain_grad=False."""
    for t in (dy, h, gain, dh):
        scaled._constant("norm_grad", t, "there is no second derivative")
    return scaled._enqueued(h, stream, lambda: _norm_grad(dy, h, gain, dh, eps, gain_grad))


def _norm_grad(dy, h, gain, dh, eps, gain_grad):
    torch = _torch()
    h2, lead = _rows("h", h)
    m, k = h2.shape
    _gain(gain, k, h2)
    eps = _eps(eps)
    d2 = _like("dy", dy, h, lead)
    e2 = None if dh is None else _like("dh", dh, h, lead)
    x2, dx = _matrix("gradient", None, h2, lead, k)
    dg = torch.empty_like(gain) if gain_grad else None
    with _on(h2.device):
        _lib.check(_lib.load_library().vt_norm_grad(
            d2.data_ptr(), _pitch(d2), h2.data_ptr(), _pitch(h2), None if e2 is None else e2.data_ptr(),
            0 if e2 is None else _pitch(e2), _types()[h2.dtype], gain.data_ptr(), _types()[gain.dtype], eps,
            x2.data_ptr(), _pitch(x2), None if dg is None else dg.data_ptr(), m, k, _current_stream(h2.device)),
            "vt_norm_grad")
    return dx, dg


_function_class = None


def _function():
    """The autograd function, made on first use: importing this module does not
    import torch."""
    global _function_class
    if _function_class is None:
        torch = _torch()

        class Norm(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, gain, residual, eps):
                ctx.eps, ctx.with_h = eps, residual is not None
                ctx.set_materialize_grads(False)
                if residual is None:
                    y, h = _forward(x, gain, None, eps, False, None, None), None
                    ctx.save_for_backward(x, gain)
                else:
                    y, h = _forward(x, gain, residual, eps, False, None, None)
                    ctx.save_for_backward(h, gain)
                return y, h

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dy, dh):
                h, gain = ctx.saved_tensors
                if dy is None and dh is None:
                    return None, None, None, None
                if dy is None:      # only h went on
                    return dh, torch.zeros_like(gain) if ctx.needs_input_grad[1] else None, dh, None
                dx, dg = _norm_grad(scaled._incoming(dy, h.dtype), h, gain,
                                    None if dh is None else scaled._incoming(dh, h.dtype), ctx.eps,
                                    ctx.needs_input_grad[1])
                return (dx if ctx.needs_input_grad[0] else None, dg,
                        dx if ctx.with_h and ctx.needs_input_grad[2] else None, None)

        _function_class = Norm
    return _function_class
