"""Softmax cross entropy behind an int8 linear layer, without keeping its logits
(include/vt_hip_gemm.h gives the formulas).

    W = scaled.pack_linear(w, s)                      # the head: w int8 [k, n], n classes
    loss = losses.cross_entropy(x, W, target)         # the mean over rows with a target
    loss.backward()                                   # differentiable in x
    losses.cross_entropy(rows, W, target, reduction="none")   # scoring: one loss a row

The loss is that of scaled.linear(x, W)'s logits in 32 bits, and its gradient the
one in the rounded rows, straight through the rounding, with the weights held
constant. Otherwise the conventions are scaled's: rows [..., k], or QuantRows;
work on torch's current stream or on `stream`; every mismatch a HipGemmError
before anything is launched.
"""
from __future__ import annotations

from ... import _lib
from ..._lib import HipGemmError
from . import scaled
from .scaled import _current_stream, _gpu, _on, _pitch, _rows, _torch, _types

REDUCTIONS = tuple(_lib.REDUCE_IDS)


def _targets(target, lead, device):
    """Targets [...] as a contiguous vector, and their VT_TARGET_*."""
    torch = _torch()
    if not isinstance(target, torch.Tensor) or target.dtype not in (torch.int64, torch.int32):
        raise HipGemmError("target must be an int64 or int32 tensor")
    if target.shape != tuple(lead) or target.device != device:
        raise HipGemmError("target must be %s on %s (got %s on %s)"
                           % (tuple(lead), device, tuple(target.shape), target.device))
    return target.reshape(-1).contiguous(), _lib.TARGET_I64 if target.dtype == torch.int64 else _lib.TARGET_I32


def _loss(x, W, target, reduction, ignore_index):
    """(what the gradient needs: a float for the rows' count, three unused, four for
    each row; the loss)."""
    torch = _torch()
    if isinstance(x, scaled.QuantRows):
        data, k, lead = x.data, x.k, tuple(x.shape[:-1])
        _gpu("x", data)
        kind, scale = (_lib.TYPE_I8_PADDED if x.padded else _lib.TYPE_I8), x.scale.data_ptr()
    else:
        data, lead = _rows("x", x)
        k, kind, scale = data.shape[1], _types()[x.dtype], None
    device = data.device
    scaled._check_weight(W, False, device, k)
    if W.n < 1:
        raise HipGemmError("a loss needs at least one class")
    t, t_type = _targets(target, lead, device)
    m = data.shape[0]
    kept = torch.empty(4 + 4 * m, dtype=torch.float32, device=device)
    each = torch.empty(tuple(lead), dtype=torch.float32, device=device)
    loss = each if reduction == "none" else torch.empty((), dtype=torch.float32, device=device)
    with _on(device):
        _lib.check(_lib.load_library().vt_cross_entropy(
            data.data_ptr(), kind, _pitch(data), scale, m, k, W.data.data_ptr(), W.meta.data_ptr(), W.n, t.data_ptr(),
            t_type, ignore_index, each.data_ptr(), kept.data_ptr() + 16, _lib.REDUCE_IDS[reduction], loss.data_ptr(),
            kept.data_ptr(), _current_stream(device)), "vt_cross_entropy")
    return kept, loss


def cross_entropy(x, W, target, *, reduction="mean", ignore_index=-100, stream=None):
    """The loss of rows x [..., k] (floating, or QuantRows) against target [...]
    (int64 or int32), for weights packed by scaled.pack_linear: float32, the mean
    over the rows that have a target, their sum, or (reduction "none") one a row.

    Rows with target ignore_index have loss 0 and no gradient; other targets
    outside 0 .. n - 1 give NaN. Differentiable in floating x.
    """
    if not isinstance(reduction, str) or reduction not in REDUCTIONS:
        raise HipGemmError("reduction must be one of %s (got %r)" % (list(REDUCTIONS), reduction))
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int) or not -2**63 <= ignore_index < 2**63:
        raise HipGemmError("ignore_index must be a 64-bit integer (got %r)" % (ignore_index,))
    if scaled._wants_grad(x):
        if stream is not None:
            raise HipGemmError("a differentiable call takes no stream")
        return _function().apply(x, W, target, reduction, ignore_index)

    def call():
        return _loss(x, W, target, reduction, ignore_index)[1]
    return scaled._enqueued(x if not isinstance(x, scaled.QuantRows) else x.data, stream, call)


_function_class = None


def _function():
    """The autograd function, made on first use: importing this module does not
    import torch."""
    global _function_class
    if _function_class is None:
        torch = _torch()

        class CrossEntropy(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, W, target, reduction, ignore_index):
                rows = scaled._quantize(x)
                kept, loss = _loss(rows, W, target, reduction, ignore_index)
                ctx.W, ctx.dtype, ctx.shape, ctx.reduction = W, x.dtype, rows.shape, reduction
                ctx.save_for_backward(rows.data, rows.scale, kept)
                return loss

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dloss):
                data, scale, kept = ctx.saved_tensors
                m, k, W = data.shape[0], ctx.W.k, ctx.W
                dx = torch.empty((m, k), dtype=ctx.dtype, device=data.device)
                each = ctx.reduction == "none"
                d = dloss.to(torch.float32).reshape(-1).contiguous()
                count = kept.data_ptr() if ctx.reduction == "mean" else None
                with _on(data.device):
                    _lib.check(_lib.load_library().vt_cross_entropy_grad(
                        data.data_ptr(), _lib.TYPE_I8_PADDED, _pitch(data), scale.data_ptr(), m, k, W.data.data_ptr(),
                        W.meta.data_ptr(), W.n, kept.data_ptr() + 16, d.data_ptr(), int(each), count, dx.data_ptr(),
                        _types()[ctx.dtype], max(k, 1), _current_stream(data.device)), "vt_cross_entropy_grad")
                return dx.reshape(ctx.shape), None, None, None, None

        _function_class = CrossEntropy
    return _function_class
