"""Scaled int8 operators: linear layers and gated feed-forward products on int8
weights with a scale for each output channel and int8 rows with a scale for
each token, and their input gradients (include/vt_hip_gemm.h gives the
formulas).

    W = scaled.pack_linear(w, s)                 # w int8 [k, n], s float32 [n]: once per weight
    y = scaled.linear(x, W)                      # x [..., k] float -> y [..., n] of x's type

    G = scaled.pack_gated(w_gate, s_gate, w_up, s_up)
    h = scaled.gated(x, G, act="silu")           # silu(gate(x)) * up(x)

    r = scaled.quantize_rows(x)                  # int8 rows and their scales, for several products
    q, k = scaled.linear(r, Wq, out_dtype=x.dtype), scaled.linear(r, Wk, out_dtype=x.dtype)

x may require gradients: linear and gated are then differentiable in it, with
the rounding to int8 passed straight through (the gradient is the one in the
rounded rows) and weights, scales and bias held constant. gated keeps its int8
rows for that, not the two products. linear_grad and gated_grad are those
gradients by themselves. Nothing else is differentiable: quantize_rows (so
training goes through floating rows, which each product rounds for itself),
the two gradients and forward mode raise HipGemmError rather than leave a
gradient out.

Same conventions as backend.run: device tensors only, every mismatch raises
HipGemmError before anything is launched, work is enqueued on torch's current
stream or on `stream` (a raw hipStream_t handle, whose order against the
operands' producers is the caller's; what a call allocates and copies itself is
on that stream too), and a call made once on a stream can be captured into a
HIP graph there. Rows may have any pitch and alignment; their last dimension
has unit stride.
"""
from __future__ import annotations

import math

from ... import _lib
from ..._lib import HipGemmError
from .backend import _current_stream, _is_int, _torch

ACTIVATIONS = tuple(_lib.ACT_IDS)

_type_ids = {}


def _types():
    if not _type_ids:
        torch = _torch()
        _type_ids.update({torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16,
                          torch.bfloat16: _lib.TYPE_BF16})
    return _type_ids


class QuantRows:
    """int8 rows and their scales: row i stands for data[i, :k] * scale[i].

    `data` is int8 [m, >= k] and `scale` float32 [m], both on one GPU. Rows
    made by quantize_rows are padded with zeros to the pitch that the products
    read in place (`padded`); others are copied so by the calls that need it.
    `shape`: what the rows were flattened from, [..., k] of m rows in all.
    """

    __slots__ = ("data", "scale", "k", "padded", "shape")

    def __init__(self, data, scale, *, k=None, padded=False, shape=None):
        torch = _torch()
        if not isinstance(data, torch.Tensor) or data.dtype != torch.int8 or data.dim() != 2:
            raise HipGemmError("data must be an int8 tensor [m, k]")
        if not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 \
                or scale.shape != data.shape[:1] or not scale.is_contiguous():
            raise HipGemmError("scale must be a contiguous float32 tensor [m]")
        if scale.device != data.device:
            raise HipGemmError("scale is on %s, data on %s" % (scale.device, data.device))
        if not _unit_rows(data):
            raise HipGemmError("data must have unit stride in its last dimension")
        m, width = data.shape
        if k is None:
            k = width
        elif not _is_int(k) or not 0 <= k <= width:
            raise HipGemmError("k must be 0 .. %d, the width of data (got %r)" % (width, k))
        if padded and width < _lib.quant_pitch(k):
            raise HipGemmError("padded rows of k = %d are at least %d wide (got %d)"
                               % (k, _lib.quant_pitch(k), width))
        shape = (m, k) if shape is None else tuple(shape)
        if not shape or not all(_is_int(d) and d >= 0 for d in shape) or shape[-1] != k \
                or math.prod(shape[:-1]) != m:
            raise HipGemmError("shape must be [..., %d] of %d rows (got %s)" % (k, m, shape))
        self.data, self.scale, self.k, self.padded, self.shape = data, scale, k, padded, shape

    @property
    def device(self):
        return self.data.device

    def dequantize(self):
        """The rows as float32 [..., k]."""
        return (self.data[:, :self.k].float() * self.scale[:, None]).reshape(self.shape)

    def __repr__(self):
        return "QuantRows(m=%d, k=%d, device=%s)" % (self.data.shape[0], self.k, self.device)


class ScaledWeight:
    """int8 weights packed for `linear` (pack_linear) or `gated` (pack_gated).

    `data` is the packed int8 matrix and `meta` its scales and bias
    (vt_scaled_pack's layout); k inputs, n outputs.
    """

    __slots__ = ("data", "meta", "k", "n", "pair")

    def __init__(self, data, meta, k, n, pair):
        torch = _torch()
        size, floats = _lib.scaled_size(k, n, pair)
        if not isinstance(data, torch.Tensor) or data.dtype != torch.int8 or data.shape != (size,) \
                or not data.is_contiguous():
            raise HipGemmError("data must be a contiguous int8 tensor of %d bytes" % size)
        if not isinstance(meta, torch.Tensor) or meta.dtype != torch.float32 or meta.shape != (floats,) \
                or not meta.is_contiguous() or meta.device != data.device:
            raise HipGemmError("meta must be a contiguous float32 tensor [%d] on %s" % (floats, data.device))
        self.data, self.meta, self.k, self.n, self.pair = data, meta, k, n, pair

    @property
    def device(self):
        return self.data.device

    def __repr__(self):
        return "ScaledWeight(k=%d, n=%d, %s, device=%s)" % (
            self.k, self.n, "gated" if self.pair else "linear", self.device)


def _enqueued(on, stream, call, record=True):
    """call(), with the raw handle `stream` as torch's current stream of the device
    of `on`: the copies and memory that the call makes on its way are then in
    order with its kernels. Its results (unless the caller holds them already)
    are recorded as used on the stream that was current, where the caller goes
    on with them."""
    device = getattr(on, "device", None)
    if stream is None or getattr(device, "type", None) != "cuda":
        return call()
    torch = _torch()
    with torch.cuda.device(device):
        before = torch.cuda.current_stream(device)
        if stream == before.cuda_stream:
            return call()
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
            result = call()
        if record:
            for t in _tensors(result):
                t.record_stream(before)
        return result


def _tensors(result):
    if isinstance(result, QuantRows):
        return result.data, result.scale
    if isinstance(result, ScaledWeight):
        return result.data, result.meta
    return result if isinstance(result, tuple) else (result,)


def _gpu(name, t):
    if t.device.type != "cuda":
        raise HipGemmError("%s must be on a gfx950 GPU (got %s); hip_gemm has no CPU path"
                           % (name, t.device))


def _weight(name, w, s, shape=None, device=None):
    torch = _torch()
    if not isinstance(w, torch.Tensor) or w.dtype != torch.int8 or w.dim() != 2:
        raise HipGemmError("%s must be an int8 torch tensor [k, n]" % name)
    _gpu(name, w)
    if shape is not None and w.shape != shape:
        raise HipGemmError("%s has shape %s, expected %s" % (name, tuple(w.shape), tuple(shape)))
    if not _unit_rows(w):
        raise HipGemmError("%s must have unit stride in its last dimension" % name)
    _channels("scale of " + name, s, w.shape[1], w.device)
    if device is not None and w.device != device:
        raise HipGemmError("%s is on %s, expected %s" % (name, w.device, device))


def _channels(name, s, n, device):
    torch = _torch()
    if not isinstance(s, torch.Tensor) or s.dtype != torch.float32 or s.shape != (n,) \
            or (n > 1 and s.stride(0) != 1):
        raise HipGemmError("%s must be a contiguous float32 tensor [%d]" % (name, n))
    if s.device != device:
        raise HipGemmError("%s is on %s, expected %s" % (name, s.device, device))


def _unit_rows(t):
    """Whether a matrix' rows have unit stride (empty ones and single columns do)."""
    return t.stride(1) == 1 or t.shape[1] <= 1 or t.shape[0] == 0


def _pitch(t):
    """Elements from one row to the next (a lone row has no next one)."""
    return t.stride(0) if t.shape[0] > 1 and t.shape[1] else max(t.shape[1], 1)


def _pack(w0, s0, w1, s1, bias):
    torch = _torch()
    k, n = w0.shape
    size, floats = _lib.scaled_size(k, n, w1 is not None)
    data = torch.empty(size, dtype=torch.int8, device=w0.device)
    meta = torch.empty(floats, dtype=torch.float32, device=w0.device)   # written whole (and not read if n = 0)
    lib = _lib.load_library()
    _lib.check(lib.vt_scaled_pack(
        w0.data_ptr(), None if w1 is None else w1.data_ptr(), _pitch(w0),
        0 if w1 is None else _pitch(w1), s0.data_ptr(), None if s1 is None else s1.data_ptr(),
        None if bias is None else bias.data_ptr(), k, n, data.data_ptr(), meta.data_ptr(),
        _current_stream(w0.device)), "vt_scaled_pack")
    return ScaledWeight(data, meta, k, n, w1 is not None)


def pack_linear(w, scale, bias=None, *, stream=None):
    """int8 weights [k, n], their channel scales float32 [n] and an optional
    float32 bias [n], packed once for `linear` and `linear_grad`."""
    _weight("w", w, scale)
    if bias is not None:
        _channels("bias", bias, w.shape[1], w.device)
    return _enqueued(w, stream, lambda: _pack(w, scale, None, None, bias))


def pack_gated(w_gate, s_gate, w_up, s_up, *, stream=None):
    """The gate and up projections of a gated feed-forward block, int8 [k, n]
    each with channel scales float32 [n], packed once for `gated` and
    `gated_grad`."""
    _weight("w_gate", w_gate, s_gate)
    _weight("w_up", w_up, s_up, w_gate.shape, w_gate.device)
    return _enqueued(w_gate, stream, lambda: _pack(w_gate, s_gate, w_up, s_up, None))


def quantize_weight(w, *, stream=None):
    """Floating weights [k, n] -> (int8 [k, n], channel scales float32 [n]): each
    channel by its largest magnitude, as quantize_rows treats a row."""
    torch = _torch()
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        raise HipGemmError("w must be a floating torch tensor [k, n]")

    def both():
        r = _quantize(w.detach().t().contiguous())
        return r.data[:, :r.k].t().contiguous(), r.scale
    return _enqueued(w, stream, both)


def _rows(name, x):
    """x [..., k] as (a matrix of unit-stride rows, its leading shape)."""
    torch = _torch()
    # Contiguous matrices on a GPU, the usual call, need no more than this.
    if type(x) is torch.Tensor and x.is_cuda and x.dtype in _types() and x.dim() == 2 and x.is_contiguous():
        return x, x.shape[:1]
    if not isinstance(x, torch.Tensor) or x.dtype not in _types():
        raise HipGemmError("%s must be a float32, float16 or bfloat16 torch tensor" % name)
    if x.dim() < 1:
        raise HipGemmError("%s must have at least one dimension" % name)
    _gpu(name, x)
    if x.dim() != 2:
        if x.numel() == 0:
            m = 1
            for d in x.shape[:-1]:
                m *= d
            return x.reshape(m, x.shape[-1]), x.shape[:-1]
        lead, x = x.shape[:-1], x.flatten(0, -2) if x.dim() > 2 else x.unsqueeze(0)
    else:
        lead = x.shape[:-1]
    if not _unit_rows(x):
        raise HipGemmError("%s must have unit stride in its last dimension" % name)
    if x.shape[0] > 1 and x.numel() and x.stride(0) < x.shape[1]:
        raise HipGemmError("%s has overlapping rows" % name)
    return x, lead


def quantize_rows(x, *, stream=None):
    """Floating rows x [..., k] -> QuantRows: each row by its largest magnitude,
    rounded to the nearest, ties to even. Not differentiable: train through
    floating rows, which linear and gated take as they are."""
    _constant("quantize_rows", x, "give linear and gated the floating rows")
    return _enqueued(x, stream, lambda: _quantize(x))


def _quantize(x):
    torch = _torch()
    x2, lead = _rows("x", x)
    m, k = x2.shape
    pitch = _lib.quant_pitch(k)
    data = torch.empty((m, pitch), dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    lib = _lib.load_library()
    _lib.check(lib.vt_quant_rows(x2.data_ptr(), _types()[x.dtype], _pitch(x2), data.data_ptr(), pitch,
                                 scale.data_ptr(), m, k, _current_stream(x.device)), "vt_quant_rows")
    return QuantRows(data, scale, k=k, padded=True, shape=tuple(lead) + (k,))


def _check_weight(W, pair, device, k):
    if not isinstance(W, ScaledWeight) or W.pair != pair:
        raise HipGemmError("weights must be packed by %s (got %s)"
                           % ("pack_gated" if pair else "pack_linear",
                              W if isinstance(W, ScaledWeight) else type(W).__name__))
    if W.data.device != device:
        raise HipGemmError("weights are on %s, rows on %s" % (W.data.device, device))
    if k is not None and k != W.k:
        raise HipGemmError("rows have %d columns, the weights take %d" % (k, W.k))


def _output(name, out, m, cols, lead, dtype, device, like=None):
    """(matrix to write, tensor to return, whether it was allocated here). `like`:
    a tensor on the device, whose new_empty takes less time where the type is its."""
    torch = _torch()
    if out is None and like is not None and like.dtype is dtype:
        out = like.new_empty((*lead, cols))
        return out, out, True
    if dtype not in _types():
        raise HipGemmError("%s type must be float32, float16 or bfloat16 (got %s)" % (name, dtype))
    if out is None:
        out = torch.empty((*lead, cols), dtype=dtype, device=device)
        return out, out, True
    if not isinstance(out, torch.Tensor) or out.dtype != dtype or out.device != device \
            or out.shape != (*lead, cols):
        raise HipGemmError("out must be %s %s on %s" % (dtype, (*lead, cols), device))
    o2 = out
    if out.dim() != 2:
        try:
            o2 = out.view(m, cols)
        except RuntimeError:
            raise HipGemmError("out must be viewable as [%d, %d]" % (m, cols)) from None
    if not _unit_rows(o2) or (m > 1 and o2.numel() and o2.stride(0) < cols):
        raise HipGemmError("out must have unit stride in its last dimension and rows that do not overlap")
    return o2, out, False


def _forward(x, W, pair, act, out_dtype, out):
    if out is not None and not isinstance(out, _torch().Tensor):
        raise HipGemmError("out must be a torch tensor (got %s)" % type(out).__name__)
    if isinstance(x, QuantRows):
        data, k = x.data, x.k
        _gpu("x", data)
        _check_weight(W, pair, data.device, k)
        if out_dtype is None:
            if out is None:
                raise HipGemmError("int8 rows need out_dtype (or out)")
            out_dtype = out.dtype
        lead = tuple(x.shape[:-1])
        kind, scale = (_lib.TYPE_I8_PADDED if x.padded else _lib.TYPE_I8), x.scale.data_ptr()
    else:
        data, lead = _rows("x", x)
        k = data.shape[1]
        _check_weight(W, pair, data.device, k)
        kind, scale = _types()[x.dtype], None
        if out_dtype is None:
            out_dtype = x.dtype if out is None else out.dtype
    m = data.shape[0]
    device = data.device
    o2, ret, allocated = _output("output", out, m, W.n, lead, out_dtype, device, data)
    stream = _current_stream(device)
    lib = _lib.load_library()
    ldy = max(W.n, 1) if allocated or o2.dim() != 2 or m < 2 or not W.n else o2.stride(-2)
    if pair:
        _lib.check(lib.vt_scaled_gated(data.data_ptr(), kind, _pitch(data), scale, m, k,
                                       W.data.data_ptr(), W.meta.data_ptr(), W.n, act,
                                       o2.data_ptr(), _types()[out_dtype], ldy, stream),
                   "vt_scaled_gated")
    else:
        _lib.check(lib.vt_scaled_linear(data.data_ptr(), kind, _pitch(data), scale, m, k,
                                        W.data.data_ptr(), W.meta.data_ptr(), W.n,
                                        o2.data_ptr(), _types()[out_dtype], ldy, stream),
                   "vt_scaled_linear")
    return ret


_forward_ad = None      # torch.autograd.forward_ad, from the first call on


def _wants_grad(x):
    global _forward_ad
    requires = getattr(x, "requires_grad", None)
    if requires is None:        # not a tensor
        return False
    if _forward_ad is None:
        _forward_ad = _torch().autograd.forward_ad
    # outside of its levels nothing has a tangent (asking for one takes 0.3 us)
    if getattr(_forward_ad, "_current_level", 0) >= 0 and _forward_ad.unpack_dual(x).tangent is not None:
        raise HipGemmError("the scaled operators have no forward-mode derivative")
    return requires and _torch().is_grad_enabled()


def _constant(name, x, instead):
    """Refuses an input whose gradient would be left out silently."""
    if _wants_grad(x):
        raise HipGemmError("%s passes no gradient on to its input: %s, or detach it" % (name, instead))


def _act_id(act):
    if not isinstance(act, str) or act not in _lib.ACT_IDS:
        raise HipGemmError("act must be one of %s (got %r)" % (list(ACTIVATIONS), act))
    return _lib.ACT_IDS[act]


def linear(x, W, *, out_dtype=None, out=None, stream=None):
    """y = x^ . (w * scale) + bias for weights packed by pack_linear.

    x: floating rows [..., k], rounded to int8 with a scale each, or QuantRows.
    The result [..., n] has x's type unless out_dtype or out says otherwise.
    """
    if _wants_grad(x):
        if out is not None or stream is not None:
            raise HipGemmError("a differentiable call takes neither out nor stream")
        return _functions()[0].apply(x, W, out_dtype)
    if stream is not None:
        return _enqueued(x, stream, lambda: _forward(x, W, False, 0, out_dtype, out), out is None)
    return _forward(x, W, False, 0, out_dtype, out)


def gated(x, W, *, act="silu", out_dtype=None, out=None, stream=None):
    """h = act(x^ . (w_gate * s_gate)) * (x^ . (w_up * s_up)) for weights packed
    by pack_gated; act is "silu" or "gelu" (its tanh form). Otherwise as linear.
    """
    a = _act_id(act)
    if _wants_grad(x):
        if out is not None or stream is not None:
            raise HipGemmError("a differentiable call takes neither out nor stream")
        return _functions()[1].apply(x, W, act, out_dtype)
    if stream is not None:
        return _enqueued(x, stream, lambda: _forward(x, W, True, a, out_dtype, out), out is None)
    return _forward(x, W, True, a, out_dtype, out)


def linear_grad(dy, W, *, out=None, stream=None):
    """dx = (dy * scale) . w^T, the gradient of `linear` in its rounded rows, for
    dy [..., n] of any floating type; dx [..., k] has the same."""
    _constant("linear_grad", dy, "there is no second derivative")
    return _enqueued(dy, stream, lambda: _linear_grad(dy, W, out), out is None)


def _linear_grad(dy, W, out):
    d, lead = _rows("dy", dy)
    _check_weight(W, False, d.device, None)
    if d.shape[1] != W.n:
        raise HipGemmError("dy has %d columns, the weights give %d" % (d.shape[1], W.n))
    m = d.shape[0]
    o2, ret, _ = _output("gradient", out, m, W.k, lead, dy.dtype, d.device, d)
    ldx = o2.stride(-2) if o2.dim() == 2 and m > 1 and W.k else max(W.k, 1)
    lib = _lib.load_library()
    _lib.check(lib.vt_scaled_linear_grad(d.data_ptr(), _types()[dy.dtype], _pitch(d), m, W.k,
                                         W.data.data_ptr(), W.meta.data_ptr(), W.n, o2.data_ptr(),
                                         ldx, _current_stream(d.device)), "vt_scaled_linear_grad")
    return ret


def gated_grad(dh, rows, W, *, act="silu", out=None, stream=None):
    """The gradient of `gated` in its rounded rows, from dh [..., n] and the
    QuantRows of the forward pass (quantize_rows of its x). dx [..., k] has dh's
    type."""
    a = _act_id(act)
    _constant("gated_grad", dh, "there is no second derivative")
    return _enqueued(dh, stream, lambda: _gated_grad(dh, rows, W, a, out), out is None)


def _gated_grad(dh, rows, W, a, out):
    d, lead = _rows("dh", dh)
    if not isinstance(rows, QuantRows):
        raise HipGemmError("rows must be the QuantRows of the forward pass")
    _check_weight(W, True, d.device, rows.k)
    if rows.device != d.device:
        raise HipGemmError("rows are on %s, dh on %s" % (rows.device, d.device))
    m = d.shape[0]
    if d.shape[1] != W.n or m != rows.data.shape[0]:
        raise HipGemmError("dh is %d x %d, the rows and weights give %d x %d"
                           % (m, d.shape[1], rows.data.shape[0], W.n))
    o2, ret, _ = _output("gradient", out, m, W.k, lead, dh.dtype, d.device, d)
    ldx = o2.stride(-2) if o2.dim() == 2 and m > 1 and W.k else max(W.k, 1)
    lib = _lib.load_library()
    _lib.check(lib.vt_scaled_gated_grad(
        d.data_ptr(), _types()[dh.dtype], _pitch(d), rows.data.data_ptr(),
        _lib.TYPE_I8_PADDED if rows.padded else _lib.TYPE_I8, _pitch(rows.data),
        rows.scale.data_ptr(), m, W.k, W.data.data_ptr(), W.meta.data_ptr(), W.n, a, o2.data_ptr(),
        ldx, _current_stream(d.device)), "vt_scaled_gated_grad")
    return ret


_function_classes = None


def _functions():
    """(linear, gated) as autograd functions, made on first use: importing this
    module does not import torch."""
    global _function_classes
    if _function_classes is None:
        torch = _torch()

        class Linear(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, W, out_dtype):
                ctx.W, ctx.dtype = W, x.dtype
                return _forward(x, W, False, 0, out_dtype, None)

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dy):
                dx = linear_grad(_incoming(dy, ctx.dtype), ctx.W)
                return dx.to(ctx.dtype), None, None

        class Gated(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, W, act, out_dtype):
                rows = _quantize(x)
                ctx.W, ctx.act, ctx.dtype, ctx.shape = W, act, x.dtype, rows.shape
                ctx.save_for_backward(rows.data, rows.scale)
                return _forward(rows, W, True, _act_id(act), out_dtype or x.dtype, None)

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dh):
                data, scale = ctx.saved_tensors
                rows = QuantRows(data, scale, k=ctx.W.k, padded=True, shape=ctx.shape)
                dx = gated_grad(_incoming(dh, ctx.dtype), rows, ctx.W, act=ctx.act)
                return dx.to(ctx.dtype), None, None, None

        _function_classes = Linear, Gated
    return _function_classes


def _incoming(d, dtype):
    """An incoming gradient as rows (autograd may hand a broadcast or transposed
    one), of a type that holds both its values and the gradient of `dtype` that
    is made of them: an output of fewer bits or less range than x takes neither
    from x's gradient."""
    if d.dtype != dtype:
        d = d.to(_torch().promote_types(d.dtype, dtype))
    if d.dim() and (d.stride(-1) != 1 or not d.is_contiguous()):
        return d.contiguous()
    return d
