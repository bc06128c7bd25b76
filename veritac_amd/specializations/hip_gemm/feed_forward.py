"""A gated feed-forward block on int8 weights, with the scaled operators together:
y = (act(x Wg) * (x Wu)) Wd.

    block = FeedForward.from_float(w_gate, w_up, w_down)    # quantised per channel, packed once
    y = block(x)                                            # x [..., d] -> y [..., d]
    step = block.capture(x)                                 # a decode step as a HIP graph
    step.x.copy_(x); step.replay(); step.y

With a norm in front, a residual beside and low-rank adapters on the down
projection, as a layer of a model has them:

    block = FeedForward(gate_up, down, norm=gain, adapters=adapters.pack_adapters(a, b))
    y, h = block(x, residual=r, which=which)                # h = x + r, y = block of norm(h)
    block = FeedForward(gate_up, down, norm=gain, adapters=(a, b, scaling))     # to train a and b

block(x) is differentiable in x with the weights held constant, and in the
residual, the gain and adapters given as (down, up, scaling), which is what
training around a quantised block needs.

`python -m veritac_amd.specializations.hip_gemm.feed_forward` runs a prefill, a
captured decode step and training steps on the GPU, one of them through a norm, a
block with adapters and the loss over an int8 head, and prints how far they are
from the same block in float32.
"""
from __future__ import annotations

import weakref

from ... import _lib
from ..._lib import HipGemmError
from . import adapters as low_rank
from . import losses, norms, scaled
from .backend import _torch


class FeedForward:
    """gate / up packed by scaled.pack_gated and down by scaled.pack_linear; norm: the
    gain [d] of a norm of the rows; adapters: beside down, as adapters.adapted takes
    them."""

    def __init__(self, gate_up, down, act="silu", *, norm=None, eps=1e-6, adapters=None):
        if not isinstance(gate_up, scaled.ScaledWeight) or not gate_up.pair:
            raise HipGemmError("gate_up must come from scaled.pack_gated")
        if not isinstance(down, scaled.ScaledWeight) or down.pair:
            raise HipGemmError("down must come from scaled.pack_linear")
        if down.k != gate_up.n:
            raise HipGemmError("down takes %d columns, the gated product gives %d" % (down.k, gate_up.n))
        if act not in scaled.ACTIVATIONS:
            raise HipGemmError("act must be one of %s (got %r)" % (list(scaled.ACTIVATIONS), act))
        if norm is not None and tuple(getattr(norm, "shape", ())) != (gate_up.k,):
            raise HipGemmError("norm must be a gain of %d columns" % gate_up.k)
        if adapters is not None and not isinstance(adapters, low_rank.Adapters):
            low_rank._triple(adapters)
        self.gate_up, self.down, self.act = gate_up, down, act
        self.norm, self.eps, self.adapters = norm, eps, adapters

    @classmethod
    def from_float(cls, w_gate, w_up, w_down, act="silu", **more):
        """From floating weights [d, n], [d, n] and [n, d] on a GPU."""
        return cls(scaled.pack_gated(*scaled.quantize_weight(w_gate), *scaled.quantize_weight(w_up)),
                   scaled.pack_linear(*scaled.quantize_weight(w_down)), act, **more)

    def __call__(self, x, *, residual=None, which=None):
        """y, or with a residual (y, x + residual). which: the rows' adapters."""
        rows, h = x, None
        if self.norm is not None:
            trains = any([scaled._wants_grad(t) for t in (x, residual, self.norm)])
            make = norms.norm if trains else norms.norm_rows    # int8 rows need no floating ones
            rows = make(x, self.norm, residual=residual, eps=self.eps)
            if residual is not None:
                rows, h = rows
        elif residual is not None:
            raise HipGemmError("a residual needs the block's norm")
        u = scaled.gated(rows, self.gate_up, act=self.act, out_dtype=None if rows is x else x.dtype)
        if self.adapters is not None:
            y = low_rank.adapted(u, self.down, self.adapters, which)
        elif which is not None:
            raise HipGemmError("the block has no adapters")
        else:
            y = scaled.linear(u, self.down)
        return y if h is None else (y, h)

    def capture(self, x, *, residual=None, which=None):
        """The block on rows like x as a HIP graph: an object with static `x`, `y`
        and (if given here) `residual`, `h` and `which`, and replay(), with
        workspaces of its own, which are made here."""
        return _CapturedBlock(self, x, residual, which)


# Streams that no captured block uses any more, by device index. The library
# keeps workspaces by stream handle: a block's stream is neither torch's (whose
# pool hands out each of 32 handles again and again) nor another block's, so
# replays and eager calls may run beside each other on any streams.
_free_streams = {}


def _own_stream(device, owner):
    """A stream for `owner` alone, back among the free ones when it is gone."""
    torch = _torch()
    free = _free_streams.setdefault(device.index, [])
    with torch.cuda.device(device):
        try:
            handle = free.pop()
            torch.cuda.synchronize(device)      # what its last owner enqueued
        except IndexError:
            handle = _lib.stream_create()
    weakref.finalize(owner, free.append, handle)
    return torch.cuda.ExternalStream(handle, device=device)


class _CapturedBlock:
    def __init__(self, block, x, residual, which):
        torch = _torch()
        self.x = x.detach().clone()
        self.residual = None if residual is None else residual.detach().clone()
        self.which = None if which is None else which.clone()
        self.graph = torch.cuda.CUDAGraph()
        self.stream = _own_stream(x.device, self.graph)
        plain = block.norm is None and block.adapters is None and residual is None and which is None
        if plain:
            self.h = torch.empty((*x.shape[:-1], block.gate_up.n), dtype=x.dtype, device=x.device)
            self.y = torch.empty((*x.shape[:-1], block.down.n), dtype=x.dtype, device=x.device)

        def step():
            if plain:
                scaled.gated(self.x, block.gate_up, act=block.act, out=self.h)
                scaled.linear(self.h, block.down, out=self.y)
                return
            out = block(self.x, residual=self.residual, which=self.which)
            self.y, self.h = (out, None) if residual is None else out

        self.stream.wait_stream(torch.cuda.current_stream(x.device))
        with torch.no_grad():
            with torch.cuda.stream(self.stream):    # the workspaces, before the capture
                step()
            with torch.cuda.graph(self.graph, stream=self.stream):
                step()
        # what the graph reads is used on its stream
        self.block = block

    def replay(self):
        """Enqueues the step on torch's current stream; y is ready in its order.
        Replays of one block share its x, y and workspaces: order them."""
        self.graph.replay()
        return self.y


def main():
    torch = _torch()
    torch.manual_seed(0)
    dev = torch.device("cuda", torch.cuda.current_device())
    d, n = 1024, 2816
    w = [torch.randn(a, b, device=dev) / a**0.5 for a, b in ((d, n), (d, n), (n, d))]
    block = FeedForward.from_float(*w)

    def plain(x):
        g = x @ w[0]
        return (g * torch.sigmoid(g) * (x @ w[1])) @ w[2]

    def off(a, b):
        return ((a.float() - b.float()).norm() / b.float().norm()).item()

    x = torch.randn(3, 200, d, device=dev, dtype=torch.bfloat16)
    print("prefill of 3 x 200 tokens: %.3f off float32" % off(block(x), plain(x.float())), flush=True)

    step = block.capture(x[:, 0])
    step.x.copy_(x[:, 7])
    step.replay()
    torch.cuda.synchronize(dev)
    print("captured decode step of 3 tokens: %.3f off float32" % off(step.y, plain(x[:, 7].float())), flush=True)

    # An adapter in front of the block: a bias that learns to undo an offset of its input.
    bias = torch.zeros(d, device=dev, requires_grad=True)
    opt = torch.optim.Adam([bias], lr=0.02)
    xs = torch.randn(512, d, device=dev)
    offset = torch.randn(d, device=dev) * 0.3
    with torch.no_grad():
        target = block(xs)
    first = last = None
    for _ in range(60):
        loss = (block(xs + offset + bias) - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        last = loss.item()
        first = last if first is None else first
    print("adapter through the block: loss %.2e -> %.2e in 60 steps" % (first, last), flush=True)

    # Low-rank adapters on the down projection and the norms' gains, trained on a
    # batch's next tokens through the norm, the block and the loss over an int8 head.
    classes, rank = 5003, 8
    head = scaled.pack_linear(*scaled.quantize_weight(torch.randn(d, classes, device=dev) / d**0.5))
    learnt = [torch.randn(1, rank, n, device=dev) / n**0.5, torch.zeros(1, d, rank, device=dev),
              torch.ones(d, device=dev), torch.ones(d, device=dev)]
    for t in learnt:
        t.requires_grad_()
    layer = FeedForward(block.gate_up, block.down, norm=learnt[2], adapters=(learnt[0], learnt[1], 2.0))
    opt = torch.optim.Adam(learnt, lr=3e-3)
    r, target = torch.randn(512, d, device=dev), torch.randint(0, classes, (512,), device=dev)
    target[-7:] = -100                      # padding
    start = end = None
    for _ in range(30):
        y, h = layer(xs, residual=r)
        z, _ = norms.norm(y, learnt[3], residual=h)
        loss = losses.cross_entropy(z, head, target)
        opt.zero_grad()
        loss.backward()
        opt.step()
        end = loss.item()
        start = end if start is None else start
    print("adapters and gains through the loss: %.3f -> %.3f in 30 steps" % (start, end), flush=True)
    return {"prefill": off(block(x), plain(x.float())), "decode": off(step.y, plain(x[:, 7].float())),
            "loss_first": first, "loss_last": last, "adapters_first": start, "adapters_last": end}


if __name__ == "__main__":
    main()
