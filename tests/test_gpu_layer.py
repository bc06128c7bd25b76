"""Norm, feed-forward block with adapters, and loss together, as a layer and its head are served and
trained (needs a gfx950 GPU)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd._lib import HipGemmError
from veritac_amd.specializations.hip_gemm import adapters, feed_forward, losses, norms, scaled

pytestmark = pytest.mark.gpu

D, N, CLASSES, RANK, COUNT = 256, 640, 1003, 8, 3


class Layer:
    def __init__(self, dev, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.w = {n: scaled.quantize_weight((rand(*s) / s[0]**0.5).to(dev))
                  for n, s in (("gate", (D, N)), ("up", (D, N)), ("down", (N, D)), ("head", (D, CLASSES)))}
        self.gate_up = scaled.pack_gated(*self.w["gate"], *self.w["up"])
        self.down, self.head = scaled.pack_linear(*self.w["down"]), scaled.pack_linear(*self.w["head"])
        self.gains = [(1 + 0.2 * rand(D)).to(dev) for _ in range(2)]
        self.a = (rand(COUNT, RANK, N) / N**0.5).to(dev, dtype)
        self.b = (rand(COUNT, D, RANK) * 0.3).to(dev, dtype)


def quantised(z):
    """z's int8 rows' values with z's gradient, in 64 bits."""
    top = z.detach().abs().amax(-1, keepdim=True)
    q = torch.round(z.detach() * 127 / top.clamp_min(1e-300)) * top / 127
    return z + (q - z.detach())


def plain(L, x, r, a, b, gains, which, target):
    """The layer and its loss in 64 bits; weights' gradients straight through the rows' rounding."""
    W = {n: w.double() * s.double() for n, (w, s) in L.w.items()}
    rms = lambda h: h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    h = x + r
    z = quantised(rms(h) * gains[0])
    g = z @ W["gate"]
    u = g * torch.sigmoid(g) * (z @ W["up"])
    y = quantised(u) @ W["down"]
    hot = torch.nn.functional.one_hot(which.clamp_min(0).long(), COUNT).double() * (which >= 0)[:, None]
    t = torch.matmul(u[:, None, None, :], a.transpose(1, 2)[None]).squeeze(2)       # [m, COUNT, RANK]
    y = y + 0.5 * torch.matmul(t[:, :, None, :], b.transpose(1, 2)[None]).squeeze(2).mul(hot[:, :, None]).sum(1)
    logits = quantised(rms(y + h) * gains[1]) @ W["head"]
    has = target >= 0
    loss = torch.logsumexp(logits, 1) - logits.gather(1, target.clamp_min(0)[:, None])[:, 0]
    return (loss * has).sum() / has.sum()


def test_training_step_against_64_bits(dev):
    """Every leaf's gradient of one step in float32. int8 roundings that 32 and 64 bits decide differently are at
    most some 1e-4 of the values, each a step of at most 1/127 of its row's largest, 4 deviations: they leave
    sqrt(1e-4) * 4 / 127 = 3e-4 of the result, over two roundings and the softmax well below 3e-3."""
    L = Layer(dev, torch.float32)
    m = 150
    g = torch.Generator().manual_seed(5)
    x, r = (torch.randn(m, D, generator=g).to(dev) for _ in range(2))
    which = torch.randint(-1, COUNT, (m,), generator=g).to(dev, torch.int32)
    target = torch.randint(0, CLASSES, (m,), generator=g).to(dev)
    target[-9:] = -100
    leaves = [t.clone().requires_grad_() for t in (x, r, L.a, L.b, *L.gains)]
    xs, rs, a, b, g0, g1 = leaves
    block = feed_forward.FeedForward(L.gate_up, L.down, norm=g0, adapters=(a, b, 0.5))
    y, h = block(xs, residual=rs, which=which)
    z, _ = norms.norm(y, g1, residual=h)
    loss = losses.cross_entropy(z, L.head, target)
    got = torch.autograd.grad(loss, leaves)
    exact = [t.detach().double().cpu().requires_grad_() for t in leaves]
    for n, (w, s) in L.w.items():
        L.w[n] = w.cpu(), s.cpu()
    want_loss = plain(L, exact[0], exact[1], exact[2], exact[3], exact[4:], which.cpu(), target.cpu())
    want = torch.autograd.grad(want_loss, exact)
    say("loss", loss.item(), want_loss.item())
    assert abs(loss.item() - want_loss.item()) <= 3e-3 * want_loss.item()
    for name, p, q in zip(("x", "residual", "down", "up", "gain", "last gain"), got, want):
        off = ((p.double().cpu() - q).norm() / q.norm()).item()
        say(name, off)
        assert off <= 3e-3, name


def test_decode_steps_captured(dev):
    """Two captured layers with other batches, replayed in turn beside eager calls, with new indices each time."""
    L = Layer(dev, torch.bfloat16, 1)
    A = adapters.pack_adapters(L.a, L.b, scaling=0.5)
    block = feed_forward.FeedForward(L.gate_up, L.down, norm=L.gains[0], adapters=A)
    steps = []
    for m in (3, 40):
        x, r = (torch.randn(m, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
        steps.append(block.capture(x, residual=r, which=torch.zeros(m, dtype=torch.int32, device=dev)))
    for seed in range(4):
        torch.manual_seed(seed)
        for s in steps:
            s.x.copy_(torch.randn(s.x.shape))
            s.residual.copy_(torch.randn(s.x.shape))
            s.which.copy_(torch.randint(-1, COUNT, s.which.shape))
        for s in steps:
            s.replay()
        torch.cuda.synchronize()
        for s in steps:
            y, h = block(s.x, residual=s.residual, which=s.which)
            assert torch.equal(s.y, y) and torch.equal(s.h, h)


def test_served_rows_are_the_trained_ones(dev):
    """int8 rows of the norm against floating ones that the products round: the adapters and the block in between."""
    L = Layer(dev, torch.float32, 2)
    x, r = torch.randn(33, D, device=dev), torch.randn(33, D, device=dev)
    block = feed_forward.FeedForward(L.gate_up, L.down, norm=L.gains[0], adapters=(L.a, L.b, 0.5))
    which = torch.arange(33, device=dev, dtype=torch.int32) % (COUNT + 1) - 1
    y, h = block(x, residual=r, which=which)
    yt, ht = block(x.clone().requires_grad_(), residual=r, which=which)
    assert torch.equal(h, ht)
    assert ((y - yt).norm() / y.norm()).item() <= 3e-3      # roundings that differ, as above


def test_blocks_refuse_what_they_have_not(dev):
    L = Layer(dev, torch.float32)
    x = torch.randn(4, D, device=dev)
    bare = feed_forward.FeedForward(L.gate_up, L.down)
    for call in (lambda: bare(x, residual=x), lambda: bare(x, which=torch.zeros(4, dtype=torch.int32, device=dev)),
                 lambda: feed_forward.FeedForward(L.gate_up, L.down, norm=L.gains[0][:5]),
                 lambda: feed_forward.FeedForward(L.gate_up, L.down, adapters=L.a)):
        with pytest.raises(HipGemmError):
            call()


def test_the_command_trains_through_all_of_it(dev):
    got = feed_forward.main()
    assert all(np.isfinite(v) for v in got.values())
