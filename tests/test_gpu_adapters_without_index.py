"""Several adapters and no index (needs a gfx950 GPU): every row has adapter 0, and the others' gradients are zeros."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_adapters import KINDS, Case, close
from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import adapters, feed_forward

pytestmark = pytest.mark.gpu


# m of 64 and less sum a gradient's rows at once, more in ranges that are joined
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n,rank,count", [(1, 64, 48, 3, 2), (40, 256, 512, 16, 3), (64, 130, 129, 33, 2), (300, 256, 512, 16, 3),
                                              (700, 100, 300, 128, 5)])
def test_no_index_is_the_first_adapter(dev, m, k, n, rank, count, kind):
    say("no index", m, k, n, rank, count, kind)
    c = Case(m, k, n, rank, count, kind, dev)
    all0 = torch.zeros(m, dtype=torch.int32, device=dev)
    R = c.ref
    R.which = all0.cpu().numpy()
    R.u, R.eu = R._first(R.x, R.down)
    y = adapters.adapted(c.x, c.W, c.triple)
    close(y, R.forward(), "y")
    got = adapters.adapted_grad(c.d, c.x, c.W, c.triple)
    for g, want, other, name in zip(got, R.grad(c.d64, kind == "bf16"), adapters.adapted_grad(c.d, c.x, c.W, c.triple, all0),
                                    ("dx", "ddown", "dup")):
        assert torch.equal(g, other), name
        close(g, want, name)
    assert not got[1][1:].any() and not got[2][1:].any()
    leaves = [t.clone().requires_grad_() for t in (c.x, c.down, c.up)]
    y = adapters.adapted(leaves[0], c.W, (leaves[1], leaves[2], c.scaling))
    for a, b in zip(torch.autograd.grad(y, leaves, c.d), got):
        assert torch.equal(a, b)


def test_a_block_without_an_index_trains_its_first_adapter(dev):
    d, n, rank = 128, 192, 4
    g = torch.Generator().manual_seed(1)
    w = [(torch.randn(a, b, generator=g) / a**0.5).to(dev) for a, b in ((d, n), (d, n), (n, d))]
    down, up = (torch.randn(3, *s, generator=g).to(dev).requires_grad_() for s in ((rank, n), (d, rank)))
    block = feed_forward.FeedForward.from_float(*w, adapters=(down, up, 0.5))
    grads = torch.autograd.grad(block(torch.randn(90, d, generator=g).to(dev)).square().sum(), (down, up))
    for t in grads:
        assert t[0].any() and not t[1:].any()
