"""Captured blocks' workspaces are nobody else's: blocks replayed beside each other and beside eager calls,
on more streams than torch's pool has."""
import gc

import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import feed_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def block(dev):
    w = [torch.randn(a, b, device=dev) / a**0.5 for a, b in ((512, 1400), (512, 1400), (1400, 512))]
    return feed_forward.FeedForward.from_float(*w)


def test_every_captured_block_has_a_stream_of_its_own(dev, block):
    x = torch.zeros(5, 512, device=dev, dtype=torch.bfloat16)
    steps = [block.capture(x) for _ in range(36)]
    own = {s.stream.cuda_stream for s in steps}
    pool = {torch.cuda.Stream(dev).cuda_stream for _ in range(64)} | {torch.cuda.current_stream(dev).cuda_stream}
    assert len(own) == 36 and not own & pool
    del steps
    gc.collect()
    assert block.capture(x).stream.cuda_stream in own       # and gives it back


@pytest.mark.parametrize("m", [5, 40, 200])
def test_blocks_and_eager_calls_beside_each_other(dev, block, m):
    """K slices of the decode kernels, partial sums and int8 rows all go through workspaces."""
    xs = [torch.randn(m, 512, device=dev, dtype=torch.bfloat16) for _ in range(6)]
    want = [block(x) for x in xs]
    steps = [block.capture(x) for x in xs[:4]]
    streams = [torch.cuda.Stream(dev) for _ in range(33)][-6:]
    torch.cuda.synchronize()
    for i in range(20):
        say("beside each other", m, i)
        eager = []
        for j, step in enumerate(steps):
            with torch.cuda.stream(streams[j]):
                step.replay()
        for j in (4, 5):
            with torch.cuda.stream(streams[j]):
                eager.append(block(xs[j]))
        torch.cuda.synchronize()
        assert all(torch.equal(s.y, y) for s, y in zip(steps, want))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[4:]))
