"""What packed linear weights keep of their scales for a loss' gradient (needs a gfx950 GPU): the largest magnitude,
in parts that the packing's workgroups find."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_scaled import dev, say  # noqa: F401
from veritac_amd.specializations.hip_gemm import scaled

pytestmark = pytest.mark.gpu


def tops(W):
    return W.meta[-16:]


# fewer workgroups than parts, as many, more; scales of less and more than a part's threads
@pytest.mark.parametrize("k,n", [(0, 1), (64, 48), (64, 200), (128, 64), (300, 129), (1024, 64), (1000, 65), (64, 4096), (64, 5000),
                                 (64, 300000), (2000, 70000)])
def test_the_largest_scale_is_kept(dev, k, n):
    say("largest scale", k, n)
    w = torch.zeros(k, n, dtype=torch.int8, device=dev)
    g = torch.Generator().manual_seed(n)
    for at in (0, n - 1, n // 2, n // 3):
        s = torch.rand(n, generator=g)
        s[at] = -7.5
        s = s.to(dev)
        W = scaled.pack_linear(w, s)
        assert tops(W).max() == 7.5 and (tops(W) >= 0).all()
        s[n // 5] = float("nan")
        assert tops(scaled.pack_linear(w, s)).isnan().any()
