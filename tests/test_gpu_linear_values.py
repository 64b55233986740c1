"""Linear layers on the GPU at values where rows or features past a matrix's end could reach a result."""
import pytest
import torch

from chpl_b200 import linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,n", [(5, 300, 40), (77, 1000, 64), (100, 4096, 64), (333, 2048, 130), (2000, 4096, 1024)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_an_infinite_weight_in_the_sum_over_tokens(cuda, T, k, n, dt):
    """With dY > 0 an infinite weight makes its feature's dX and their sum infinite, not NaN, whatever the tile's rows
    past the last token; the other features keep their bits."""
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    dy = torch.rand(T, n, device="cuda", generator=g).add_(0.5).to(dt)
    w = torch.randn(n, k, device="cuda", generator=g).to(dt)
    one = linear.backward(dy, None, w, need_dw=False, need_db=False, dx_sum=True)
    w[n // 2, k // 3], w[n // 3, k - 1] = float("inf"), float("-inf")
    two = linear.backward(dy, None, w, need_dw=False, need_db=False, dx_sum=True)
    for was, now in ((one[0], two[0]), (one[3][None], two[3][None])):
        assert bool((now[:, k // 3] == float("inf")).all()) and bool((now[:, -1] == float("-inf")).all())
        keep = torch.ones(k, dtype=torch.bool, device="cuda")
        keep[k // 3] = keep[k - 1] = False
        assert torch.equal(was[:, keep], now[:, keep])
