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


@pytest.mark.parametrize("T,k,n", [(200003, 40, 72), (70001, 264, 33), (8192, 100, 9000)])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_sums_over_many_tokens(cuda, T, k, n, grad):
    """db and dX's sum of more chunks than a block has warps: an FP32 sum's error of 2^-24 of a partial sum for each of
    a run's terms, of random signs, and the result's rounding."""
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    dy = torch.empty(T, n, device="cuda").normal_(generator=g).bfloat16()
    w = torch.empty(n, k, device="cuda").normal_(0.0, n ** -0.5, generator=g).bfloat16()
    dx, _, db, total = linear.backward(dy, None, w, need_dw=False, grad_dtype=grad, dx_sum=True)
    D = torch.cat([part.double() @ w.double() for part in dy.split(20000)])
    for got, v in ((db, dy.double()), (total, D)):
        want, size = v.sum(0), v.square().sum(0).sqrt()
        lim = 2.0 ** -23 * (n / 16 + T ** 0.5) * size.norm() + (2.0 ** -8 if grad is torch.bfloat16 else 2.0 ** -24) * want.norm()
        assert (got.double() - want).norm() <= lim
    held = [db.clone(), total.clone()]
    linear.backward(dy, None, w, need_dw=False, db=held[0], dx_sum=held[1], grad_dtype=grad, accumulate=True)
    again = linear.backward(dy, None, w, need_dw=False, grad_dtype=grad, dx_sum=True)
    assert torch.equal(again[2], db) and torch.equal(again[3], total) and torch.equal(again[0], dx)
    if grad is torch.float32:
        assert torch.equal(held[0], db + db) and torch.equal(held[1], total + total)
