"""GPU: the gradient of the picked gate weights brought back to the logits, against the formula in 64 bits."""
import pytest
import torch

from triton_amd.routing import routing
from triton_amd.tensor import FP32, wrap_torch_tensor
from triton_amd.topk import topk, topk_backward

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def by_formula(x, indx, d, softmax):
    """(dx [T, E], what float32 may be off by) in 64 bits; picks may repeat or be outside."""
    x, d, i = x.double().cpu(), d.double().cpu(), indx.long().cpu()
    there = (i >= 0) & (i < x.shape[1])
    i = torch.where(there, i, 0)
    d = torch.where(there, d, 0.0)
    slack = torch.zeros_like(d)
    if softmax:
        z = torch.where(there, torch.gather(x, 1, i), -torch.inf)
        p = torch.nan_to_num(torch.softmax(z, 1)) * there
        dot = (p * d).sum(1, keepdim=True)
        size = p * (d.abs() + (p * d.abs()).sum(1, keepdim=True))
        # z - max is rounded once, which exp multiplies by its size (up to 60 here); exp is off by 2 half steps, a sum by one for each of its
        # 6 levels, the division by 2: 80 half steps cover p in both of its places, and the products and the difference
        slack = 80 * 2.0 ** -24 * size
        d = p * (d - dot)
    dx, off, k = torch.zeros_like(x), torch.zeros_like(x), i.shape[1]
    dx.scatter_add_(1, i, torch.where(there, d, 0.0))
    off.scatter_add_(1, i, torch.where(there, slack + k * 2.0 ** -24 * d.abs(), 0.0))
    return dx, off


def within(got, want, slack):
    bound = HALF_STEP[got.dtype] * want.abs() * (1 + 2.0 ** -8) + 1.01 * slack + LEAST[got.dtype]
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"off by up to {float((err / bound).max()):.3f} of what rounding allows"


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 128, 4), (3, 5, 5), (77, 60, 6), (1021, 128, 4), (300, 512, 16), (65, 513, 8), (40, 500, 17), (9, 4099, 64), (5, 32767, 33),
                                   (4097, 33, 1)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softmax", [True, False])
def test_formula(T, E, k, dtype, softmax, device):
    torch.manual_seed(T + E)
    x = (3 * torch.randn(T, E, device=device)).to(dtype)
    indx = torch.topk(x.float(), k, dim=1).indices.to(torch.int16)
    d = torch.randn(T, k, device=device)
    for given in (d.to(dtype), d):                     # gate weights' gradients in the logits' type, and in float32
        got = topk_backward(x, indx, given, apply_softmax=softmax)
        assert got.dtype == dtype and got.shape == x.shape
        within(got, *by_formula(x, indx, given, softmax))
        chosen = torch.zeros(T, E, device=device).scatter_(1, indx.long(), 1.0)
        assert not bool(got[chosen == 0].any())
    # other strides and starts
    wide = torch.empty(T, 2 * E + 3, dtype=dtype, device=device)[:, 1:2 * E + 1:2].copy_(x)
    i2, d2 = torch.cat([indx, indx], 1)[:, k:], torch.stack([d, d], 2)[:, :, 1]
    assert torch.equal(topk_backward(wide, i2, d2, apply_softmax=softmax), got)
    assert torch.equal(topk_backward(x, indx.t().contiguous().t(), d, apply_softmax=softmax), got)


def test_gradient_of_topk_by_autograd_and_differences(device):
    torch.manual_seed(0)
    x, d = torch.randn(50, 40, device=device), torch.randn(50, 3, device=device)
    picked = topk(x, 3)
    got = topk_backward(x, picked.indx, d)
    leaf = x.double().cpu().requires_grad_()
    z = torch.gather(leaf, 1, picked.indx.long().cpu())
    (torch.softmax(z, 1) * d.double().cpu()).sum().backward()
    assert float((got.double().cpu() - leaf.grad).abs().max()) < 80 * 2.0 ** -24 * 2 * float(d.abs().max())
    way, step = torch.randn(50, 40, device=device).double(), 2.0 ** -10
    f = lambda x: float((torch.softmax(torch.gather(x, 1, picked.indx.long()), 1) * d.double()).sum())  # noqa: E731
    rise = (f(x.double() + step * way) - f(x.double() - step * way)) / (2 * step)
    assert abs(rise - float((got.double() * way).sum())) < 1e-5 * float((got.double() * way).abs().sum())


def test_of_routing_and_of_live_rows(device):
    torch.manual_seed(1)
    x = torch.randn(64, 32, device=device).bfloat16()
    r = routing(x, 4)
    got = topk_backward(x, r.indx, torch.ones(64, 4, device=device).bfloat16())
    assert float(got.float().abs().max()) < 2.0 ** -20         # (the weights' sum is 1 whatever the logits)
    part = topk(x, 4, n_rows=20)
    d = torch.randn(64, 4, device=device).bfloat16()
    got = topk_backward(x, part.indx, d, n_rows=20)
    assert not bool(got[20:].any()) and torch.equal(got[:20], topk_backward(x[:20], part.indx[:20], d[:20]))
    wrapped = wrap_torch_tensor(x.float(), dtype=FP32, shape=[20, 32], shape_max=[64, 32])
    assert torch.equal(topk_backward(wrapped, part.indx, d.float()), topk_backward(x.float(), part.indx, d.float(), n_rows=20))


def test_picks_outside_and_twice(device):
    x = torch.randn(4, 24, device=device)
    indx = torch.tensor([[0, -1, 5], [24, 32767, -32768], [7, 7, 7], [3, 3, 1]], dtype=torch.int16, device=device)
    d = torch.randn(4, 3, device=device)
    for softmax in (True, False):
        got = topk_backward(x, indx, d, apply_softmax=softmax)
        within(got, *by_formula(x, indx, d, softmax))
        assert not bool(got[1].any()) and int((got[3] != 0).sum()) <= 2


def test_infinite_logits(device):
    """A picked -inf has weight 0 and no gradient; a row of nothing else is NaN at its picks, as its weights are."""
    inf = float("inf")
    x = torch.tensor([[0.0, -inf, 1.0, 2.0], [-inf, -inf, -inf, -inf], [0.0, float("nan"), 1.0, 2.0]], device=device)
    indx = torch.tensor([[3, 1], [0, 1], [3, 2]], dtype=torch.int16, device=device)
    got = topk_backward(x, indx, torch.ones(3, 2, device=device))
    assert bool((got[0] == 0).all()) and torch.equal(torch.isnan(got[1]).cpu(), torch.tensor([True, True, False, False])) and not bool(torch.isnan(got[2]).any())


def test_nothing_there(device):
    for T, E, k in ((0, 8, 2), (3, 0, 0), (3, 8, 0)):
        got = topk_backward(torch.randn(T, E, device=device), torch.zeros(T, k, dtype=torch.int16, device=device), torch.zeros(T, k, device=device))
        assert tuple(got.shape) == (T, E) and not bool(got.any())


def test_another_stream_and_a_graph(device):
    torch.manual_seed(2)
    x, d = torch.randn(64, 128, device=device), torch.randn(64, 4, device=device)
    indx = torch.topk(x, 4, dim=1).indices.to(torch.int16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = topk_backward(x, indx, d)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(mine, topk_backward(x, indx, d))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = topk_backward(x, indx, d)
    for _ in range(4):
        d.copy_(torch.randn(64, 4, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, topk_backward(x, indx, d))
