"""GPU: every form that the kernels of `dispatch`, `combine` and their gradients take by the size of a call, against the formulas in 64 bits: 16, 64 and 256 lanes to
a token, rows through the caches and past them, rows of whole 16-byte pieces and others, and more picks than one turn takes beside 256 lanes."""
import pytest
import torch

from triton_amd.dispatch import combine, combine_backward, dispatch, dispatch_backward

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # the smallest value above zero

# tokens, picks, elements, lanes to a token in 16 bits and in float32
PAST_THE_CACHES = [(30000, 8, 128, 16, 16), (9000, 8, 515, 16, 64), (9000, 8, 259, 16, 16), (8200, 4, 1064, 64, 64), (8200, 4, 1063, 64, 64), (2400, 4, 2880, 256, 256),
                   (2400, 4, 2877, 256, 256), (1100, 12, 2880, 256, 256), (1400, 12, 2061, 256, 256)]     # (259 elements of 16 bits still go through them)
MANY_PICKS = [(50, 17, 2880, 256, 256), (300, 9, 2061, 256, 256)]


def made(T, k, H, dtype, device, drop=0.1):
    g = torch.Generator(device=device).manual_seed(T + k + H)
    randn = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
    n = T * k
    p = torch.randperm(n, generator=g, device=device).to(torch.int32)
    p = torch.where(torch.rand(n, generator=g, device=device) < drop, -1, p).to(torch.int32).view(T, k)
    return p, randn(T, H).to(dtype), randn(n, H).to(dtype), torch.rand(T, k, generator=g, device=device)


def near(got, want, dtype, slack=0.0):
    """One rounding to `dtype`, `slack` (what float32 sums may be off by, itself rounded) before it."""
    bound = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + 1.01 * slack + LEAST[dtype]
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"off by up to {float((err / bound).max()):.3f} of what rounding allows"


def additions(H, lanes, dtype):
    """The steps of a sum over a row: a piece's elements, a lane's pieces, those that join a wave's lanes, and the waves."""
    V = 4 if dtype == torch.float32 else 8
    return V + -(-H // V // lanes) + min(lanes, 64).bit_length() - 1 + (3 if lanes == 256 else 0)


@pytest.mark.parametrize("T,k,H,lanes16,lanes32", PAST_THE_CACHES + MANY_PICKS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_all(T, k, H, lanes16, lanes32, dtype, device):
    p, x, rows, gates = made(T, k, H, dtype, device)
    there, at = p >= 0, p.clamp(min=0).long()
    before = torch.full((T * k, H), 3.0, dtype=dtype, device=device)
    free = torch.ones(T * k, dtype=torch.bool, device=device)
    free[p[there].long()] = False
    # ---- rows from tokens
    got, plain = dispatch(x, p, gates=gates, out=before.clone()), dispatch(x, p, out=before.clone())
    drows, dg = combine_backward(x, p, rows=rows, gates=gates, out=before.clone())
    assert torch.equal(drows, got)
    for t in (got, plain):
        assert bool((t[free] == 3).all())
    assert torch.equal(plain[at][there], x[:, None].expand(T, k, H)[there])
    near(got[at][there], (x.double()[:, None] * gates.double()[..., None])[there], dtype)
    del got, plain, drows, before
    # ---- tokens from rows, a pick at a time
    y, ones, (dx, dg2) = combine(rows, p, gates=gates), combine(rows, p), dispatch_backward(rows, p, x=x, gates=gates)
    assert torch.equal(dx, y)
    total = [torch.zeros(T, H, dtype=torch.float64, device=device) for _ in range(4)]
    dots, size = torch.empty(T, k, dtype=torch.float64, device=device), torch.empty(T, k, dtype=torch.float64, device=device)
    for j in range(k):
        row = torch.where(there[:, j, None], rows[at[:, j]].double(), 0.0)
        term, product = row * gates[:, j, None].double(), row * x.double()
        for sum_, of in zip(total, (term, term.abs(), row, row.abs())):
            sum_ += of
        dots[:, j], size[:, j] = product.sum(1), product.abs().sum(1)
    near(y, total[0], dtype, (k + 1) * 2.0 ** -24 * total[1])
    near(ones, total[2], dtype, (k + 1) * 2.0 ** -24 * total[3])
    for d in (dg, dg2):
        near(d, dots, torch.float32, additions(H, lanes32 if dtype == torch.float32 else lanes16, dtype) * 2.0 ** -24 * size)
        assert bool((d[~there] == 0).all())


@pytest.mark.parametrize("T,k,H,lanes16,lanes32", PAST_THE_CACHES[-4:] + MANY_PICKS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_in_the_place_of_the_rows_and_again(T, k, H, lanes16, lanes32, dtype, device):
    """combine_backward into the rows that it reads, and each function a second time: the same bits."""
    p, x, rows, gates = made(T, k, H, dtype, device)
    want, dgates = combine_backward(x, p, rows=rows, gates=gates, out=rows.clone())
    back = dispatch_backward(rows, p, x=x, gates=gates)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(dispatch_backward(rows, p, x=x, gates=gates), back))
        assert torch.equal(combine_backward(x, p, rows=rows, gates=gates)[1], dgates)
    got, same = combine_backward(x, p, rows=rows, gates=gates, out=rows)
    assert got is rows and torch.equal(got, want) and torch.equal(same, dgates)


@pytest.mark.parametrize("T,H,lanes", [(2600, 5760, 64), (9000, 256, 16), (40, 5760, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_products_beside_large_ones(T, H, lanes, dtype, device):
    """A row whose products are one of 1 per lane and 2^-25 else, each of which a sum of 1 and more would lose: a piece's products are added up by themselves, so
    that a sum has as many steps as a lane has pieces, a piece elements, and the joins."""
    V = 4 if dtype == torch.float32 else 8
    pieces = H // V
    y = torch.full((1, H), 2.0 ** -25, dtype=dtype, device=device)
    y[0, :min(pieces, lanes) * V:V] = 1.0
    rows, x, gates = y.expand(T, H).contiguous(), torch.ones(T, H, dtype=dtype, device=device), torch.ones(T, 1, device=device)
    p = torch.arange(T, dtype=torch.int32, device=device)[:, None]
    want = y.double().sum()
    steps = additions(H, lanes, dtype)
    for dg in (combine_backward(x, p, rows=rows, gates=gates)[1], dispatch_backward(rows, p, x=x, gates=gates)[1]):
        assert bool(((dg.double() - want).abs() <= 1.01 * steps * 2.0 ** -24 * want).all()), (float(dg[0, 0]) / float(want) - 1) * 2 ** 24
