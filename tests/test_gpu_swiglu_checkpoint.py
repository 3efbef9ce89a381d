"""GPU: SwiGLU that keeps its input in 8 bits, and the gradient from that, against the formulas in 64 bits; what is kept against `downcast_to_mxfp`."""
import pytest
import torch

from triton_amd.numerics_details.mxfp import downcast_to_mxfp, upcast_from_mxfp
from triton_amd.swiglu import PrecisionConfig, swiglu_backward, swiglu_checkpoint

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
ALPHA = 1.702
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def kept_by_downcast(a):
    """What `downcast_to_mxfp` makes of rows that are filled up with zeros to whole groups."""
    L = a.shape[-1]
    values, scales = downcast_to_mxfp(torch.nn.functional.pad(a, (0, -L % 32)).contiguous(), torch.float8_e4m3fn, -1)
    return values[..., :L], scales


def read(values, scales):
    L = values.shape[-1]
    full = torch.nn.functional.pad(values.view(torch.uint8), (0, -L % 32)).view(torch.float8_e4m3fn)
    return upcast_from_mxfp(full, scales, torch.float32, -1)[..., :L]


def glu64(a, limit):
    """(out, s, g, l, the pairs that the limit lets through) in 64 bits."""
    a = a.double()
    g, l = a[..., 0::2], a[..., 1::2]
    free = (g <= limit, l.abs() <= limit) if limit is not None else (torch.ones_like(g).bool(), torch.ones_like(l).bool())
    if limit is not None:
        g, l = g.clamp(max=limit), l.clamp(-limit, limit)
    s = torch.sigmoid(ALPHA * g)
    return g * s * (l + 1), s, g, l, free


def within(got, want, slack, dtype):
    """One rounding to `dtype`, and `slack` for what float32 arithmetic may be off by before it."""
    bound = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + 1.01 * slack + LEAST[dtype]
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"off by up to {float((err / bound).max()):.3f} of what rounding allows"


def slack_of_s(g):
    # exp2's argument: alpha, the constant, and two products are rounded, which exp2 multiplies by |alpha g|; exp2 and the reciprocal are off by
    # two half steps each, the sum by one
    return (4 * (ALPHA * g).abs() + 5) * 2.0 ** -24


def laid(t, how):
    if how == "pitch":
        return torch.empty((t.shape[0], t.shape[1] + 48), dtype=t.dtype, device=t.device)[:, 16:16 + t.shape[1]].copy_(t)
    if how == "odd":
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)
    return t.t().contiguous().t() if how == "turned" else t


SHAPES = [(1, 1), (1, 16), (3, 5), (2, 20), (65, 48), (7, 1005), (130, 264), (33, 2880), (4099, 36), (5, 4100)]


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how,limit", [("dense", 7.0), ("pitch", None), ("odd", 0.5), ("turned", 7.0)])
def test_forward_and_backward(M, N, dtype, how, limit, device):
    torch.manual_seed(M + N)
    a = (torch.randn(M, 2 * N, device=device) * torch.exp(torch.randn(M, 1, device=device))).to(dtype)
    pc = PrecisionConfig(limit=limit)
    out, values, scales = swiglu_checkpoint(laid(a, how), ALPHA, pc)
    want_v, want_s = kept_by_downcast(a)
    assert values.dtype == torch.float8_e4m3fn and scales.dtype == torch.uint8
    assert torch.equal(values.view(torch.uint8), want_v.view(torch.uint8)) and torch.equal(scales, want_s)
    want, s, g, l, _ = glu64(a, limit)
    tiny = 2.0 ** -125 * (g.abs() + 1) * (l.abs() + 1)      # (a sigmoid below 2^-126 may be zero)
    within(out, want, (slack_of_s(g) + 3 * 2.0 ** -24) * want.abs() + tiny, dtype)
    # ---- backward, at the kept values
    d = torch.randn(M, N, device=device).to(dtype)
    da, again = swiglu_backward(laid(d, how), laid(values.view(torch.uint8), how).view(torch.float8_e4m3fn) if how != "turned" else values, laid(scales, how),
                                ALPHA, pc, return_out=True)
    want, s, g, l, free = glu64(read(values, scales), limit)
    tiny = 2.0 ** -125 * (g.abs() + 1) * (l.abs() + 1)
    within(again, want, (slack_of_s(g) + 3 * 2.0 ** -24) * want.abs() + tiny, dtype)
    d, ag = d.double(), (ALPHA * g).abs()
    slope = 1 + ALPHA * g * (1 - s)
    # the slope times s, as s + alpha (g s - (g s) s): s is off as above, g s, the difference and alpha are rounded, the sum by a half step (of these
    # three, which count alpha g (1 - s), two are written so and one as alpha g)
    slack = 2.0 ** -24 * (2 * ag * (1 - s) + slope.abs() + ag) + ag * s * slack_of_s(g)
    factor = (d * (l + 1) * s).abs()
    dgate = torch.where(free[0], d * (l + 1) * s * slope, 0.0)
    within(da[:, 0::2], dgate, factor * (slack + slope.abs() * (slack_of_s(g) + 4 * 2.0 ** -24)) + tiny * d.abs(), dtype)
    dlinear = torch.where(free[1], d * g * s, 0.0)
    within(da[:, 1::2], dlinear, dlinear.abs() * (slack_of_s(g) + 3 * 2.0 ** -24) + tiny * d.abs(), dtype)
    alone, none = swiglu_backward(d.to(dtype), values, scales, ALPHA, pc)
    assert none is None and torch.equal(alone, da)


def test_leading_axes_and_nothing_there(device):
    a = torch.randn(2, 3, 64, device=device)
    out, values, scales = swiglu_checkpoint(a, ALPHA, PrecisionConfig(limit=7.0))
    assert tuple(out.shape) == (2, 3, 32) and tuple(values.shape) == (2, 3, 64) and tuple(scales.shape) == (2, 3, 2)
    da, again = swiglu_backward(torch.ones_like(out), values, scales, ALPHA, PrecisionConfig(limit=7.0), return_out=True)
    assert da.shape == a.shape and again.shape == out.shape
    one, v1, s1 = swiglu_checkpoint(a[1, 2], ALPHA, PrecisionConfig(limit=7.0))
    assert torch.equal(one, out[1, 2]) and torch.equal(s1, scales[1, 2])
    for shape in ((0, 64), (5, 0), (0, 0), (0, 3, 32)):
        out, values, scales = swiglu_checkpoint(torch.empty(shape, device=device), ALPHA, PrecisionConfig(limit=None))
        assert tuple(out.shape) == (*shape[:-1], shape[-1] // 2) and tuple(values.shape) == shape
        da, again = swiglu_backward(out, values, scales, ALPHA, PrecisionConfig(limit=None), return_out=True)
        assert tuple(da.shape) == shape and again.shape == out.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_extremes_are_kept_as_downcast_keeps_them(dtype, device):
    """Groups of nothing but zeros, of the smallest and largest numbers, with infinities and NaN, and maxima at and beside 448 * 2^e."""
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    a = torch.randn(12, 64, device=device).to(dtype)
    a[0] = 0
    a[1] = a[1] * small
    a[2] = small * torch.finfo(dtype).eps
    a[3, 5], a[4, 7] = big, -big
    a[5, 33], a[6, 2], a[7, 40] = float("inf"), float("-inf"), float("nan")
    for i, v in enumerate((448.0, 450.0, 446.0, 1.75)):
        a[8 + i] = a[8 + i].clamp(-1, 1)
        a[8 + i, 3] = v
    out, values, scales = swiglu_checkpoint(a, ALPHA, PrecisionConfig(limit=7.0))
    want_v, want_s = kept_by_downcast(a)
    assert torch.equal(scales, want_s) and torch.equal(values.view(torch.uint8), want_v.view(torch.uint8))
    want = glu64(a, 7.0)[0]
    nan = torch.isnan(a[:, 0::2]) | torch.isnan(a[:, 1::2])
    assert torch.equal(torch.isnan(out), nan | torch.isnan(want))
    d = torch.ones_like(out)
    da, again = swiglu_backward(d, values, scales, ALPHA, PrecisionConfig(limit=7.0), return_out=True)
    kept = read(values, scales)
    lost = torch.isnan(kept[:, 0::2]) | torch.isnan(kept[:, 1::2])
    assert torch.equal(torch.isnan(again), lost) and bool(lost[5, 16:].all() and not lost[5, :16].any() and lost[7, 20] and int(lost[7].sum()) == 1)
    assert bool(torch.isnan(da[:, 0::2])[lost].all()) and not bool(torch.isnan(da[:, 0::2])[~lost].any())


@pytest.mark.parametrize("M,N", [(8100, 1001), (8100, 1002), (8100, 1003), (700, 98), (3, 1), (5, 2), (5, 3), (9, 5), (300, 33)])
@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_rows_as_whole_ones(M, N, dtype, device):
    """Rows that end inside a piece: bit for bit what the same rows give with zeros behind them."""
    torch.manual_seed(N)
    a, d = torch.randn(M, 2 * N, device=device).to(dtype), torch.randn(M, N, device=device).to(dtype)
    filled = lambda t, to: torch.nn.functional.pad(t, (0, -t.shape[1] % to))
    pc = PrecisionConfig(limit=1.5)
    out, values, scales = swiglu_checkpoint(a, ALPHA, pc)
    want = swiglu_checkpoint(filled(a, 32), ALPHA, pc)
    assert torch.equal(out, want[0][:, :N]) and torch.equal(values.view(torch.uint8), want[1].view(torch.uint8)[:, :2 * N]) and torch.equal(scales, want[2])
    da, again = swiglu_backward(d, values, scales, ALPHA, pc, return_out=True)
    want_da, want_again = swiglu_backward(filled(d, 16), want[1], scales, ALPHA, pc, return_out=True)
    assert torch.equal(da, want_da[:, :2 * N]) and torch.equal(again, want_again[:, :N])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("limit", [None, 7.0])
def test_the_lowest_and_the_greatest_values(dtype, limit, device):
    """A gate at the type's lowest value (kept as -2^128) gives zeros, one at the greatest its linear value, where they are kept alone in their groups."""
    most = torch.finfo(dtype).max
    a = torch.zeros(6, 32, dtype=dtype, device=device)
    for row, g in enumerate((-most, most, -most / 2, most / 2, -most * 0.6, 2.0 ** 120)):
        a[row, 6] = g
    a[5, 7] = a[0, 7] = a[2, 7] = -most
    d = torch.full((6, 16), 2.0, dtype=dtype, device=device)
    pc = PrecisionConfig(limit=limit)
    out, values, scales = swiglu_checkpoint(a, ALPHA, pc)
    da, again = swiglu_backward(d, values, scales, ALPHA, pc, return_out=True)
    power = torch.ldexp(torch.ones(6, 1, dtype=torch.float64, device=device), scales.double() - 127)
    want, s, g, l, free = glu64(values.double() * torch.where(scales == 0, 0.0, power), limit)
    slope = 1 + ALPHA * g * (1 - s)
    for got, right in ((da[:, 0::2], torch.where(free[0], 2 * (l + 1) * s * slope, 0.0)), (da[:, 1::2], torch.where(free[1], 2 * g * s, 0.0)), (again, want)):
        near = right.clamp(-2.0 ** 128, 2.0 ** 128)   # (beyond the type's range both are infinite, or its greatest value stands for 2^128)
        got = got.double().clamp(-2.0 ** 128, 2.0 ** 128)
        slack = 1.01 * HALF_STEP[dtype] + slack_of_s(g.clamp(-100, 100)) + 4 * 2.0 ** -24
        assert bool(((got - near).abs() <= slack * near.abs() + LEAST[dtype]).all())
    assert bool((da[0, 6:8] == 0).all() and again[0, 3] == 0 and out[0, 3] == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("limit", [float("inf"), 1e300])
def test_a_limit_beyond_the_numbers_is_none(dtype, limit, device):
    """An infinite limit, or one that float32 has no number for, cuts nothing off: bit for bit what no limit gives, also at values that are kept as 2^128."""
    torch.manual_seed(4)
    most = torch.finfo(dtype).max
    a = torch.randn(9, 96, device=device).to(dtype)
    for row, (at, v) in enumerate(((6, most), (7, most), (6, -most), (7, -most), (6, float("inf")), (7, float("-inf")), (6, most / 2), (6, float("nan")))):
        a[row, at] = v
    d = torch.randn(9, 48, device=device).to(dtype)
    kept, free = swiglu_checkpoint(a, ALPHA, PrecisionConfig(limit=limit)), swiglu_checkpoint(a, ALPHA, PrecisionConfig(limit=None))
    bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert all(torch.equal(bits(x), bits(y)) for x, y in zip(kept, free))
    got = swiglu_backward(d, *kept[1:], ALPHA, PrecisionConfig(limit=limit), return_out=True)
    want = swiglu_backward(d, *kept[1:], ALPHA, PrecisionConfig(limit=None), return_out=True)
    lost = torch.isnan(read(*kept[1:]))
    for x, y in zip(got, want):
        assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(nan=0.0), y.nan_to_num(nan=0.0))
    assert not bool(torch.isnan(got[0][:4])[~lost[:4]].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("alpha", [0.0, 2.0 ** -126, -2.0 ** -126, -1.0])
def test_the_lowest_value_with_a_flat_sigmoid(dtype, alpha, device):
    """A gate kept as -2^128 whose sigmoid is no zero, as alpha is (nearly) 0 or negative: it counts as the lowest of float32 there too."""
    most = torch.finfo(dtype).max
    a = torch.zeros(2, 32, dtype=dtype, device=device)
    a[0, 6], a[1, 6] = -most, most
    pc, d = PrecisionConfig(limit=None), torch.full((2, 16), 0.25, dtype=dtype, device=device)
    _, values, scales = swiglu_checkpoint(a, alpha, pc)
    da, again = swiglu_backward(d, values, scales, alpha, pc, return_out=True)
    g = torch.tensor([-2.0 ** 128, 2.0 ** 128], dtype=torch.float64, device=device)
    s = torch.sigmoid(alpha * g)
    # (no more than |alpha g| = 4 where the sigmoid is neither 0 nor 1: a float32 exponential and reciprocal, and the steps behind them, are off by 2^-18 at most)
    for got, want in ((again[:, 3], g * s), (da[:, 6], 0.25 * (s + alpha * g * s * (1 - s))), (da[:, 7], 0.25 * g * s)):
        want = want.clamp(-float(most), float(most))
        got = got.double().clamp(-float(most), float(most))
        assert bool(((got - want).abs() <= (HALF_STEP[dtype] + 2.0 ** -18) * want.abs() + LEAST[dtype]).all()), (got, want)


def test_at_the_limit_the_gradient_passes(device):
    """7 and -7 are kept exactly and are not beyond a limit of 7; the next values are."""
    a = torch.tensor([[7.0, 7.0, 7.0, -7.0, 7.5, 0.5, 0.5, 7.5, -9.0, -7.5, 0.0, 0.0]], device=device)
    out, values, scales = swiglu_checkpoint(a, ALPHA, PrecisionConfig(limit=7.0))
    assert torch.equal(read(values, scales), a)
    da, _ = swiglu_backward(torch.ones_like(out), values, scales, ALPHA, PrecisionConfig(limit=7.0))
    assert torch.equal(da[0] != 0, torch.tensor([1, 1, 1, 1, 0, 1, 1, 0, 1, 0, 1, 0], device=device).bool())


def test_gradient_is_that_of_differences(device):
    """Along a direction, in 64 bits of the forward formula: the kernel's gradient times the direction."""
    torch.manual_seed(1)
    a = torch.randn(40, 320, device=device)
    out, values, scales = swiglu_checkpoint(a, ALPHA, PrecisionConfig(limit=None))
    at, way, d = read(values, scales).double(), torch.randn(40, 320, device=device).double(), torch.randn(40, 160, device=device)
    da, _ = swiglu_backward(d, values, scales, ALPHA, PrecisionConfig(limit=None))
    step = 2.0 ** -10
    rise = float(((glu64(at + step * way, None)[0] - glu64(at - step * way, None)[0]) * d.double()).sum()) / (2 * step)
    # (the third derivative times step^2 / 6 is below 1e-5 of the terms)
    assert abs(rise - float((da.double() * way).sum())) < 1e-5 * float((da.double() * way).abs().sum())


def test_elements_past_32_bits(device):
    """Rows whose bytes lie past 4 GB, and group numbers past 2^26: the last rows are those of a call on them alone."""
    M, N = 2 ** 20 + 5, 1040
    a = torch.empty(M, 2 * N, dtype=torch.bfloat16, device=device)
    a[-7:] = torch.randn(7, 2 * N, device=device)
    a[:-7].zero_()
    pc = PrecisionConfig(limit=7.0)
    out, values, scales = swiglu_checkpoint(a, ALPHA, pc)
    few = swiglu_checkpoint(a[-7:], ALPHA, pc)
    assert all(torch.equal(x[-7:].view(torch.uint8), y.view(torch.uint8)) for x, y in zip((out, values, scales), few))
    assert not bool(out[:-7].any()) and not bool(scales[:-7].any())
    da, again = swiglu_backward(out, values, scales, ALPHA, pc, return_out=True)
    da7, again7 = swiglu_backward(out[-7:], values[-7:], scales[-7:], ALPHA, pc, return_out=True)
    assert torch.equal(da[-7:], da7) and torch.equal(again[-7:], again7) and not bool(da[:-7].any())


def test_another_stream_and_a_graph(device):
    torch.manual_seed(2)
    a, d, pc = torch.randn(64, 512, device=device).bfloat16(), torch.randn(64, 256, device=device).bfloat16(), PrecisionConfig(limit=7.0)

    def step():
        kept = swiglu_checkpoint(a, ALPHA, pc)
        return (kept[0], kept[1].view(torch.uint8), kept[2], *swiglu_backward(d, kept[1], kept[2], ALPHA, pc, return_out=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(mine, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        a.copy_(torch.randn(64, 512, device=device))
        d.copy_(torch.randn(64, 256, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, step()))
