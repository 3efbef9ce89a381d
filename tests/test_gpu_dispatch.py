"""GPU: rows of tokens to the rows of their experts and back (`dispatch`, `combine`) and their gradients, against the formulas in 64 bits: every type,
tokens and picks without a row, rows that nothing names, odd sizes, pitches and starts, more picks than one turn of the kernels takes."""
import ctypes

import pytest
import torch

from triton_amd import _lib
from triton_amd.dispatch import combine, combine_backward, dispatch, dispatch_backward
from triton_amd.routing import routing

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # the smallest value above zero


def places(T, k, n, drop=0.0, beyond=False):
    """int32 [T, k]: distinct rows of [0, n), -1 (or numbers past the rows) where a pick has none."""
    p = torch.randperm(n)[:T * k].to(torch.int32)
    p = torch.where(torch.rand(T * k) < drop, torch.where(torch.rand(T * k) < 0.5, n, n + 2 ** 20) if beyond else -torch.ones(T * k), p).to(torch.int32)
    return p.view(T, k)


def laid(t, device, how):
    """`t` on the device: dense, with a pitch, at an odd start, or with the axes exchanged."""
    t = t.to(device)
    if how == "pitch":
        room = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=device)
        return room[:, 8:8 + t.shape[1]].copy_(t)
    if how == "odd":
        room = torch.full((t.numel() + 1,), float("nan"), dtype=t.dtype, device=device)
        return room[1:].view(t.shape).copy_(t)
    return t.t().contiguous().t() if how == "turned" else t


def rounded(got, want, dtype, slack=0.0):
    """One rounding to `dtype`, `slack` (what float32 sums may be off by, itself rounded) before it."""
    bound = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + 1.01 * slack + LEAST[dtype]
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"off by up to {float((err / bound).max()):.3f} of what rounding allows"


def of(p, rows):
    """rows[p] in 64 bits [T, k, H], zeros without a row."""
    there = (p >= 0) & (p < rows.shape[0])
    return torch.where(there[..., None], rows.double()[torch.where(there, p, 0).long()], 0.0) if rows.shape[0] else torch.zeros(*p.shape, rows.shape[1]).double()


def scattered(p, values, into):
    there = (p >= 0) & (p < into.shape[0])
    out = into.double().clone()
    out[p[there].long()] = values[there]
    return out


CASES = [(1, 1, 1, 1, 0.0), (1, 4, 2880, 4, 0.0), (3, 2, 7, 6, 0.3), (5, 8, 64, 50, 0.2), (17, 3, 1063, 60, 0.0), (65, 4, 520, 260, 0.1), (9, 9, 96, 81, 0.2),
         (6, 17, 264, 110, 0.1), (4100, 2, 136, 8300, 0.1), (4099, 1, 33, 4099, 0.0), (4101, 11, 40, 45111, 0.1), (33, 6, 3000, 198, 1.0),
         (8200, 2, 264, 16400, 0.1), (4200, 9, 1100, 37800, 0.1), (2600, 3, 1064, 7900, 0.2), (2501, 2, 2600, 5002, 0.1), (700, 12, 256, 8400, 0.0)]


@pytest.mark.parametrize("T,k,H,n,drop", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("how,gate_type", [("dense", torch.float32), ("pitch", torch.bfloat16), ("odd", torch.float32), ("turned", torch.float16), ("dense", None)])
def test_all(T, k, H, n, drop, dtype, how, gate_type, device):
    torch.manual_seed(T + 7 * k + H)
    p = places(T, k, n, drop, beyond=how == "pitch")
    x, rows = torch.randn(T, H).to(dtype), torch.randn(n, H).to(dtype)
    gates = None if gate_type is None else torch.rand(T, k).to(gate_type)
    g64 = torch.ones(T, k, 1).double() if gates is None else gates.double()[..., None]
    gd = None if gates is None else laid(gates, device, "turned" if how == "turned" else "dense")
    xd, rd, pd = laid(x, device, how), laid(rows, device, how), p.to(device)
    if how == "pitch":
        pd = torch.cat([pd, pd], 1)[:, :k]
    before = torch.randn(n, H).to(dtype)
    # ---- dispatch
    want = scattered(p, x.double()[:, None] * g64, before)
    got = laid(before, device, how if how != "turned" else "dense")
    assert dispatch(xd, pd, gates=gd, out=got) is got
    if gates is None:
        assert torch.equal(got.cpu(), want.to(dtype))
    else:
        rounded(got, want, dtype)
    there = (p >= 0) & (p < n)
    assert torch.equal(torch.ones(n).index_fill(0, p[there].long(), 0).bool()[:, None] & (got.cpu() != before), torch.zeros(n, H).bool()), "rows that no pick names"
    # ---- combine
    terms = of(p, rows) * g64
    slack = (k + 1) * 2.0 ** -24 * terms.abs().sum(1)
    rounded(combine(rd, pd, gates=gd), terms.sum(1), dtype, slack)
    # ---- their gradients: the same sums and copies, and products over a row: a lane's chain of them, and a few more additions
    # (every lane adds up H / 64 elements and a piece at most, then 6 + 3 partial sums are joined)
    longest = (H / 64 + 8 + 10) * 2.0 ** -24
    products = of(p, rows) * x.double()[:, None]
    out = laid(before, device, how if how != "turned" else "dense")
    drows, dg = combine_backward(xd, pd, rows=rd if gates is not None else None, gates=gd, out=out)
    assert drows is out and torch.equal(drows, got)
    dx, dg2 = dispatch_backward(rd, pd, x=xd, gates=gd)
    rounded(dx, terms.sum(1), dtype, slack)
    if gates is None:
        assert dg is None and dg2 is None
    else:
        for d in (dg, dg2):
            assert d.dtype == gate_type and tuple(d.shape) == (T, k)
            rounded(d, products.sum(-1), gate_type, longest * products.abs().sum(-1))
            assert bool((d.cpu()[~there] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_new_rows_without_out(dtype, device):
    """Every pick has a row: the result is whole, and combining it with one pick's weight gives the token again."""
    torch.manual_seed(0)
    r = routing(torch.randn(300, 32, device=device), 4)
    x = torch.randn(300, 264, device=device).to(dtype)
    p = r.row_sorted_indx.view(300, 4)
    rows = dispatch(x, p)
    assert torch.equal(rows, x[r.gather_indx.long()])
    one = torch.tensor([0.0, 1.0, 0.0, 0.0], device=device).expand(300, 4)
    assert torch.equal(combine(rows, p, gates=one), x)
    drows, none = combine_backward(x, p)
    assert none is None and torch.equal(drows, rows)


def test_bits_are_copied(device):
    """Without gates: NaN patterns, subnormal numbers and both zeros come out as they went in."""
    for dtype, bits in ((torch.bfloat16, torch.int16), (torch.float16, torch.int16)):
        x = torch.arange(-32768, 32768, dtype=torch.int32, device=device).to(bits).view(64, 1024).view(dtype)
        p = torch.arange(64, dtype=torch.int32, device=device).flip(0).view(64, 1)
        for start in (0, 1):
            part = x[:, start:]
            assert torch.equal(dispatch(part, p).view(bits).flip(0), part.contiguous().view(bits))


def test_special_values_stay_where_they_are(device):
    """Infinities and NaN of a row reach its token only, and those of rows that no pick names nobody; a gate of 0 keeps a NaN."""
    rows = torch.full((8, 40), float("nan"), device=device)
    rows[0], rows[1], rows[2] = 1.0, float("inf"), 2.0
    p = torch.tensor([[0, 2], [1, 0], [2, 7], [-1, 2 ** 30]], dtype=torch.int32, device=device)
    gates = torch.tensor([[1.0, 0.5], [1.0, 1.0], [1.0, 0.0], [float("nan"), float("inf")]], device=device)
    y = combine(rows, p, gates=gates)
    assert bool((y[0] == 2).all() and torch.isinf(y[1]).all() and torch.isnan(y[2]).all() and (y[3] == 0).all())
    dx, dg = dispatch_backward(rows, p, x=torch.ones(4, 40, device=device), gates=gates)
    assert torch.equal(torch.isnan(dg).cpu(), torch.tensor([[False, False], [False, False], [False, True], [False, False]])) and bool((dg[3] == 0).all())


@pytest.mark.parametrize("T,k,H,n", [(0, 4, 64, 8), (5, 0, 64, 8), (5, 4, 0, 20), (5, 4, 64, 0), (0, 0, 0, 0)])
def test_nothing_there(T, k, H, n, device):
    p = torch.full((T, k), 3, dtype=torch.int32, device=device)
    x, rows, gates = torch.randn(T, H, device=device), torch.randn(n, H, device=device), torch.rand(T, k, device=device)
    kept = torch.ones(n, H, device=device)
    if n < 1 or T * k == 0:
        assert torch.equal(dispatch(x, p, gates=gates, out=kept), torch.ones(n, H, device=device))
    y, (dx, dg) = combine(rows, p, gates=gates), dispatch_backward(rows, p, x=x, gates=gates)
    assert tuple(y.shape) == tuple(dx.shape) == (T, H) and tuple(dg.shape) == (T, k)
    if H == 0 or n == 0:
        assert bool((dg == 0).all())
    if k == 0 or n == 0:
        assert bool((y == 0).all())
    if T * k == 0 or n == 0:
        drows, dg = combine_backward(x, p, rows=rows, gates=gates, out=kept)
        assert bool((drows == 1).all()) and bool((dg == 0).all())


def test_rows_past_four_gigabytes(device):
    """Rows whose bytes lie beyond what 32 bits count, at both ends of the tensor."""
    n, H = 2 ** 19, 4608
    rows = torch.zeros(n, H, dtype=torch.bfloat16, device=device)            # 4.8 GB
    x = torch.randn(4, H, device=device).to(torch.bfloat16)
    p = torch.tensor([[n - 1, 0], [n // 2, 3], [n - 2, n // 2 + 1], [5, n - 7]], dtype=torch.int32, device=device)
    gates = torch.rand(4, 2, device=device)
    dispatch(x, p, out=rows)
    assert torch.equal(rows[p.long()], x[:, None].expand(4, 2, H)) and int((rows != 0).any(1).sum()) == 8
    want = x.double() * gates.double().sum(1, keepdim=True)
    rounded(combine(rows, p, gates=gates), want.cpu(), torch.bfloat16, 3 * 2.0 ** -24 * want.abs().cpu())
    drows, dg = combine_backward(x, p, rows=rows, gates=gates, out=rows)      # (every element is read before it is written)
    want = x.double().square().sum(1, keepdim=True).expand(4, 2).cpu()
    rounded(dg, want, torch.float32, (H / 64 + 18) * 2.0 ** -24 * want)


def test_gradients_are_those_of_differences(device):
    """Along a direction: both functions are linear in the rows and in the gates, so a difference over any step is the gradient's product."""
    torch.manual_seed(3)
    T, k, H = 37, 4, 72
    p = places(T, k, T * k, 0.1).to(device)
    x, dx, dy = (torch.randn(T, H, device=device) for _ in range(3))
    rows, drows = torch.randn(T * k, H, device=device), torch.randn(T * k, H, device=device)
    gates, dgates = torch.rand(T, k, device=device), torch.randn(T, k, device=device)
    dot = lambda a, b: float((a.double() * b.double()).sum())  # noqa: E731
    g_rows, g_gates = combine_backward(dy, p, rows=rows, gates=gates, out=torch.zeros_like(rows))
    both = lambda e: combine(rows + e * drows, p, gates=gates), lambda e: combine(rows, p, gates=gates + e * dgates)  # noqa: E731
    for f, grad, way in zip(both, (g_rows, g_gates), (drows, dgates)):
        assert abs(dot(f(0.5), dy) - dot(f(-0.5), dy) - dot(grad, way)) < 1e-5 * dot(way.abs(), grad.abs())
    up = torch.randn(T * k, H, device=device)
    g_x, g_gates = dispatch_backward(up, p, x=x, gates=gates)
    f = lambda x, g: dot(dispatch(x, p, gates=g, out=torch.zeros_like(rows)), up)  # noqa: E731
    assert abs(f(x + 0.5 * dx, gates) - f(x - 0.5 * dx, gates) - dot(g_x, dx)) < 1e-5 * dot(g_x.abs(), dx.abs())
    assert abs(f(x, gates + 0.5 * dgates) - f(x, gates - 0.5 * dgates) - dot(g_gates, dgates)) < 1e-5 * dot(g_gates.abs(), dgates.abs())


def test_same_result_whatever_the_batch(device):
    """A token's sums do not depend on how many tokens there are within one form of the launch, and repeat bit for bit."""
    torch.manual_seed(5)
    T, k, H = 500, 4, 1000
    p, rows, gates, dy = places(T, k, T * k).to(device), torch.randn(T * k, H, device=device), torch.rand(T, k, device=device), torch.randn(T, H, device=device)
    y, (_, dg) = combine(rows, p, gates=gates), combine_backward(dy, p, rows=rows, gates=gates)
    for _ in range(3):
        assert torch.equal(combine(rows, p, gates=gates), y) and torch.equal(combine_backward(dy, p, rows=rows, gates=gates)[1], dg)
    assert torch.equal(combine(rows, p[:7], gates=gates[:7]), y[:7])


def test_another_stream_and_a_graph(device):
    torch.manual_seed(6)
    T, k, H = 64, 4, 520
    p, gates = places(T, k, T * k).to(device), torch.rand(T, k, device=device)
    x, rows = torch.randn(T, H, device=device).bfloat16(), torch.randn(T * k, H, device=device).bfloat16()

    def step():
        return (dispatch(x, p, gates=gates), combine(rows, p, gates=gates), *combine_backward(x, p, rows=rows, gates=gates), *dispatch_backward(rows, p, x=x, gates=gates))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(mine, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for _ in range(4):
        x.copy_(torch.randn(T, H, device=device))
        gates.copy_(torch.rand(T, k, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


@pytest.mark.parametrize("T,k,H", [(40, 4, 264), (3000, 2, 1032), (9, 11, 77), (9000, 3, 64), (9001, 3, 1037), (700, 2, 2050), (50, 3, 5), (300, 4, 2060), (64, 2, 4108), (2400, 3, 1026)])
def test_gradient_in_the_place_of_the_rows(T, k, H, device):
    """combine_backward into the rows that it reads: what it gives elsewhere.  (Rows whose last piece is another wave's than the one before it are among them: what
    one wave stores, the other must have read, or store itself.)"""
    torch.manual_seed(T)
    for dtype in (torch.bfloat16, torch.float32):
        p, gates = places(T, k, T * k, 0.1).to(device), torch.rand(T, k, device=device)
        dy, rows = torch.randn(T, H, device=device).to(dtype), torch.randn(T * k, H, device=device).to(dtype)
        want, dgates = combine_backward(dy, p, rows=rows, gates=gates, out=rows.clone())
        got, same = combine_backward(dy, p, rows=rows, gates=gates, out=rows)
        assert got is rows and torch.equal(got, want) and torch.equal(same, dgates)


@pytest.mark.parametrize("T,k,H", [(9001, 4, 1037), (2000, 3, 1037), (700, 2, 2050), (9000, 3, 60), (30, 5, 9), (30001, 4, 301)])
def test_ragged_rows_as_whole_ones(T, k, H, device):
    """Rows that are no whole 16-byte pieces: bit for bit what the same rows give with zeros behind them."""
    torch.manual_seed(H)
    n = T * k
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        p, gates = places(T, k, n, 0.1).to(device), torch.rand(T, k, device=device)
        x, rows = torch.randn(T, H, device=device).to(dtype), torch.randn(n, H, device=device).to(dtype)
        filled = lambda t: torch.nn.functional.pad(t, (0, -H % 8))
        rest = filled(torch.zeros(n, H, device=device).to(dtype))
        assert torch.equal(dispatch(x, p, gates=gates, out=torch.zeros_like(rows)), dispatch(filled(x), p, gates=gates, out=rest)[:, :H])
        assert torch.equal(combine(rows, p, gates=gates), combine(filled(rows), p, gates=gates)[:, :H])
        for got, want in zip(dispatch_backward(rows, p, x=x, gates=gates), dispatch_backward(filled(rows), p, x=filled(x), gates=gates)):
            assert torch.equal(got, want[:, :got.shape[1]])
        for got, want in zip(combine_backward(x, p, rows=rows, gates=gates, out=torch.zeros_like(rows)),
                             combine_backward(filled(x), p, rows=filled(rows), gates=gates, out=rest)):
            assert torch.equal(got, want[:, :got.shape[1]])


def test_rows_that_are_too_long(device):
    """2^31 elements and more to a row are refused, before anything is made of them."""
    p = torch.zeros(1, 1, dtype=torch.int32, device=device)
    for H in (2 ** 31, 2 ** 32 + 8):
        long = torch.zeros(1, 1, dtype=torch.bfloat16, device=device).expand(1, H)
        for call in (dispatch, combine, combine_backward, dispatch_backward):
            with pytest.raises(NotImplementedError):
                call(long, p)


@pytest.mark.parametrize("T,k,H", [(5, 3, 40), (300, 2, 1037), (50, 4, 2880), (64, 9, 2061)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_products_without_gates(T, k, H, dtype, device):
    """The C entry points give the rows' products without gate weights too (each counts as 1)."""
    torch.manual_seed(H)
    n = T * k
    p = places(T, k, n, 0.1)
    tokens, rows = torch.randn(T, H).to(dtype), torch.randn(n, H).to(dtype)
    pd, td, rd = p.to(device), tokens.to(device), rows.to(device)
    products = (of(p, rows) * tokens.double()[:, None])
    slack = (H / 16 + 18) * 2.0 ** -24 * products.abs().sum(-1)      # (16 lanes or more add up a row, and are joined)
    for spread, out in ((True, torch.full((n, H), 3.0, dtype=dtype, device=device)), (False, torch.empty(T, H, dtype=dtype, device=device))):
        src, other = (td, rd) if spread else (rd, td)
        dots = torch.empty(T, k, device=device)
        a = _lib.TokenRowsArgs(src=src.data_ptr(), src_stride=H, dst=out.data_ptr(), dst_stride=H, row_indx=pd.data_ptr(), row_indx_stride=k, gates_dtype=_lib.F32,
                               other=other.data_ptr(), other_stride=H, dots=dots.data_ptr(), dots_stride=k, dtype=_lib.dtype_code(dtype), T=T, k=k, H=H, n_rows=n)
        entry = _lib.lib().tamd_dispatch if spread else _lib.lib().tamd_combine
        assert entry(ctypes.byref(a), ctypes.sizeof(a), _lib.stream_ptr(device)) == 0
        rounded(dots, products.sum(-1), torch.float32, slack)
        if spread:
            assert torch.equal(out.cpu(), scattered(p, tokens.double()[:, None].expand(T, k, H), torch.full((n, H), 3.0)).to(dtype))
        else:
            terms = of(p, rows)
            rounded(out, terms.sum(1), dtype, (k + 1) * 2.0 ** -24 * terms.abs().sum(1))
