"""GPU: products over ragged rows (`matmul` with ragged metadata of both operands), the gradients of all experts' weights, against products in 64 bits."""
import pytest
import torch

from triton_amd.matmul import PrecisionConfig, matmul
from triton_amd.tensor import make_ragged_tensor_metadata

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def ragged(sizes, rows, device):
    return make_ragged_tensor_metadata(torch.tensor(sizes, dtype=torch.int32, device=device), rows)


def check(got, x, d, sizes, dtype):
    """Every slice against its product; float32 sums of n products of 16-bit numbers (exact in float32) are off by n half steps of the sum of
    their sizes at most, the result is rounded once."""
    at = 0
    assert got.dtype == dtype and tuple(got.shape) == (len(sizes), x.shape[1], d.shape[1])
    for e, n in enumerate(sizes):
        a, b = x[at:at + n].double().t().contiguous(), d[at:at + n].double()
        want, size = a @ b, a.abs() @ b.abs()
        bound = HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -8) + 1.01 * (n + 1) * 2.0 ** -24 * size + LEAST[dtype]
        err = (got[e].double() - want).abs()
        assert bool((err <= bound).all()), (e, n, float((err / bound).max()))
        at += n


def laid(t, how):
    if how == "pitch":
        return torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=t.device)[:, 8:8 + t.shape[1]].copy_(t)
    if how == "odd":
        return torch.full((t.numel() + 1,), float("nan"), dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)
    return t.t().contiguous().t() if how == "turned" else t


SIZES = [[1], [0], [33, 0, 1, 95, 32, 31], [0, 0, 700, 5], [64] * 9, [513, 2, 0, 129]]


@pytest.mark.parametrize("M,N", [(1, 1), (8, 16), (7, 130), (128, 128), (264, 136), (300, 96), (129, 257)])
@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("dtype,out,how", [(torch.bfloat16, None, "dense"), (torch.float16, torch.float32, "pitch"), (torch.float16, None, "odd"),
                                           (torch.bfloat16, torch.float16, "turned")])
def test_small(M, N, sizes, dtype, out, how, device):
    torch.manual_seed(M + N + len(sizes))
    rows = sum(sizes)
    x, d = torch.randn(rows, M, device=device).to(dtype), torch.randn(rows, N, device=device).to(dtype)
    # rows behind the last slice hold NaN, and take no part
    more = torch.full((5, 1), float("nan"), dtype=dtype, device=device)
    xs, ds = laid(torch.cat([x, more.expand(5, M)]), how), laid(torch.cat([d, more.expand(5, N)]), how)
    md = ragged(sizes, rows, device)
    got = matmul(xs.t(), ds, None, md, md, precision_config=PrecisionConfig(out_dtype=out))
    check(got, x, d, sizes, out or dtype)
    assert torch.equal(matmul(xs.t(), ds, None, None, md, precision_config=PrecisionConfig(out_dtype=out)), got)


@pytest.mark.parametrize("M,N,sizes", [(2048, 2056, [300, 257, 0, 400]), (520, 8200, [256, 600, 513, 258]), (4097, 1030, [400, 300]), (256, 256, [3000, 9, 0, 4100]),
                                       (64, 72, [5000, 1]), (1000, 8, [2049, 2048, 2047]), (96, 33, [70000]), (4100, 2600, [320, 350, 0, 700, 400]), (2600, 4104, [333, 650, 0, 700])])
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, None), (torch.float16, torch.float32)])
def test_larger_tiles_and_splits(M, N, sizes, dtype, out, device):
    torch.manual_seed(M + N)
    rows = sum(sizes)
    x, d = torch.randn(rows, M, device=device).to(dtype), torch.randn(rows, N, device=device).to(dtype)
    md = ragged(sizes, rows, device)
    got = matmul(x.t(), d, None, md, md, precision_config=PrecisionConfig(out_dtype=out))
    check(got, x, d, sizes, out or dtype)
    for _ in range(2):
        assert torch.equal(matmul(x.t(), d, None, md, md, precision_config=PrecisionConfig(out_dtype=out)), got)


@pytest.mark.parametrize("E", [2, 7, 40, 64, 65])
@pytest.mark.parametrize("M,N", [(136, 264), (40, 33)])
def test_long_slices_of_all_lengths(E, M, N, device):
    """Slices whose longest ones go first: every one has its turn, whatever the order of their lengths, those of equal and of no length among them."""
    torch.manual_seed(E)
    share = torch.rand(E) * (torch.rand(E) < 0.8)
    share[-1] = share[0] = share.max()
    for sizes in ([1100] * E, (share * 2 * 1100).int().tolist() if E > 2 else [0, 1500], list(range(1000, 1000 + E)), [1030 + E - e for e in range(E)]):
        rows = sum(sizes)
        x, d = torch.randn(rows, M, device=device).bfloat16(), torch.randn(rows, N, device=device).bfloat16()
        md = ragged(sizes, rows, device)
        check(matmul(x.t(), d, None, md, md), x, d, sizes, torch.bfloat16)


@pytest.mark.parametrize("M,N,sizes", [(136, 72, [40, 0, 50]), (64, 64, [3000, 100])])
def test_into_given_results(M, N, sizes, device):
    """c with pitches of its own: only the results are written."""
    torch.manual_seed(1)
    rows, E = sum(sizes), len(sizes)
    x, d = torch.randn(rows, M, device=device).bfloat16(), torch.randn(rows, N, device=device).bfloat16()
    md = ragged(sizes, rows, device)
    for skip in (0, 1, 8):
        room = torch.full((E, M + 3, N + 16), 5.0, device=device)
        c = room[:, 1:1 + M, skip:skip + N]
        assert matmul(x.t(), d, None, md, md, c=c) is c
        check(c, x, d, sizes, torch.float32)
        c.fill_(5.0)
        assert bool((room == 5).all())


def test_values_of_other_slices_do_not_reach(device):
    """NaN and infinities in a slice's rows make that slice's results NaN or infinite, and only in their columns."""
    sizes = [40, 33, 60]
    x, d = torch.randn(133, 136, device=device).half(), torch.randn(133, 264, device=device).half()
    md = ragged(sizes, 133, device)
    clean = matmul(x.t(), d, None, md, md)
    x[40:73, 5] = float("nan")
    d[72, 200] = float("inf")
    got = matmul(x.t(), d, None, md, md)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert bool(torch.isnan(got[1][5]).all()) and not bool(torch.isfinite(got[1][:, 200]).any())
    keep = torch.ones(136, 264, dtype=torch.bool, device=device)
    keep[5], keep[:, 200] = False, False
    assert torch.equal(got[1][keep], clean[1][keep])


@pytest.mark.parametrize("M,N,rows,E", [(0, 8, 10, 2), (8, 0, 10, 2), (8, 8, 0, 2), (16, 24, 0, 1)])
def test_nothing_there(M, N, rows, E, device):
    md = ragged([rows] + [0] * (E - 1), rows, device)
    got = matmul(torch.randn(rows, M, device=device).bfloat16().t(), torch.randn(rows, N, device=device).bfloat16(), None, md, md)
    assert tuple(got.shape) == (E, M, N) and not bool(got.any() if rows == 0 else False)


def test_offsets_past_the_rows_are_cut(device):
    """Metadata made for more rows than there are: what is there is summed, nothing else is read."""
    x, d = torch.randn(50, 64, device=device).bfloat16(), torch.randn(50, 64, device=device).bfloat16()
    md = ragged([30, 40, 50], 120, device)
    check(matmul(x.t(), d, None, md, md), x, d, [30, 20, 0], torch.bfloat16)


def test_padded_slices(device):
    """Slices that begin on multiples of 64, with NaN in the rows between them: only a slice's own rows are summed."""
    sizes, starts = [40, 0, 64, 3], [0, 64, 64, 128]
    x, d = torch.full((200, 72), float("nan"), device=device).bfloat16(), torch.full((200, 136), float("nan"), device=device).bfloat16()
    for n, at in zip(sizes, starts):
        x[at:at + n], d[at:at + n] = torch.randn(n, 72, device=device), torch.randn(n, 136, device=device)
    md = ragged(sizes, 200, device)
    md.slice_offs = torch.tensor([*starts, 192], dtype=torch.int32, device=device)
    rows = torch.cat([torch.arange(at, at + n) for n, at in zip(sizes, starts)]).to(device)
    check(matmul(x.t(), d, None, md, md), x[rows], d[rows], sizes, torch.bfloat16)


def test_rows_past_four_gigabytes(device):
    """A slice whose rows lie beyond what 32 bits count."""
    rows, M, N = 2 ** 19 + 100, 4352, 64
    x, d = torch.zeros(rows, M, dtype=torch.bfloat16, device=device), torch.zeros(rows, N, dtype=torch.bfloat16, device=device)
    x[-100:], d[-100:] = torch.randn(100, M, device=device), torch.randn(100, N, device=device)
    sizes = [rows - 100 - 7, 7, 100]
    md = ragged(sizes, rows, device)
    got = matmul(x.t(), d, None, md, md)
    assert not bool(got[:2].any())
    check(got[2:], x[-100:], d[-100:], [100], torch.bfloat16)


def test_another_stream_and_a_graph(device):
    torch.manual_seed(2)
    for M, N in ((136, 264), (64, 64)):     # (64 x 64: with partial sums)
        x, d = torch.randn(2000, M, device=device).bfloat16(), torch.randn(2000, N, device=device).bfloat16()
        md = ragged([1100, 900], 2000, device)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            mine = matmul(x.t(), d, None, md, md)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(mine, matmul(x.t(), d, None, md, md))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = matmul(x.t(), d, None, md, md)
        for _ in range(4):
            x.copy_(torch.randn(2000, M, device=device))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, matmul(x.t(), d, None, md, md))


def test_results_that_are_too_large(device):
    """2^24 rows or columns and more are refused, before anything is made of them."""
    md = ragged([2], 2, device)
    for n in (2 ** 24, 2 ** 32 + 8):
        wide, d = torch.zeros(1, 1, dtype=torch.bfloat16, device=device).expand(2, n), torch.zeros(2, 8, dtype=torch.bfloat16, device=device)
        for a, b in ((wide.t(), d), (d.t(), wide)):
            with pytest.raises(NotImplementedError):
                matmul(a, b, None, md, md)


def overlapping(rows, C, dtype, device, step):
    """[rows, C] whose rows begin `step` elements after each other: one row again and again, or a window that slides."""
    return torch.randn((rows - 1) * step + C if rows else 0, device=device).to(dtype).as_strided((rows, C), (step, 1))


@pytest.mark.parametrize("sizes", [[1], [5, 1, 0, 40], [40, 3], [64, 31, 33], [3000, 9, 700]], ids=str)
@pytest.mark.parametrize("M,N", [(8, 16), (64, 136), (33, 72)])
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.float32), (torch.float16, None)])
def test_rows_that_overlap(M, N, sizes, dtype, out, device):
    """Expanded operands and sliding windows, one of them or both: a slice sums its own rows, not those that its last stage reaches."""
    torch.manual_seed(M + len(sizes))
    rows = sum(sizes)
    dense = lambda C: torch.randn(rows, C, device=device).to(dtype)  # noqa: E731
    md = ragged(sizes, rows, device)
    for step in (0, 8):
        for x, d in ((overlapping(rows, M, dtype, device, step), dense(N)), (dense(M), overlapping(rows, N, dtype, device, step)),
                     (overlapping(rows, M, dtype, device, step), overlapping(rows, N, dtype, device, step))):
            check(matmul(x.t(), d, None, md, md, precision_config=PrecisionConfig(out_dtype=out)), x, d, sizes, out or dtype)


def test_gradient_of_a_bias(device):
    """Ones times the gradient of a sum over tokens, both expanded: whole numbers, exactly."""
    for sizes in ([40, 3], [40, 0, 1, 300]):
        K, md = sum(sizes), ragged(sizes, sum(sizes), device)
        one, dy = torch.ones(1, 8, dtype=torch.bfloat16, device=device).expand(K, 8), torch.ones(1, 16, dtype=torch.bfloat16, device=device).expand(K, 16)
        got = matmul(one.t(), dy, None, md, md, precision_config=PrecisionConfig(out_dtype=torch.float32))
        assert torch.equal(got, torch.tensor(sizes, device=device).float()[:, None, None].expand(-1, 8, 16))


def test_overlapping_rows_behind_a_slice_do_not_reach(device):
    """A window that slides over NaN behind the first slice's rows, times whole rows: the first slice is clean."""
    sizes = [40, 25]
    flat = torch.randn(64 * 8 + 64, device=device).bfloat16()
    flat[39 * 8 + 64:] = float("nan")                       # (what the first forty windows do not reach)
    windows, whole = flat.as_strided((65, 64), (8, 1)), torch.randn(65, 72, device=device).bfloat16()
    md = ragged(sizes, 65, device)
    for x, d in ((windows, whole), (whole, windows)):
        got = matmul(x.t(), d, None, md, md)
        check(got[:1], x[:40], d[:40], [40], torch.bfloat16)
        assert bool(torch.isnan(got[1]).any())


@pytest.mark.parametrize("M,N,sizes", [(4100, 2624, [320, 350, 0, 700, 400]), (2600, 4160, [333, 650, 0, 700]), (136, 128, [40, 0, 50]), (300, 192, [500, 9])])
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float16, torch.float16)])
def test_results_on_whole_lines(M, N, sizes, dtype, out, device):
    """Rows of results that begin on lines of 128 bytes, with M no whole tiles: the large tiles of both shapes, and small ones; and rows that end inside a line, or a
    piece, with nothing written behind them."""
    torch.manual_seed(M + N)
    rows, E = sum(sizes), len(sizes)
    x, d = torch.randn(rows, M, device=device).to(dtype), torch.randn(rows, N, device=device).to(dtype)
    md = ragged(sizes, rows, device)
    assert N * out.itemsize % 128 == 0
    got = matmul(x.t(), d, None, md, md, precision_config=PrecisionConfig(out_dtype=out))
    check(got, x, d, sizes, out)
    for less in (1, 13, 40):
        room = torch.full((E, M, N), 5.0, dtype=out, device=device)
        c, fewer = room[:, :, :N - less], d[:, :N - less]
        assert c.data_ptr() % 128 == 0
        matmul(x.t(), fewer, None, md, md, c=c)
        check(c, x, fewer, sizes, out)
        assert bool((room[:, :, N - less:] == 5).all())


@pytest.mark.parametrize("sizes", [[1], [2, 3, 0, 40], [700]], ids=str)
@pytest.mark.parametrize("scale", [1e-4, 1e-5, 1e-6])
def test_subnormal_float16(sizes, scale, device):
    """Products that are added at the place of the largest, for which a number below 2^-14 counts as 2^-14: every one of n products, the running sum and the last
    rounding are off by a step of float32 at most at that place.  One row alone is exact."""
    torch.manual_seed(len(sizes))
    rows = sum(sizes)
    md = ragged(sizes, rows, device)
    x, d = (scale * torch.randn(rows, 136, device=device)).half(), torch.randn(rows, 264, device=device).half()
    for a, b in ((x, d), (d, x), (x, x)):
        got, at = matmul(a.t(), b, None, md, md, precision_config=PrecisionConfig(out_dtype=torch.float32)), 0
        for e, n in enumerate(sizes):
            p, q = a[at:at + n].double().t().contiguous(), b[at:at + n].double()
            bound = 2 * (n + 2) * 2.0 ** -24 * (p.abs().clamp(min=2.0 ** -14) @ q.abs().clamp(min=2.0 ** -14)) if n > 1 else 0.0
            assert bool(((got[e].double() - p @ q).abs() <= bound).all()), (e, n)
            at += n
