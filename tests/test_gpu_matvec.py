"""GPU: `matvec` with the weights of `pack_int4` against the formula in 64 bits.

The bound of an element is derived: a group's float32 sums (of x, and of x (16 + q) behind it) pass at most 2 * (128 + 8) additions, each off by
at most 2^-24 of the magnitudes added up, |x| (16 + q + 16 + z), the sum over the groups at most 136 more (K <= 4096 with groups of 32): 408 of them
stay below 2^-15 of |s| |x| (32 + q + z); the result is rounded once, by at most half a step."""
import pytest
import torch

from triton_amd.matvec import Int4Weights, matvec, pack_int4

pytestmark = pytest.mark.gpu


def make(K, N, group, zeros, scale_dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (K // 2, N), dtype=torch.uint8, generator=g)
    scales = (0.02 * torch.randn(K // group, N, generator=g)).to(scale_dtype)
    z = torch.randint(0, 16, (K // group, N), dtype=torch.uint8, generator=g) if zeros else None
    q = torch.stack([codes & 15, codes >> 4], 1).reshape(K, N).double()
    s64 = scales.double().repeat_interleave(group, 0)
    z64 = torch.full((K, N), 8.0, dtype=torch.float64) if z is None else z.double().repeat_interleave(group, 0)
    w = pack_int4(codes.to(device), scales.to(device), None if z is None else z.to(device), group)
    return w, (q - z64) * s64, (32 + q + z64) * s64.abs()


def rows(M, K, dtype, device, seed=1):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def check(y, x, dense, mag, bias=None):
    want = x.cpu().double() @ dense
    err = 2.0**-15 * (x.cpu().double().abs() @ mag)
    if bias is not None:
        want, err = want + bias.cpu().double(), err + 2.0**-24 * bias.cpu().double().abs()
    off, bound = (y.cpu().double() - want).abs(), err + (want.abs() + err) * torch.finfo(y.dtype).eps / 2
    assert torch.isfinite(y).all() and (off <= bound).all(), f"{(off / bound).max():.2f} of the bound"


@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("M,K,N,dtype,scale", [
    (1, 128, 16, torch.bfloat16, torch.bfloat16), (1, 128, 1, torch.float16, torch.float16), (2, 384, 17, torch.bfloat16, torch.float16),
    (15, 1152, 100, torch.float16, torch.bfloat16), (16, 4096, 33, torch.bfloat16, torch.bfloat16), (17, 256, 48, torch.float16, torch.float16),
    (32, 640, 31, torch.bfloat16, torch.bfloat16), (33, 2176, 64, torch.float16, torch.float16), (64, 512, 130, torch.bfloat16, torch.float16),
    (65, 256, 20, torch.bfloat16, torch.bfloat16), (200, 128, 19, torch.float16, torch.float16)])
def test_product(M, K, N, dtype, scale, group, zeros, device):
    w, dense, mag = make(K, N, group, zeros, scale, device)
    x = rows(M, K, dtype, device)
    for out in (dtype, torch.float32):
        y = matvec(x, w, out_dtype=out)
        assert y.dtype == out and tuple(y.shape) == (M, N)
        check(y, x, dense, mag)


@pytest.mark.parametrize("K,group", [(32, 32), (96, 32), (160, 32), (1056, 32), (64, 64), (192, 64), (1088, 64)])
def test_last_block_not_whole(K, group, device):
    for M in (1, 20, 40):
        w, dense, mag = make(K, 50, group, True, torch.bfloat16, device)
        x = rows(M, K, torch.bfloat16, device)
        check(matvec(x, w, out_dtype=torch.float32), x, dense, mag)


def test_wide_and_many_strips(device):
    w, dense, mag = make(256, 20011, 64, True, torch.float16, device)
    for M in (1, 3, 50):
        x = rows(M, 256, torch.float16, device)
        check(matvec(x, w, out_dtype=torch.float32), x, dense, mag)


@pytest.mark.parametrize("bias", [torch.float32, torch.bfloat16, torch.float16])
def test_bias_and_types(bias, device):
    w, dense, mag = make(256, 70, 128, False, torch.bfloat16, device)
    b = torch.randn(70).to(bias).to(device)
    for x_type, out in ((torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16), (torch.bfloat16, None)):
        x = rows(5, 256, x_type, device)
        y = matvec(x, w, b, out_dtype=out)
        assert y.dtype == (out or x_type)
        check(y, x, dense, mag, b)


def test_a_vector_strides_and_output(device):
    w, dense, mag = make(320, 40, 64, True, torch.bfloat16, device)
    x = rows(6, 320, torch.bfloat16, device)
    want = matvec(x, w)
    one = matvec(x[2], w)
    assert tuple(one.shape) == (40,) and torch.equal(one, want[2])
    wide = torch.zeros(6, 700, dtype=x.dtype, device=device)
    for at in (16, 5):
        wide[:, at:at + 320] = x
        assert torch.equal(matvec(wide[:, at:at + 320], w), want)
    assert torch.equal(matvec(x.t().contiguous().t(), w), want)
    assert torch.equal(matvec(x[:1].expand(6, 320), w), want[:1].expand(6, 40))
    far = torch.empty(5 * (1 << 28) + 320, dtype=x.dtype, device=device).as_strided((6, 320), (1 << 28, 1))
    far.copy_(x)
    assert torch.equal(matvec(far, w), want)
    out = torch.full((6, 64), 3.0, dtype=torch.float32, device=device)
    got = matvec(x, w, out=out[:, 8:48])
    assert got.data_ptr() == out[:, 8:].data_ptr() and torch.equal(out[:, 8:48], matvec(x, w, out_dtype=torch.float32))
    assert (out[:, :8] == 3).all() and (out[:, 48:] == 3).all()
    bias = torch.randn(80, device=device)[::2]
    assert torch.equal(matvec(x, w, bias), matvec(x, w, bias.contiguous()))
    assert matvec(x[:0], w).shape == (0, 40)


def test_special_values(device):
    """Scales of zero, a whole column of zero points, rows that are not finite: those rows alone."""
    w, dense, mag = make(256, 48, 64, True, torch.bfloat16, device)
    x = rows(4, 256, torch.bfloat16, device)
    want = matvec(x, w, out_dtype=torch.float32)
    bad = x.clone()
    bad[1, 7], bad[2, 200] = float("nan"), float("inf")
    y = matvec(bad, w, out_dtype=torch.float32)
    assert torch.equal(y[[0, 3]], want[[0, 3]]) and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    zero = Int4Weights(w.data, torch.zeros_like(w.scales), w.zeros, w.shape, w.group_size)
    assert (matvec(x, zero) == 0).all()


def test_unpack_gives_back(device):
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 256, (48, 37), dtype=torch.uint8, generator=g).to(device)
    scales = torch.randn(3, 37, generator=g).to(torch.float16).to(device)
    zeros = torch.randint(0, 16, (3, 37), dtype=torch.uint8, generator=g).to(device)
    for z in (zeros, None):
        w = pack_int4(codes.t().contiguous().t(), scales, z, 32)
        c, s, back = w.unpack()
        assert torch.equal(c, codes) and torch.equal(s, scales) and (back is None if z is None else torch.equal(back, z))


def test_repeated_streams_and_a_graph(device):
    w, dense, mag = make(1024, 300, 32, True, torch.bfloat16, device)
    x = rows(9, 1024, torch.bfloat16, device)
    want = matvec(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(matvec(x, w), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = matvec(x, w)
    for seed in (4, 5, 6):
        x.copy_(rows(9, 1024, torch.bfloat16, device, seed))
        graph.replay()
        assert torch.equal(y, matvec(x, w))


def test_refusals(device):
    w, _, _ = make(128, 16, 64, False, torch.bfloat16, device)
    x = rows(2, 128, torch.bfloat16, device)
    for call in (lambda: matvec(x.float(), w), lambda: matvec(x, w, out_dtype=torch.float64), lambda: matvec(x, w, torch.zeros(16, device=device, dtype=torch.float64))):
        with pytest.raises(NotImplementedError):
            call()
    for call in (lambda: matvec(x[:, :64], w), lambda: matvec(x, w, torch.zeros(15, device=device)), lambda: matvec(x, w, out=torch.zeros(2, 15, device=device)),
                 lambda: matvec(x, Int4Weights(w.data, w.scales, None, (256, 16), 64)), lambda: matvec(x, w, torch.zeros(16))):
        with pytest.raises(AssertionError):
            call()
