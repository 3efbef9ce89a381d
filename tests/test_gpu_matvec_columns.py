"""GPU: `matvec` of more than a few rows and so many columns that waves have strips of their own, against the formula in 64 bits
(the bound is the one of test_gpu_matvec: no element passes more additions here, and two parts of K meet in one more)."""
import pytest
import torch

from test_gpu_matvec import check, make, rows
from triton_amd.matvec import matvec

pytestmark = pytest.mark.gpu


def columns(device, extra, strips=5):
    """Columns of so many strips of 16 per CU, and `extra`: from two on waves have a strip of their own, from five on two."""
    return 16 * strips * torch.cuda.get_device_properties(device).multi_processor_count + extra


@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("M,K,extra,dtype", [(17, 128, 0, torch.bfloat16), (33, 384, 1, torch.float16), (64, 256, 19, torch.bfloat16), (48, 512, 113, torch.float16),
                                             (70, 640, 40, torch.bfloat16)])
def test_product(M, K, extra, dtype, group, zeros, device):
    w, dense, mag = make(K, columns(device, extra), group, zeros, torch.bfloat16, device)
    x = rows(M, K, dtype, device)
    for out in (dtype, torch.float32):
        check(matvec(x, w, out_dtype=out), x, dense, mag)


@pytest.mark.parametrize("K,group", [(32, 32), (96, 32), (160, 32), (192, 64), (1056, 32)])
def test_last_block_not_whole(K, group, device):
    for strips in (5, 2, 1):
        w, dense, mag = make(K, columns(device, 7 if strips > 1 else -9, strips), group, True, torch.float16, device)
        for M in (20, 40, 61):
            x = rows(M, K, torch.bfloat16, device)
            check(matvec(x, w, out_dtype=torch.float32), x, dense, mag)


def test_padding_is_left_alone(device):
    """Rows of x and of the output lie in wider tensors full of NaN: none comes in, none is written over; a row that is
    not finite stays alone; the same call gives the same bits."""
    N = columns(device, 5)
    w, dense, mag = make(160, N, 32, True, torch.bfloat16, device)
    b = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(device)
    x = rows(50, 160, torch.bfloat16, device)
    wide = torch.full((52, 176), float("nan"), dtype=x.dtype, device=device)
    wide[1:51, 8:168] = x
    out = torch.full((52, N + 24), float("nan"), device=device)
    y = matvec(wide[1:51, 8:168], w, b, out=out[1:51, 8:N + 8])
    check(y, x, dense, mag, b)
    edge = out.clone()
    edge[1:51, 8:N + 8] = float("nan")
    assert torch.isnan(edge).all()
    bad = x.clone()
    bad[7, 3] = float("nan")
    again = matvec(bad, w, b, out_dtype=torch.float32)
    assert torch.isnan(again[7]).all() and torch.equal(again[:7], y[:7]) and torch.equal(again[8:], y[8:])


@pytest.mark.parametrize("M,group", [(9, 32), (12, 128), (16, 64)])
def test_rows_whose_inner_dimension_is_long(M, group, device):
    w, dense, mag = make(6272, columns(device, 9), group, True, torch.bfloat16, device)
    x = rows(M, 6272, torch.float16, device)
    check(matvec(x, w), x, dense, 2 * mag)   # (6272 rows pass half as many groups again as the bound's 4096)


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, False), (128, True)])
@pytest.mark.parametrize("M,K,strips,extra,dtype", [(17, 128, 2, 1, torch.bfloat16), (33, 384, 2, 50, torch.float16), (64, 1152, 3, 0, torch.bfloat16),
                                                    (130, 256, 4, 15, torch.bfloat16), (40, 256, 1, 1, torch.float16), (64, 256, 2, 0, torch.bfloat16),
                                                    (20, 1152, 1, 0, torch.bfloat16), (48, 384, 1, 0, torch.float16), (61, 128, 1, -7, torch.float16),
                                                    (25, 2176, 1, 17, torch.bfloat16)])
def test_fewer_strips(M, K, strips, extra, dtype, group, zeros, device):
    w, dense, mag = make(K, columns(device, extra, strips), group, zeros, torch.float16, device)
    x = rows(M, K, dtype, device)
    for out in (dtype, torch.float32):
        check(matvec(x, w, out_dtype=out), x, dense, mag)
