"""GPU: `matvec` of rows at the ends of bfloat16's and float16's range, through every kernel, against the formula in 64 bits (bound of test_gpu_matvec)."""
import pytest
import torch

from test_gpu_matvec import check, make
from test_gpu_matvec_columns import columns
from triton_amd.matvec import matvec, pack_int4

pytestmark = pytest.mark.gpu
# rows in registers (one strip, some in turn), through LDS (4, 8, 16 rows, tiles of 16 and 32, two strips), strips of the waves' own
CALLS = [(1, 384, 40, 0), (16, 512, 3, 3), (16, 4096, 40, 0), (3, 6272, 40, 0), (8, 6272, 40, 0), (16, 6272, 40, 0), (9, 6272, 9, 5), (33, 256, 40, 0), (20, 256, 7, 1),
         (48, 256, 7, 2), (64, 256, 7, 2), (30, 256, 7, 3), (64, 160, 7, 5)]


def weights(K, N, group, zeros, device, size):
    """Scales around `size`."""
    w, dense, mag = make(K, N, group, zeros, torch.bfloat16, device)
    codes, scales, z = w.unpack()
    exact = (scales.double() * (size / 0.02)).to(torch.bfloat16)
    ratio = torch.where(scales == 0, 0.0, exact.double() / scales.double()).repeat_interleave(group, 0).cpu()
    return pack_int4(codes, exact, z, group), dense * ratio, mag * ratio


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("M,K,extra,strips", CALLS)
def test_largest_values(M, K, extra, strips, group, zeros, device):
    """Rows of the largest value, of one sign and of both, one value of that size alone, and an ordinary row beside them."""
    K = -(-K // group) * group
    N = columns(device, extra, strips) if strips else extra
    for dtype, size in ((torch.bfloat16, 2.0**-22), (torch.float16, 2.0**-6)):
        w, dense, mag = weights(K, N, group, zeros, device, size)
        most = torch.finfo(dtype).max
        x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype)
        x[M // 2] = most
        x[M - 1] = most * (1 - 2 * (torch.arange(K) % 2).to(dtype))
        if M > 4:
            x[1] = -most
            x[2, :] = 0
            x[2, K // 3] = most
        x = x.to(device)
        check(matvec(x, w, out_dtype=torch.float32), x, dense, mag)
        if dtype == torch.bfloat16:
            check(matvec(x, w), x, dense, mag)


@pytest.mark.parametrize("M,K,extra,strips", CALLS)
def test_small_values(M, K, extra, strips, device):
    """Values of 2^-117 on, and of bfloat16's smallest normal and subnormal ones: no bits lost."""
    K = -(-K // 64) * 64
    N = columns(device, extra, strips) if strips else extra
    w, dense, mag = weights(K, N, 64, True, device, 2.0**20)
    x = (torch.randn(M, K, generator=torch.Generator().manual_seed(M)).abs() + 1).to(torch.bfloat16) * 2.0**-117
    check(matvec(x.to(device), w, out_dtype=torch.float32), x, dense, mag)
    least = 2.0**-126 * (torch.arange(M * K).view(M, K) % 257 - 128).double() / 128   # (multiples of 2^-133, both signs)
    for least in (least, least * (torch.arange(K) % 61 == 5)):
        x = least.to(torch.bfloat16)
        assert torch.equal(x.double(), least) and x.any()
        check(matvec(x.to(device), w, out_dtype=torch.float32), x, dense, mag)
