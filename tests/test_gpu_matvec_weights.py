"""GPU: `matvec` refuses weights that are not of the types that `pack_int4` gives them, instead of reading their bytes as if they were."""
import pytest
import torch

from test_gpu_matvec import make, rows
from triton_amd.matvec import Int4Weights, matvec

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [False, True])
def test_types(out, device):
    w, _, _ = make(256, 40, 64, True, torch.bfloat16, device)
    x = rows(3, 256, torch.bfloat16, device)
    want = matvec(x, w)
    call = lambda v: matvec(x, v, out=torch.empty_like(want) if out else None)  # noqa: E731
    assert torch.equal(call(Int4Weights(w.data, w.scales, w.zeros, w.shape, w.group_size)), want)
    for data, scales, zeros in ((w.data.int(), w.scales, w.zeros), (w.data.view(torch.int8), w.scales, w.zeros), (w.data, w.scales, w.zeros.int()),
                                (w.data, w.scales, w.zeros.to(torch.bfloat16)), (w.data, w.scales.float(), w.zeros), (w.data, w.scales.double(), w.zeros)):
        with pytest.raises(AssertionError, match="pack_int4"):
            call(Int4Weights(data, scales, zeros, w.shape, w.group_size))
