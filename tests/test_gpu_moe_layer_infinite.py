"""GPU: `moe_layer` where h passes float32's range (bfloat16) or float16's: an infinite h times positive weights is infinite, as in the formula, for every
way in which the waves of the down projection share K, and the other tokens keep their bits."""
import pytest
import torch

from test_gpu_moe_layer import Layer, inputs
from triton_amd.numerics_details.mxfp import downcast_to_mxfp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("values,scales", [("strided", "strided"), ("blocks", "shuffled")])
@pytest.mark.parametrize("T,E,k", [(1, 4, 1), (4, 4, 2), (20, 16, 2), (40, 4, 2), (64, 128, 4)])
@pytest.mark.parametrize("H,I", [(32, 32), (64, 160), (64, 384), (32, 1056), (32, 2048), (32, 3200), (512, 96)])
def test_infinite_h(H, I, T, E, k, values, scales, device):
    layer = Layer(device, E, H, I, bias=None)
    for n, (K, N) in enumerate(((H, 2 * I), (I, H))):
        v, s = downcast_to_mxfp(torch.ones(E, K, N, dtype=torch.bfloat16, device=device), torch.uint8, axis=-2)
        layer.w[n].copy_(v)
        layer.s[n].copy_(s)
    for dtype, large in ((torch.bfloat16, 1e30), (torch.float16, 6e4)):
        x, logits = inputs(T, E, H, dtype, device)
        x *= 0.01
        call = lambda: layer.call(x, logits, k, (values, values), (scales, scales), alpha=1.0, limit=None)  # noqa: E731
        good = call()
        x[T // 2] = large
        y = call()
        others = [t for t in range(T) if t != T // 2]
        assert torch.isfinite(good).all() and (y[T // 2] == float("inf")).all() and torch.equal(y[others], good[others])
