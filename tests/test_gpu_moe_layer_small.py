"""GPU: `moe_layer` with activations so small that h lies among float16's smallest values, against the layer's definition in 64 bits (bound of
test_gpu_moe_layer; a rounding to float16 is off by half a step, which is 2^-25 below 2^-14)."""
import pytest
import torch

from test_gpu_moe_layer import Layer, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("values,scales", [("strided", "strided"), ("blocks", "shuffled")])
@pytest.mark.parametrize("size", [2.0**-2, 2.0**-6, 2.0**-10, 2.0**-13, 2.0**-16])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 32, 32), (3, 8, 4, 160, 1120), (9, 4, 1, 64, 288), (20, 4, 2, 96, 416)])
def test_small_activations(T, E, k, H, I, size, values, scales, device):
    layer = Layer(device, E, H, I, bias=None, spread=2.0)
    for dtype in (torch.float16, torch.bfloat16):
        x, logits = inputs(T, E, H, torch.float32, device)
        x = (x * size / 16).to(dtype)
        got = layer.call(x, logits, k, (values, values), (scales, scales))
        want, err = layer.expected(x, logits, k)
        least = 2.0**-25 if dtype == torch.float16 else 0.0
        if dtype == torch.float16:   # (h to a multiple of 2^-35, an error of 2^-36 each)
            err = err + 2.0**-36 * max(d.abs().sum(0).max().item() for d in layer.dense[1]) * k
        bound = err + ((want.abs() + err) * torch.finfo(dtype).eps / 2).clamp(min=least)
        off = (got.cpu().double() - want).abs()
        assert (off <= bound).all(), f"{(off / bound).max():.2f} of the bound"
