"""GPU: `sample` of a row by one workgroup and by the launches that share a row out: the same token, and the definition's."""
import numpy as np
import pytest
import torch

from test_gpu_sampling import INF, check, normal, settings, uniform
from triton_amd.sampling import sample

pytestmark = pytest.mark.gpu


def rows_of(kind, V, dtype, device):
    z = normal(12, V, torch.float32, device, seed=5)
    if kind == "ties":
        z = (2 * z).round() / 2
    elif kind == "flat":
        z = torch.zeros_like(z) + 1e-4 * z
    elif kind == "equal":
        z = torch.full_like(z, 0.5)
    elif kind == "infinite":
        z[:, 7::1001] = INF
        z[3] = -INF
        z[4, 1:] = -INF
        z[5, ::2] = float("nan")
    elif kind == "masked":
        z[:, torch.arange(V, device=device) % 3 != 1] = torch.finfo(torch.float32).min
    return z.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["normal", "ties", "flat", "equal", "infinite", "masked"])
def test_same_token_either_way(kind, dtype, device):
    """20001 logits are one workgroup's; with 12766 behind them that nobody may draw several workgroups share the row.  (Both lengths
    leave the weights as many bits.)"""
    V = 20001
    z = rows_of(kind, V, dtype, device)
    padded = torch.full((12, 32767), -INF, dtype=dtype, device=device)
    padded[:, :V] = z
    u = uniform(12, device, seed=9)
    for seed in range(4):
        s = settings(12, device, seed)
        alone = sample(z, u, **s)
        assert torch.equal(alone, sample(padded, u, **s)), (kind, seed)
        each = torch.cat([sample(padded[i:i + 1], u[i:i + 1], **{n: v[i:i + 1] for n, v in s.items()}) for i in range(12)])
        assert torch.equal(alone, each)


@pytest.mark.parametrize("R,V", [(2, 16385), (3, 24000), (3, 24001), (2, 40000), (260, 9001), (300, 26000)])
def test_lengths_at_the_borders(R, V, device):
    check(normal(R, V, torch.float32, device, seed=V), uniform(R, device, seed=R), **settings(R, device, R))


def test_the_longest_row(device):
    V = 1 << 20
    z = normal(2, V, torch.float32, device, seed=3)
    check(z, uniform(2, device), temperature=0.9, top_k=0, top_p=0.95, min_p=0.0)
    many = normal(1, V, torch.float32, device, seed=4).expand(300, V)   # (rows on one another: a stride of zero)
    u = torch.linspace(0, 0.999, 300, device=device)
    few = torch.cat([sample(many[:1], u[i:i + 1], 0.9, 0, 0.95) for i in (0, 57, 299)])
    assert torch.equal(sample(many, u, 0.9, 0, 0.95)[[0, 57, 299]], few)


def test_row_by_row_or_together(device):
    """A row's token depends on neither the batch nor the rows beside it."""
    z, u = normal(600, 30011, torch.bfloat16, device, seed=8), uniform(600, device, seed=2)
    s = settings(600, device, 4)
    together = sample(z, u, **s)
    for i in (0, 1, 255, 256, 511, 599):
        assert together[i].item() == sample(z[i:i + 1], u[i:i + 1], **{n: v[i:i + 1] for n, v in s.items()}).item()
    assert np.array_equal(together[100:140].cpu().numpy(), sample(z[100:140], u[100:140], **{n: v[100:140] for n, v in s.items()}).cpu().numpy())
