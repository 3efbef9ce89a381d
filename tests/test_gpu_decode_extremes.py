"""GPU: the smallest and largest calls of `moe_layer`, `matvec` and `sample`: one expert, long inner dimensions, rows far apart, many rows."""
import pytest
import torch

import test_gpu_matvec
import test_gpu_sampling
from test_gpu_moe_layer import Layer, inputs
from triton_amd.matvec import matvec
from triton_amd.sampling import sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 17, 64])
def test_one_expert(T, device):
    layer = Layer(device, 1, 64, 96)
    x, logits = inputs(T, 1, 64, torch.bfloat16, device)
    layer.check(layer.call(x, logits, 1), x, logits, 1)


def test_sixteen_picks_of_five_hundred_experts(device):
    layer = Layer(device, 512, 32, 32)
    x, logits = inputs(32, 512, 32, torch.float16, device)
    layer.check(layer.call(x, logits, 16, ("blocks", "strided"), ("shuffled", "strided")), x, logits, 16)


@pytest.mark.parametrize("M", [1, 7, 16, 20, 64])
def test_long_rows(M, device):
    """131072 K: a wave adds up 128 groups, as many as the bound's, and the eight waves are added as there."""
    w, dense, mag = test_gpu_matvec.make(131072, 40, 128, True, torch.bfloat16, device)
    x = test_gpu_matvec.rows(M, 131072, torch.bfloat16, device)
    test_gpu_matvec.check(matvec(x, w, out_dtype=torch.float32), x, dense, mag)


@pytest.mark.parametrize("M,N", [(5, 48), (40, 48), (64, 5000), (64, 34000)])
def test_rows_of_x_and_y_far_apart(M, N, device):
    """x as far apart as is read in place, and an output whose rows lie past 32 bits."""
    w, _, _ = test_gpu_matvec.make(256, N, 64, True, torch.float16, device)
    x = test_gpu_matvec.rows(M, 256, torch.bfloat16, device)
    want = matvec(x, w)
    step = (1 << 23) - 8
    far = torch.empty((M - 1) * step + 256, dtype=x.dtype, device=device).as_strided((M, 256), (step, 1))
    far.copy_(x)
    assert torch.equal(matvec(far, w), want)
    out = torch.empty((M - 1) * (1 << 27) + N, dtype=x.dtype, device=device).as_strided((M, N), (1 << 27, 1))
    matvec(far, w, out=out)
    assert torch.equal(out, want)


def test_logits_far_apart(device):
    V = 40000
    z = test_gpu_sampling.normal(3, V, torch.bfloat16, device)
    u, settings = test_gpu_sampling.uniform(3, device), dict(temperature=0.8, top_k=30, top_p=0.9)
    far = torch.empty(2 * ((1 << 30) + 1) + V, dtype=z.dtype, device=device).as_strided((3, V), ((1 << 30) + 1, 1))
    far.copy_(z)
    assert torch.equal(sample(far, u, **settings), sample(z, u, **settings))


def test_more_rows_than_go_at_once(device):
    """4200 rows that several workgroups share: in two rounds of launches over one workspace."""
    R, V = 4200, 26000
    z = torch.randn(R, V, generator=torch.Generator(device=device).manual_seed(1), device=device, dtype=torch.bfloat16)
    u, s = test_gpu_sampling.uniform(R, device), test_gpu_sampling.settings(R, device, 3)
    together = sample(z, u, **s)
    for a, b in ((0, 40), (4080, 4130), (4190, 4200)):
        assert torch.equal(together[a:b], sample(z[a:b], u[a:b], **{n: v[a:b] for n, v in s.items()}))
    few = torch.tensor([0, 1, 4095, 4096, 4199], device=device)
    test_gpu_sampling.check(z[few], u[few], **{n: v[few] for n, v in s.items()})


def test_very_many_short_rows(device):
    z = torch.randn(100003, 33, generator=torch.Generator(device=device).manual_seed(2), device=device)
    u = test_gpu_sampling.uniform(100003, device)
    got = sample(z, u, top_k=4)
    for at in (0, 65535, 65536, 100002):
        assert got[at].item() == sample(z[at:at + 1], u[at:at + 1], top_k=4).item()
    assert torch.equal(sample(z, u, temperature=0.0).long(), z.argmax(1))
