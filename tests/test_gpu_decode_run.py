"""GPU: steps of generation from `moe_layer`, `matvec` and `sample` as they are used: each operator against its definition on what the one
before it gave, the same steps from a captured graph, and a batch with rows that no request is in."""
import pytest
import torch

import test_gpu_matvec
import test_gpu_sampling
from test_gpu_moe_layer import Layer
from triton_amd.matvec import matvec
from triton_amd.sampling import sample

pytestmark = pytest.mark.gpu
E, K_PICKS, H, I, V = 12, 3, 256, 160, 40007


class Model:
    """An embedding, two expert layers with residuals, and a head of 4-bit weights."""

    def __init__(self, device):
        g = torch.Generator().manual_seed(0)
        self.embedding = torch.randn(V, H, generator=g).to(torch.bfloat16).to(device)
        self.routers = [(0.1 * torch.randn(H, E, generator=g)).to(device) for _ in range(2)]
        self.layers = [Layer(device, E, H, I, seed=n, spread=0.1) for n in (1, 2)]
        self.head, self.head64, self.head_size = test_gpu_matvec.make(H, V, 64, True, torch.bfloat16, device)

    def step(self, tokens, u, seen=None, **settings):
        x = self.embedding[tokens.clamp(min=0)]   # (fewer than 64 rows: one kernel, no synchronization)
        for router, layer in zip(self.routers, self.layers):
            logits = x.float() @ router
            y = layer.call(x, logits, K_PICKS, ("blocks", "strided"), ("shuffled", "strided"))
            if seen is not None:
                seen.append((layer, x, logits, y))
            x = x + 0.05 * y
        logits = matvec(x, self.head, out_dtype=torch.float32)
        token = sample(logits, u, **settings)
        if seen is not None:
            seen.append((x, logits, token))
        return token.long()


@pytest.mark.parametrize("T", [1, 5, 17, 64])
def test_every_operator_on_what_the_last_one_gave(T, device):
    m = Model(device)
    tokens = torch.arange(T, device=device) * 601
    settings = test_gpu_sampling.settings(T, device, 6)
    for n in range(2):
        u, seen = test_gpu_sampling.uniform(T, device, seed=n), []
        tokens = m.step(tokens, u, seen, **settings)
        for layer, x, logits, y in seen[:2]:
            layer.check(y, x, logits, K_PICKS)
        x, logits, token = seen[2]
        test_gpu_matvec.check(logits, x, m.head64, m.head_size)
        test_gpu_sampling.check(logits, u, **settings)
        assert torch.equal(token.long(), tokens) and tokens.min() >= 0


def test_captured_steps(device):
    """A step captured once and replayed token by token writes what eager steps write."""
    m, T = Model(device), 6
    settings = dict(temperature=0.9, top_k=50, top_p=0.95)
    u = torch.empty(T, device=device)
    start = torch.arange(T, device=device) * 77
    numbers = [test_gpu_sampling.uniform(T, device, seed=40 + n) for n in range(5)]
    want, tokens = [], start
    for n in numbers:
        tokens = m.step(tokens, n, **settings)
        want.append(tokens)
    held = start.clone()
    u.copy_(numbers[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(held, u, **settings)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.copy_(m.step(held, u, **settings))
    for _ in range(2):
        held.copy_(start)
        for n, w in zip(numbers, want):
            u.copy_(n)
            graph.replay()
            assert torch.equal(held, w)
            m.step(start, u, **settings)   # eager work in between


def test_rows_without_a_request(device):
    """What lies in rows of the batch that no request is in -- NaN, infinities -- does not reach the others."""
    m, T = Model(device), 9
    u = test_gpu_sampling.uniform(T, device)
    layer, head = m.layers[0], m.head
    x = m.embedding[:T].clone()
    logits = x.float() @ m.routers[0]
    want = layer.call(x, logits, K_PICKS)
    for junk in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).max):
        x2, l2 = x.clone(), logits.clone()
        x2[[2, 7]], l2[[2]] = junk, float("nan")
        y = layer.call(x2, l2, K_PICKS)
        keep = [0, 1, 3, 4, 5, 6, 8]
        assert torch.equal(y[keep], want[keep])
        z, z_want = matvec(y, head, out_dtype=torch.float32), matvec(want, head, out_dtype=torch.float32)
        assert torch.equal(z[keep], z_want[keep])
        assert torch.equal(sample(z, u, top_p=0.9)[keep], sample(z_want, u, top_p=0.9)[keep])
