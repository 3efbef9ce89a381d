"""GPU: `sample` against its definition in 64 bits: the same tokens, no tolerance.

A token differs only where u times the mass lies within 2^-37 of the row's mass of a border between two tokens (a chance of less than
2^-20 per row of a thousand tokens): the uniform numbers that decide are put in the middle between borders."""
import numpy as np
import pytest
import torch

from triton_amd.sampling import sample

pytestmark = pytest.mark.gpu
INF = float("inf")


def order_of(z):
    z = np.where(np.isnan(z), -np.inf, z)
    order = np.argsort(-z, kind="stable")
    return z[order], order


def kept_of(z, temperature, top_k, top_p, min_p):
    """(weights, tokens) of what a row keeps, in its order."""
    z, order = order_of(z)
    if z[0] == -np.inf:
        return np.zeros(0), order[:0]
    if not temperature > 0:
        return np.ones(1), order[:1]
    with np.errstate(invalid="ignore"):
        w = np.where(z == z[0], 1.0, 0.0 if z[0] == np.inf else np.exp((z - z[0]) / temperature))
    w[z == -np.inf] = 0
    n = len(w) if top_k <= 0 else min(int(top_k), len(w))
    if top_p < 1:
        n = min(n, 1 + int(np.searchsorted(np.cumsum(w[:n]), top_p * w[:n].sum(), side="left")))
    n = max(1, min(n, int((w >= min(min_p, 1.0)).sum())))
    return w[:n], order[:n]


def expected(z, u, temperature, top_k, top_p, min_p):
    w, tokens = kept_of(z, temperature, top_k, top_p, min_p)
    if not len(w):
        return -1
    c = np.cumsum(w)
    return int(tokens[min(len(w) - 1, int(np.searchsorted(c, u * c[-1], side="right")))])


def settings(R, device, seed, **fixed):
    """Per-row settings as the float32 / int32 tensors that the call gets."""
    g = torch.Generator().manual_seed(seed)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (R,), generator=g)]  # noqa: E731
    s = {"temperature": pick(0.0, 0.3, 1.0, 1.7), "top_k": pick(0, 1, 3, 40, 100000).to(torch.int32), "top_p": pick(1.0, 0.97, 0.6, 0.0), "min_p": pick(0.0, 0.0, 0.05, 1.0)}
    s.update({n: torch.full((R,), v, dtype=s[n].dtype) for n, v in fixed.items()})
    return {n: v.to(device) for n, v in s.items()}


def check(logits, u, **s):
    got = sample(logits, u, **s).tolist()
    rows = {n: (v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(len(got), np.float32(v), np.float64)) for n, v in s.items()}
    rows = {**{"temperature": np.ones(len(got)), "top_k": np.zeros(len(got)), "top_p": np.ones(len(got)), "min_p": np.zeros(len(got))}, **rows}
    z, r = logits.double().cpu().numpy(), u.double().cpu().numpy()
    want = [expected(z[i], r[i], *(rows[n][i] for n in ("temperature", "top_k", "top_p", "min_p"))) for i in range(len(got))]
    assert got == want, [(i, g, w) for i, (g, w) in enumerate(zip(got, want)) if g != w][:5]


def normal(R, V, dtype, device, seed=0, spread=2.5):
    return (spread * torch.randn(R, V, generator=torch.Generator().manual_seed(seed))).to(dtype).to(device)


def uniform(R, device, seed=1):
    return torch.rand(R, generator=torch.Generator().manual_seed(seed)).to(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (5, 63), (40, 1000), (9, 4097), (70, 5003), (3, 50001), (300, 257)])
def test_mixed_settings(R, V, dtype, device):
    check(normal(R, V, dtype, device), uniform(R, device), **settings(R, device, 2))


@pytest.mark.parametrize("fixed", [{}, {"temperature": 0.0}, {"top_k": 1}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.95}, {"top_p": 0.0}, {"min_p": 0.1},
                                   {"temperature": 0.25, "top_k": 20, "top_p": 0.5, "min_p": 0.02}, {"top_k": 1 << 30}, {"temperature": 50.0, "top_p": 0.3},
                                   {"temperature": 1e-6}, {"temperature": 3e38}])
def test_settings_for_all_rows(fixed, device):
    for R, V in ((2, 20000), (33, 3001)):
        check(normal(R, V, torch.float32, device), uniform(R, device), **fixed)


@pytest.mark.parametrize("spread", [0.0, 1e-6, 1e-3, 0.1, 30.0, 1e30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_and_steep_rows(spread, dtype, device):
    """All alike (the index decides), nearly alike, a handful of values that thousands share, and rows where one holds everything."""
    R, V = 6, 12345
    check(normal(R, V, dtype, device, spread=spread), uniform(R, device), **settings(R, device, 5, temperature=1.0))


def test_many_ties(device):
    """Four values, thousands of each; top-k and top-p end inside them, at the lower indices."""
    z = torch.randint(0, 4, (12, 30011), generator=torch.Generator().manual_seed(0)).float().to(device)
    u = (torch.arange(12) + 0.37).div(12.1).to(device)
    check(z, u, top_k=10001)
    check(z, u, top_p=0.7123)
    check(z, u, top_k=20000, top_p=0.911, min_p=0.2)
    check(z, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_special_logits(dtype, device):
    z = normal(10, 3000, dtype, device)
    z[0] = -INF
    z[1] = float("nan")
    z[2, 1:] = -INF
    z[3, :2999] = float("nan")
    z[4, [7, 2000, 2500]] = INF
    z[5] = torch.finfo(dtype).min
    z[6, 11] = torch.finfo(dtype).max
    z[7, ::2] = 0.0
    z[7, 1::2] = -0.0
    z[8, torch.rand(3000, generator=torch.Generator().manual_seed(3)).to(device) < 0.9] = -INF
    z[9] = INF
    for s in ({}, {"top_k": 5}, {"top_p": 0.5}, {"min_p": 0.3}, {"temperature": 0.0}, {"temperature": 0.4, "top_p": 0.9}):
        check(z, uniform(10, device), **s)
    assert sample(z, uniform(10, device))[:2].tolist() == [-1, -1]


def test_uniform_numbers_at_the_ends(device):
    z = normal(7, 999, torch.float32, device)
    z[4:] = 1.0
    u = torch.tensor([0.0, 1.0 - 2.0**-24, 0.5, 2.0**-149, 0.0, 1.0 - 2.0**-24, 0.25], device=device)
    check(z, u)
    check(z, u, top_k=3)
    # out of range: as the nearest in range; NaN: 0
    odd = torch.tensor([-1.0, 1.0, 7.0, float("nan"), -0.0, INF, -INF], device=device)
    like = torch.tensor([0.0, 1.0 - 2.0**-24, 1.0 - 2.0**-24, 0.0, 0.0, 1.0 - 2.0**-24, 0.0], device=device)
    assert torch.equal(sample(z, odd, top_k=9), sample(z, like, top_k=9))


def test_settings_out_of_range_in_tensors(device):
    R = 6
    z, u = normal(R, 500, torch.float32, device), uniform(R, device)
    nan = float("nan")
    full = lambda v, t=torch.float32: torch.full((R,), v, dtype=t, device=device)  # noqa: E731
    assert torch.equal(sample(z, u, temperature=full(-2.0)), sample(z, u, temperature=0.0))
    assert torch.equal(sample(z, u, temperature=full(nan)), sample(z, u, temperature=0.0))
    assert torch.equal(sample(z, u, top_p=full(nan)), sample(z, u)) and torch.equal(sample(z, u, top_p=full(4.0)), sample(z, u))
    assert torch.equal(sample(z, u, top_p=full(-1.0)), sample(z, u, top_k=1))
    assert torch.equal(sample(z, u, min_p=full(nan)), sample(z, u)) and torch.equal(sample(z, u, min_p=full(9.0)), sample(z, u, min_p=1.0))
    assert torch.equal(sample(z, u, top_k=full(-3, torch.int32)), sample(z, u))
    check(z, u, temperature=full(INF), top_p=full(0.5))


def test_the_distribution(device):
    """Tokens come as often as their probabilities say: one row's settings, 20000 uniform numbers one in the middle of each 20000th."""
    z = torch.tensor([1.0, 3.0, 2.0, 3.0, -1.0], device=device)
    R = 20000
    u = ((torch.arange(R, dtype=torch.float64) + 0.5) / R).float().to(device)
    t = sample(z.expand(R, 5), u, top_k=4)
    p = torch.softmax(z.double(), 0)
    p[4] = 0
    count = torch.bincount(t.long(), minlength=5).double()
    # (u rounded to float32 moves no more than one of the 20000 across each border)
    assert ((count / R - p / p.sum()).abs() <= 2.0 / R).all() and count[4] == 0


def test_strides_batches_and_streams(device):
    R, V = 9, 2003
    z, u, s = normal(R, V, torch.bfloat16, device), uniform(R, device), settings(R, device, 7)
    want = sample(z, u, **s)
    wide = torch.full((R, 2 * V), 50.0, dtype=z.dtype, device=device)
    wide[:, 3:3 + V] = z
    assert torch.equal(sample(wide[:, 3:3 + V], u, **s), want)
    assert torch.equal(sample(z.t().contiguous().t(), u, **s), want)
    two = torch.stack([u, u], 1)[:, 0]
    assert torch.equal(sample(z, two, **{n: torch.stack([v, v], 1)[:, 1] for n, v in s.items()}), want)
    for r in range(R):   # a row by itself gives what it gives in the batch
        assert sample(z[r:r + 1], u[r:r + 1], **{n: v[r:r + 1] for n, v in s.items()}).item() == want[r].item()
    far = torch.empty(2 * (1 << 30) + V, dtype=torch.bfloat16, device=device).as_strided((3, V), (1 << 30, 1))
    far.copy_(z[:3])
    assert torch.equal(sample(far, u[:3], **{n: v[:3] for n, v in s.items()}), want[:3])
    del far, wide
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for stream in streams:
        with torch.cuda.stream(stream):
            got += [sample(z, u, **s) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    assert sample(z[:0], u[:0]).shape == (0,)


def test_in_graphs(device):
    held = [(normal(R, V, torch.float32, device), uniform(R, device), settings(R, device, R)) for R, V in ((3, 20001), (80, 1500))]
    graphs = []
    for z, u, s in held:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            sample(z, u, **s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            t = sample(z, u, **s)
        graphs.append((g, t))
    for seed in (11, 12, 13):
        for (z, u, s), (g, t) in zip(held, graphs):
            z.copy_(normal(*z.shape, torch.float32, device, seed))
            u.copy_(uniform(u.shape[0], device, seed))
            g.replay()
        for (z, u, s), (g, t) in zip(held, graphs):
            assert torch.equal(t, sample(z, u, **s))
            check(z, u, **s)


def test_refusals(device):
    z, u = normal(2, 10, torch.float32, device), uniform(2, device)
    for bad in ({"temperature": -1.0}, {"top_p": -0.1}, {"min_p": 1.5}, {"temperature": float("nan")}):
        with pytest.raises(ValueError):
            sample(z, u, **bad)
    for call in (lambda: sample(z[0], u), lambda: sample(z, u[:1]), lambda: sample(z, u.double()), lambda: sample(z, u.cpu()), lambda: sample(z[:, :0], u),
                 lambda: sample(z, u, top_k=torch.tensor([1, 2], device=device)), lambda: sample(z, u, top_p=torch.tensor([0.5], device=device))):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(NotImplementedError):
        sample(z.double(), u)
    with pytest.raises(NotImplementedError):
        sample(torch.zeros(1, (1 << 20) + 1, device=device), u[:1])
