"""GPU: `moe_layer` where the experts of a strip of columns are dealt out to several workgroups, and a workgroup has parts of several
strips, against the definition in 64 bits (the bound is the one of test_gpu_moe_layer: adding up the parts is one
addition more per part, of at most 32 + K/32 + 8 + 16 of which K <= 2048 leaves more than a hundred unused below the bound)."""
import pytest
import torch

from test_gpu_moe_layer import Layer, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("values,scales", [("strided", "strided"), ("blocks", "shuffled")])
@pytest.mark.parametrize("T,E,k,H,I,dtype", [
    (16, 16, 4, 4800, 64, torch.bfloat16),      # a workgroup has the end of a strip, a whole one and the beginning of a third
    (12, 12, 1, 4128, 32, torch.float16),       # 258 strips
    (64, 20, 8, 2048, 96, torch.bfloat16),      # half a strip for each
    (3, 40, 16, 64, 192, torch.float16),        # more workgroups than experts of strips
    (9, 64, 2, 96, 1056, torch.bfloat16)])
def test_layer(T, E, k, H, I, dtype, values, scales, device):
    layer = Layer(device, E, H, I)
    x, logits = inputs(T, E, H, dtype, device)
    y = layer.call(x, logits, k, (values, values), (scales, scales))
    layer.check(y, x, logits, k)
    for _ in range(3):
        assert torch.equal(layer.call(x, logits, k, (values, values), (scales, scales)), y)


@pytest.mark.parametrize("T,E,k,I", [(20, 12, 8, 4128), (3, 12, 8, 4128), (16, 12, 3, 2880), (30, 12, 6, 2880), (7, 40, 1, 2336)])
def test_rounds_of_blocks(T, E, k, I, device):
    """More blocks of K than one round of the eight waves takes, or as many as three for each; one to fifteen rows per expert."""
    layer = Layer(device, E, 64, I, spread=0.05)
    x, logits = inputs(T, E, 64, torch.bfloat16, device)
    got = layer.call(x, logits, k, ("blocks", "blocks"), ("shuffled", "shuffled")).cpu().double()
    want, err = layer.expected(x, logits, k)
    # (32 + 129 + 24 + parts additions: below 2^-15 of what is added up, twice the bound's)
    assert ((got - want).abs() <= 2 * err + want.abs() * torch.finfo(torch.bfloat16).eps / 2 * 1.01).all()


def test_few_of_the_experts_are_picked(device):
    """Every token picks the same two of many: how many there are is known on the GPU alone.  No bias; the output's
    neighbours are left as they were; a token that is not finite stays alone."""
    layer = Layer(device, 48, 288, 128, bias=None)
    x, logits = inputs(10, 48, 288, torch.bfloat16, device)
    logits[:, [5, 40]] += 20.0
    out = torch.full((12, 320), 7.0, dtype=torch.bfloat16, device=device)
    y = layer.call(x, logits, 2, out=out[1:11, 16:304])
    layer.check(y, x, logits, 2)
    assert (out[0] == 7).all() and (out[11] == 7).all() and (out[:, :16] == 7).all() and (out[:, 304:] == 7).all()
    bad = x.clone()
    bad[4, 7] = float("nan")
    again = layer.call(bad, logits, 2)
    assert torch.isnan(again[4]).all() and torch.equal(again[:4], y[:4]) and torch.equal(again[5:], y[5:])


def test_two_graphs_and_two_streams(device):
    """Captured calls keep workspaces of their own; replays in turn, and side by side, give what eager calls give."""
    layer = Layer(device, 24, 512, 64)
    calls = [inputs(n, 24, 512, torch.bfloat16, device, seed=n) for n in (7, 13)]
    want = [layer.call(x, lo, 4) for x, lo in calls]
    graphs, outs = [], []
    for x, lo in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.call(x, lo, 4))
        graphs.append(g)
    for _ in range(4):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        for o in outs:
            o.zero_()
        assert torch.equal(layer.call(*calls[0], 4), want[0])
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer.call(*calls[i], 4))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)
