"""GPU: a training step of an expert layer from the operators that it is made of, forward and backward, eager and captured.

Forward: routing, dispatch, up projection, SwiGLU kept in 8 bits, down projection, combine.  Backward: the gradients of all of these, down to the tokens, the gate's
logits and every weight and bias.  Weights are bfloat16."""
import pytest
import torch

from triton_amd.dispatch import combine, combine_backward, dispatch, dispatch_backward
from triton_amd.matmul import matmul
from triton_amd.numerics_details.mxfp import upcast_from_mxfp
from triton_amd.routing import routing
from triton_amd.swiglu import PrecisionConfig, swiglu_backward, swiglu_checkpoint
from triton_amd.topk import topk_backward

pytestmark = pytest.mark.gpu
ALPHA, LIMIT = 1.702, 7.0
PC = PrecisionConfig(limit=LIMIT)
T, H, I, E, K = 300, 256, 192, 16, 4


def inputs(device):
    torch.manual_seed(0)
    r = lambda *s: torch.randn(*s, device=device)  # noqa: E731
    return {"x": r(T, H).bfloat16(), "logits": r(T, E) + r(E), "w1": (r(E, H, 2 * I) / 16).bfloat16(), "b1": 0.1 * r(E, 2 * I), "w2": (r(E, I, H) / 14).bfloat16(),
            "b2": 0.1 * r(E, H), "dy": r(T, H).bfloat16()}


def step(s):
    """Everything that a step computes, by name."""
    r = routing(s["logits"], K)
    md, p, gates = r.ragged_metadata, r.row_sorted_indx.view(T, K), r.vals
    xs = dispatch(s["x"], p)
    a = matmul(xs, s["w1"], s["b1"], md)
    h, values, scales = swiglu_checkpoint(a, ALPHA, PC)
    ys = matmul(h, s["w2"], s["b2"], md)
    y = combine(ys, p, gates=gates)
    # ---- backward: of a only the 8 bits are left, and h is made again from them
    dys, dgates = combine_backward(s["dy"], p, rows=ys, gates=gates)
    dh = matmul(dys, s["w2"].transpose(1, 2), None, md)
    da, h2 = swiglu_backward(dh, values, scales, ALPHA, PC, return_out=True)
    dw2 = matmul(h2.t(), dys, None, md, md)
    dxs = matmul(da, s["w1"].transpose(1, 2), None, md)
    dw1 = matmul(xs.t(), da, None, md, md)
    one = torch.ones(T * K, 8, dtype=torch.bfloat16, device=y.device)      # (a bias's gradient is a product with ones)
    db1, db2 = matmul(one.t(), da, None, md, md)[:, 0], matmul(one.t(), dys, None, md, md)[:, 0]
    dx, _ = dispatch_backward(dxs, p)
    dlogits = topk_backward(s["logits"], r.indx, dgates)
    return {"y": y, "dx": dx, "dlogits": dlogits, "dw1": dw1, "dw2": dw2, "db1": db1, "db2": db2, "kept": (a, values.view(torch.uint8), scales)}


def by_autograd(s, kept):
    """The same in 64 bits, with what the activation's gradient is taken at replaced by what was kept of it."""
    leaf = {n: s[n].double().cpu().requires_grad_() for n in ("x", "logits", "w1", "b1", "w2", "b2")}
    vals, picked = torch.topk(leaf["logits"], K, dim=1)
    gates = torch.softmax(vals, 1)
    flat = picked.flatten()
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(T * K)
    a, values, scales = kept
    at = upcast_from_mxfp(values.view(torch.float8_e4m3fn), scales, torch.float32, -1).double().cpu()
    y = torch.zeros(T, H, dtype=torch.float64)
    for e in range(E):
        t, j = torch.nonzero(picked == e, as_tuple=True)
        z = leaf["x"][t] @ leaf["w1"][e] + leaf["b1"][e]
        z = z + (at[place[t * K + j]] - z).detach()
        g, l = z[:, 0::2].clamp(max=LIMIT), z[:, 1::2].clamp(-LIMIT, LIMIT)
        out = (g * torch.sigmoid(ALPHA * g) * (l + 1)) @ leaf["w2"][e] + leaf["b2"][e]
        y = y.index_add(0, t, gates[t, j, None] * out)
    (y * s["dy"].double().cpu()).sum().backward()
    return y.detach(), {n: v.grad for n, v in leaf.items()}


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def test_gradients(device):
    s = inputs(device)
    got = step(s)
    y, grad = by_autograd(s, got["kept"])
    # Between an input and a result lie at most eight roundings to bfloat16 (2^-9 of a value in the mean, 2^-8 at most), each of which a product with weights of
    # random signs hands on as it is: 8 * 2^-8 is above what they add up to.  y is computed from the activation's input itself, of which e4m3 keeps
    # 2^-4 at most (the reference takes it from what was kept): that enters y once, by a function of slope 1.1 at most and times (l + 1).
    for name, to in (("dx", "x"), ("dlogits", "logits"), ("dw1", "w1"), ("dw2", "w2"), ("db1", "b1"), ("db2", "b2")):
        bound = 8 * 2.0 ** -8 + (2.0 ** -4 if name == "dlogits" else 0.0)      # (its factor is the experts' rows, which come from a itself, as y does)
        assert off(got[name], grad[to]) < bound, (name, off(got[name], grad[to]))
    assert off(got["y"], y) < 2.0 ** -4 + 8 * 2.0 ** -8


def test_captured(device):
    s = inputs(device)
    flat = lambda d: [t for v in d.values() for t in (v if isinstance(v, tuple) else (v,))]  # noqa: E731
    step(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(s)
    for i in range(4):
        torch.manual_seed(10 + i)
        for name in ("x", "logits", "dy"):
            s[name].copy_(torch.randn(s[name].shape, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(held), flat(step(s)))), i


def test_two_captured_steps_share_nothing(device):
    """Two graphs of steps on inputs of their own, replayed in turn and on two streams: each gives what it gives alone."""
    one, two = inputs(device), inputs(device)
    for name in ("x", "logits", "dy"):
        two[name].copy_(torch.randn(two[name].shape, device=device))
    flat = lambda d: [t for v in d.values() for t in (v if isinstance(v, tuple) else (v,))]  # noqa: E731
    want = [[t.clone() for t in flat(step(s))] for s in (one, two)]
    graphs, held = [], []
    for s in (one, two):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            held.append(flat(step(s)))
        graphs.append(graph)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, stream in zip(graphs, side):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for h, w in zip(held, want) for a, b in zip(h, w))
