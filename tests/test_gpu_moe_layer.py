"""GPU: `moe_layer` against the layer's definition in 64 bits, on the sizes and routings where it can go wrong.

The bound of an element is derived, not fitted.  A float32 sum of the kernels passes at most 32 + K/32 + 8 + 16 additions, each off
by at most 2^-23 of what is added up (K <= 2048 here: 2^-16 of the sum of magnitudes); the activation's exponential and reciprocal and the two
16-bit planes of h leave 2^-16 of h; the gate weights' exponentials 2^-19; the result is rounded once, by at most half a step."""
import pytest
import torch

from oracle.mxfp_ref import upcast_from_mxfp_ref
from triton_amd.matmul import FnSpecs, FusedActivation, PrecisionConfig, matmul
from triton_amd.moe_layer import moe_layer
from triton_amd.numerics_details.mxfp import downcast_to_mxfp
from triton_amd.reduce import reduce
from triton_amd.routing import routing
from triton_amd.swiglu import swiglu_fn
from triton_amd.tensor import FP4, convert_layout, wrap_torch_tensor
from triton_amd.tensor_details.layout import CDNA4MXScaleLayout, CDNA4MXValueLayout

pytestmark = pytest.mark.gpu
SUM, ACT, GATE = 2.0**-16, 2.0**-16, 2.0**-19


def swiglu_spec(alpha=1.702, limit=7.0):
    return FusedActivation(FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2), (alpha, limit))


class Layer:
    """Quantised weights on the GPU in any layout, and their values in 64 bits."""

    def __init__(self, device, E, H, I, seed=0, bias=torch.float32, spread=0.3):
        g = torch.Generator().manual_seed(seed)
        self.E, self.H, self.I = E, H, I
        self.w, self.s, self.dense = [], [], []
        for K, N in ((H, 2 * I), (I, H)):
            w = (torch.randn(E, K, N, generator=g) * spread).to(torch.bfloat16).to(device)
            v, s = downcast_to_mxfp(w, torch.uint8, axis=-2)
            self.w.append(v)
            self.s.append(s)
            self.dense.append(upcast_from_mxfp_ref(v.cpu(), s.cpu(), torch.float32, axis=-2).double())
        self.bias = [None, None] if bias is None else [torch.randn(E, n, generator=g).to(bias).to(device) for n in (2 * I, H)]

    def call(self, x, logits, k, values=("strided", "strided"), scales=("strided", "strided"), alpha=1.702, limit=7.0, out=None):
        w = [convert_layout(wrap_torch_tensor(v, dtype=FP4), CDNA4MXValueLayout()) if kind == "blocks" else v for v, kind in zip(self.w, values)]
        pc = [PrecisionConfig(b_mx_scale=convert_layout(wrap_torch_tensor(s), CDNA4MXScaleLayout()) if kind == "shuffled" else s, b_microblock_size=32)
              for s, kind in zip(self.s, scales)]
        return moe_layer(x, logits, k, w[0], self.bias[0], w[1], self.bias[1], pc[0], pc[1], swiglu_spec(alpha, limit), out=out)

    def expected(self, x, logits, k, alpha=1.702, limit=7.0):
        """(values, bound) [T, H] in 64 bits."""
        x, logits = x.cpu().double(), logits.cpu().double()
        b = [torch.zeros(self.E, n, dtype=torch.float64) if v is None else v.cpu().double() for v, n in zip(self.bias, (2 * self.I, self.H))]
        y, err = torch.zeros(x.shape[0], self.H, dtype=torch.float64), torch.zeros(x.shape[0], self.H, dtype=torch.float64)
        for t in range(x.shape[0]):
            order = sorted(range(self.E), key=lambda e: (-logits[t, e].item(), e))[:k]
            e_l = torch.exp(logits[t, order] - logits[t, order[0]])
            for e, gate in zip(order, (e_l / e_l.sum()).tolist()):
                a = x[t] @ self.dense[0][e] + b[0][e]
                mag = SUM * (x[t].abs() @ self.dense[0][e].abs() + b[0][e].abs())
                g, l = a[0::2], a[1::2]
                if limit is not None:
                    g, l = g.clamp(max=limit), l.clamp(-limit, limit)
                h = g * torch.sigmoid(alpha * g) * (l + 1)
                e_h = mag[0::2] * 1.1 * (l.abs() + 1) + mag[1::2] * g.abs() + ACT * (g.abs() * (l.abs() + 1))
                r = h @ self.dense[1][e] + b[1][e]
                y[t] += gate * r
                err[t] += gate * (e_h @ self.dense[1][e].abs() + (SUM + GATE) * (h.abs() @ self.dense[1][e].abs() + b[1][e].abs()))
        return y, err

    def check(self, got, x, logits, k, **kw):
        want, err = self.expected(x, logits, k, **kw)
        off = (got.cpu().double() - want).abs()
        bound = err + (want.abs() + err) * torch.finfo(got.dtype).eps / 2
        assert torch.isfinite(got).all()
        assert (off <= bound).all(), f"{(off / bound).max():.2f} of the bound"


def inputs(T, E, H, dtype, device, seed=1, logits=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, H, generator=g).to(dtype).to(device), torch.randn(T, E, generator=g).to(logits).to(device)


@pytest.mark.parametrize("values,scales", [("strided", "strided"), ("blocks", "shuffled"), ("blocks", "strided"), ("strided", "shuffled")])
@pytest.mark.parametrize("T,E,k,H,I,dtype", [
    (1, 8, 2, 32, 32, torch.bfloat16), (1, 8, 2, 160, 96, torch.float16), (3, 8, 8, 288, 160, torch.bfloat16),
    (8, 60, 4, 320, 416, torch.float16), (9, 4, 1, 1184, 64, torch.bfloat16), (16, 130, 6, 64, 1120, torch.bfloat16),
    (17, 4, 2, 96, 224, torch.float16), (33, 3, 2, 256, 128, torch.bfloat16), (64, 2, 2, 128, 96, torch.float16), (64, 512, 8, 32, 64, torch.bfloat16)])
def test_layer(T, E, k, H, I, dtype, values, scales, device):
    layer = Layer(device, E, H, I)
    x, logits = inputs(T, E, H, dtype, device)
    layer.check(layer.call(x, logits, k, (values, values), (scales, scales)), x, logits, k)


@pytest.mark.parametrize("H,I", [(512, 512), (1056, 96), (1536, 64), (2016, 128), (96, 2048)])
def test_rounds_of_blocks(H, I, device):
    """Every number of blocks per wave, K of one round and of several, and a last block that is not whole."""
    layer = Layer(device, 3, H, I, spread=0.1)
    for T in (1, 5, 20):
        x, logits = inputs(T, 3, H, torch.bfloat16, device)
        layer.check(layer.call(x, logits, 2, ("blocks", "blocks"), ("shuffled", "shuffled")), x, logits, 2)


def test_long_k(device):
    """More blocks of K than one round of the eight waves takes."""
    layer = Layer(device, 2, 5760, 32, spread=0.02)
    x, logits = inputs(2, 2, 5760, torch.bfloat16, device)
    got = layer.call(x, logits, 1, ("blocks", "strided"), ("shuffled", "strided")).cpu().double()
    want, err = layer.expected(x, logits, 1)
    # (the sums are longer than the bound's: 32 + 180 + 24 additions stay below 2^-15)
    assert ((got - want).abs() <= 2 * err + want.abs() * torch.finfo(torch.bfloat16).eps / 2 * 1.01).all()


@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_ties_and_masked_logits(logits_dtype, device):
    """Equal logits go to the lower expert; -inf and the type's lowest value are picked last and weigh nothing; equal picks weigh the same."""
    layer = Layer(device, 70, 64, 64)
    x, logits = inputs(6, 70, 64, torch.bfloat16, device, logits=logits_dtype)
    logits[0] = 0.0
    logits[1] = -float("inf")
    logits[1, 69] = 1.0
    logits[2] = torch.finfo(logits_dtype).min
    logits[2, 3] = 2.0
    logits[3] = torch.finfo(logits_dtype).max
    logits[4, ::2] = -0.0
    logits[4, 1::2] = 0.0
    layer.check(layer.call(x, logits, 4), x, logits, 4)


def test_a_row_without_an_expert_is_nan_as_in_routing(device):
    layer = Layer(device, 8, 64, 64)
    x, logits = inputs(3, 8, 64, torch.bfloat16, device)
    logits[1] = -float("inf")
    y = layer.call(x, logits, 2)
    assert torch.isnan(routing(logits, 2).vals[1]).all() and torch.isnan(y[1]).all()
    keep = torch.tensor([0, 2], device=device)
    assert torch.equal(y[keep], layer.call(x[keep], logits[keep], 2))


def test_nan_and_infinities_stay_with_their_tokens(device):
    """A NaN scale in an expert and NaN or infinite activations reach the tokens that use them and no other."""
    layer = Layer(device, 4, 128, 128)
    x, logits = inputs(12, 4, 128, torch.bfloat16, device)
    logits = torch.full_like(logits, -20.0)
    logits[torch.arange(12), torch.arange(12) % 4] = 1.0
    good = layer.call(x, logits, 1)
    for n in (0, 1):
        scale = layer.s[n].clone()
        layer.s[n][2] = 255
        y = layer.call(x, logits, 1)
        layer.s[n].copy_(scale)
        hit = torch.arange(12) % 4 == 2
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], good[~hit])
    x2 = x.clone()
    x2[5] = float("nan")
    x2[6, 3] = float("inf")
    y = layer.call(x2, logits, 1)
    others = [t for t in range(12) if t not in (5, 6)]
    assert torch.isnan(y[5]).all() and torch.equal(y[others], good[others])


@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("alpha,limit", [(1.0, None), (1.702, 0.5)])
def test_biases_and_activation(bias, alpha, limit, device):
    layer = Layer(device, 5, 96, 64, bias=bias)
    x, logits = inputs(4, 5, 96, torch.bfloat16, device)
    layer.check(layer.call(x, logits, 3, alpha=alpha, limit=limit), x, logits, 3, alpha=alpha, limit=limit)


def test_strides_and_output(device):
    """Rows that are not dense, rows that do not start on 16 bytes, expanded rows, logits with any strides, an output between other columns."""
    layer = Layer(device, 6, 96, 64)
    x, logits = inputs(7, 6, 96, torch.bfloat16, device)
    want = layer.call(x, logits, 2)
    wide = torch.zeros(7, 200, dtype=x.dtype, device=device)
    for at in (8, 3):
        wide[:, at:at + 96] = x
        assert torch.equal(layer.call(wide[:, at:at + 96], logits, 2), want)
    assert torch.equal(layer.call(x, logits.t().contiguous().t(), 2), want)
    assert torch.equal(layer.call(x.t().contiguous().t(), logits, 2), want)
    same = layer.call(x[:1].expand(7, 96), logits[:1].expand(7, 6), 2)
    assert torch.equal(same, want[:1].expand(7, 96))
    out = torch.full((7, 160), 5.0, dtype=x.dtype, device=device)
    got = layer.call(x, logits, 2, out=out[:, 32:128])
    assert got.data_ptr() == out[:, 32:].data_ptr() and torch.equal(out[:, 32:128], want)
    assert (out[:, :32] == 5).all() and (out[:, 128:] == 5).all()
    assert layer.call(x[:0], logits[:0], 2).shape == (0, 96)


def test_rows_far_apart(device):
    """Strides whose products pass 32 bits."""
    layer = Layer(device, 4, 64, 64)
    x, logits = inputs(3, 4, 64, torch.bfloat16, device)
    far = torch.empty(2 * (1 << 30) + 64, dtype=torch.bfloat16, device=device).as_strided((3, 64), (1 << 30, 1))
    far.copy_(x)
    assert torch.equal(layer.call(far, logits, 2), layer.call(x, logits, 2))


@pytest.mark.parametrize("T,dtype", [(1, torch.bfloat16), (13, torch.float16), (64, torch.bfloat16)])
def test_against_the_chain(T, dtype, device):
    """The same layer as routing -> matmul -> matmul -> reduce runs it: within the chain's own roundings, h and the experts' rows to 16 bits."""
    E, k, H, I = 16, 4, 512, 256
    layer = Layer(device, E, H, I, spread=0.05)
    x, logits = inputs(T, E, H, dtype, device)
    got = layer.call(x, logits, k)
    r = routing(logits, k)
    pc = [PrecisionConfig(b_mx_scale=s, b_microblock_size=32) for s in layer.s]
    h = matmul(x, layer.w[0], layer.bias[0], r.ragged_metadata, gather_indx=r.gather_indx, precision_config=pc[0], fused_activation=swiglu_spec())
    y = matmul(h, layer.w[1], layer.bias[1], r.ragged_metadata, scatter_indx=r.scatter_indx, precision_config=pc[1], gammas=r.expert_sorted_gate_weights)
    z, _ = reduce(y.view(T, k, H), dim=1)
    layer.check(got, x, logits, k)
    # half a step each: h under |W2|, every expert's row, the sum (and the gate weights' type is float32 in both)
    half = torch.finfo(dtype).eps / 2
    h64, y64 = torch.zeros(T, H, dtype=torch.float64), y.cpu().double().abs().view(T, k, H).sum(1)
    for row, (flat, e) in enumerate(zip(r.scatter_indx.tolist(), torch.repeat_interleave(torch.arange(E), r.col_sum.cpu().long()).tolist())):
        gate = r.vals.cpu().double().reshape(-1)[flat]
        h64[flat // k] += gate * (h[row].cpu().double().abs() @ layer.dense[1][e].abs())
    _, err = layer.expected(x, logits, k)
    bound = 2 * err + 1.01 * half * (h64 + y64 + z.cpu().double().abs() + got.cpu().double().abs())
    assert ((got.cpu().double() - z.cpu().double()).abs() <= bound).all()


def test_repeated_streams_and_other_contents_of_memory(device):
    """The same bits from call to call, on another stream, and whatever the workspace held."""
    layer = Layer(device, 16, 256, 128)
    x, logits = inputs(24, 16, 256, torch.bfloat16, device)
    want = layer.call(x, logits, 4)
    junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=device) for _ in range(8)]
    del junk
    assert torch.equal(layer.call(x, logits, 4), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [layer.call(x, logits, 4) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_in_graphs(device):
    """Two captured graphs with a pool of their own each, replayed in turn with new inputs and eager work in between."""
    layer = Layer(device, 16, 128, 96)
    cases = [(2, 4), (30, 3)]
    held, graphs = [inputs(T, 16, 128, torch.bfloat16, device) for T, _ in cases], []
    for (x, logits), (_, k) in zip(held, cases):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.call(x, logits, k, scales=("strided", "strided"))
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y = layer.call(x, logits, k)
        graphs.append((g, y))
    for seed in (3, 4, 5):
        for (x, logits), (T, k), (g, y) in zip(held, cases, graphs):
            nx, nl = inputs(T, 16, 128, torch.bfloat16, device, seed=seed)
            x.copy_(nx)
            logits.copy_(nl)
            g.replay()
        for (x, logits), (_, k), (g, y) in zip(held, cases, graphs):
            assert torch.equal(y, layer.call(x, logits, k))
