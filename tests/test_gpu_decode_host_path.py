"""GPU: the native host path of `moe_layer`, `matvec` and `sample` against their general path, bit for bit, and what `moe_layer` refuses."""
import pytest
import torch

import test_gpu_matvec
from test_gpu_host_path import BothPaths
from test_gpu_moe_layer import Layer, inputs, swiglu_spec
from triton_amd.matmul import FnSpecs, FusedActivation, PrecisionConfig
from triton_amd.matvec import matvec
from triton_amd.moe_layer import moe_layer
from triton_amd.sampling import sample
from triton_amd.swiglu import swiglu_fn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("values,scales", [("strided", "strided"), ("blocks", "shuffled"), ("blocks", "strided"), ("strided", "shuffled")])
@pytest.mark.parametrize("form,covered", [("plain", True), ("no bias", True), ("no limit", True), ("bf16 logits", True), ("one token", True),
                                          ("x off 16 bytes", False), ("logits turned", False), ("odd bias", False), ("no tokens", False)])
def test_moe_layer(form, covered, values, scales, device, monkeypatch):
    layer = Layer(device, 9, 96, 64, bias=None if form == "no bias" else torch.bfloat16 if form == "odd bias" else torch.float32)
    x, logits = inputs(1 if form == "one token" else 5, 9, 96, torch.bfloat16, device, logits=torch.bfloat16 if form == "bf16 logits" else torch.float32)
    if form == "x off 16 bytes":
        wide = torch.zeros(5, 104, dtype=x.dtype, device=device)
        wide[:, 3:99] = x
        x = wide[:, 3:99]
    elif form == "logits turned":
        logits = logits.t().contiguous().t()
    elif form == "odd bias":
        held = torch.zeros(9 * 96 + 1, dtype=torch.bfloat16, device=device)
        held[1:] = layer.bias[1].reshape(-1)
        layer.bias[1] = held[1:].view(9, 96)
    elif form == "no tokens":
        x, logits = x[:0], logits[:0]
    call = lambda: (layer.call(x, logits, 2, (values, values), (scales, scales), limit=None if form == "no limit" else 7.0), )  # noqa: E731
    assert BothPaths(monkeypatch, "moe_layer")(call) == covered


@pytest.mark.parametrize("form,covered", [("plain", True), ("bias", True), ("float32 out", True), ("pitch", True), ("zeros", True), ("x off 16 bytes", False),
                                          ("a vector", True), ("bias with a stride", False), ("columns", False), ("no rows", False)])
def test_matvec(form, covered, device, monkeypatch):
    w, _, _ = test_gpu_matvec.make(192, 75, 64, form == "zeros", torch.float16, device)
    x, bias, out = test_gpu_matvec.rows(6, 192, torch.bfloat16, device), None, None
    if form == "bias":
        bias = torch.randn(75, device=device).half()
    elif form == "float32 out":
        out = torch.float32
    elif form in ("pitch", "x off 16 bytes"):
        wide = torch.zeros(6, 208, dtype=x.dtype, device=device)
        at = 8 if form == "pitch" else 5
        wide[:, at:at + 192] = x
        x = wide[:, at:at + 192]
    elif form == "a vector":
        x = x[1]
    elif form == "bias with a stride":
        bias = torch.randn(150, device=device)[::2]
    elif form == "columns":
        x = x.t().contiguous().t()
    elif form == "no rows":
        x = x[:0]
    both = BothPaths(monkeypatch, "matvec")
    if form == "a vector":   # (the general path makes a row of it, which the native one takes)
        native, general = matvec(x, w), matvec(x[None], w, out=torch.empty(1, 75, dtype=x.dtype, device=device))[0]
        assert torch.equal(native, general)
    else:
        assert both(lambda: (matvec(x, w, bias, out), )) == covered


@pytest.mark.parametrize("form,covered", [("numbers", True), ("tensors", True), ("integers", True), ("pitch", True), ("columns", False), ("u with a stride", False),
                                          ("negative top_k", False), ("no rows", False)])
@pytest.mark.parametrize("V", [700, 40001])
def test_sample(form, covered, V, device, monkeypatch):
    g = torch.Generator().manual_seed(V)
    logits, u = (2 * torch.randn(6, V, generator=g)).to(device), torch.rand(6, generator=g).to(device)
    settings = dict(temperature=0.8, top_k=40, top_p=0.9, min_p=0.01)
    if form == "tensors":
        settings = dict(temperature=torch.linspace(0, 1, 6, device=device), top_k=torch.arange(6, dtype=torch.int32, device=device),
                        top_p=torch.linspace(0.5, 1, 6, device=device), min_p=torch.linspace(0, 0.2, 6, device=device))
    elif form == "integers":
        settings = dict(temperature=1, top_k=0, top_p=1, min_p=0)
    elif form == "pitch":
        wide = torch.full((6, V + 13), float("nan"), device=device)
        wide[:, 5:V + 5] = logits
        logits = wide[:, 5:V + 5]
    elif form == "columns":
        logits = logits.t().contiguous().t()
    elif form == "u with a stride":
        u = torch.stack([u, u], 1)[:, 0]
    elif form == "negative top_k":
        settings["top_k"] = -3
    elif form == "no rows":
        logits, u = logits[:0], u[:0]
    assert BothPaths(monkeypatch, "sample")(lambda: (sample(logits, u, **settings), )) == covered


def test_moe_layer_refuses(device):
    layer = Layer(device, 4, 64, 32)
    x, logits = inputs(3, 4, 64, torch.bfloat16, device)
    pc = [PrecisionConfig(b_mx_scale=s, b_microblock_size=32) for s in layer.s]

    def call(x=x, logits=logits, k=2, w1=layer.w[0], b1=layer.bias[0], w2=layer.w[1], b2=layer.bias[1], pc1=pc[0], pc2=pc[1], act=swiglu_spec(), out=None):
        return moe_layer(x, logits, k, w1, b1, w2, b2, pc1, pc2, act, out=out)

    assert call().shape == (3, 64)
    many = torch.zeros(65, 64, dtype=x.dtype, device=device), torch.zeros(65, 4, device=device)
    other = FusedActivation(FnSpecs("gelu", swiglu_fn, ("alpha", "limit"), reduction_n=2), (1.0, 1.0))
    for kw in (dict(x=x.float()), dict(x=many[0], logits=many[1]), dict(act=other), dict(act=None), dict(logits=logits.double()), dict(pc1=None),
               dict(pc2=PrecisionConfig()), dict(b1=layer.bias[0].double()), dict(w1=torch.zeros(4, 64, 64, dtype=x.dtype, device=device)),
               dict(pc1=PrecisionConfig(b_mx_scale=layer.s[0], b_microblock_size=32, out_dtype=torch.float32)),
               dict(pc2=PrecisionConfig(b_mx_scale=layer.s[1], b_microblock_size=32, acc_scale=2.0))):
        with pytest.raises(NotImplementedError):
            call(**kw)
    for kw in (dict(logits=logits[:2]), dict(k=5), dict(k=0), dict(w1=layer.w[0][:3]), dict(w2=layer.w[0]), dict(b1=layer.bias[0][:, 1:]), dict(logits=logits.cpu()),
               dict(b2=layer.bias[1].cpu()), dict(out=torch.empty(3, 63, dtype=x.dtype, device=device)), dict(out=torch.empty(3, 64, device=device)),
               dict(x=x[:, :32])):
        with pytest.raises(AssertionError):
            call(**kw)
    with pytest.raises(ValueError):
        call(x=x[:, :48], w1=layer.w[0][:, :24], w2=layer.w[1][:, :, :48])
