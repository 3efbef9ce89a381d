"""GPU: the native host path of the training operators against the general one: the same results, and the calls that each takes."""
import pytest
import torch

from triton_amd import _native
from triton_amd.dispatch import combine, combine_backward, dispatch, dispatch_backward
from triton_amd.matmul import PrecisionConfig as Precision
from triton_amd.matmul import matmul
from triton_amd.routing import routing
from triton_amd.swiglu import PrecisionConfig, swiglu_backward, swiglu_checkpoint
from triton_amd.tensor import make_ragged_tensor_metadata
from triton_amd.topk import topk_backward

pytestmark = pytest.mark.gpu
NAMES = ("dispatch", "combine", "dispatch_backward", "combine_backward", "swiglu_checkpoint", "swiglu_backward", "topk_backward", "matmul_ragged_k")


def calls(device, dtype):
    """(name, call) of plain calls, which the native path takes."""
    torch.manual_seed(0)
    T, k, H, E, N = 70, 4, 136, 16, 40
    logits = torch.randn(T, E, device=device).to(dtype)
    r = routing(logits, k)
    p = r.row_sorted_indx.view(T, k)
    x, rows = torch.randn(T, H, device=device).to(dtype), torch.randn(T * k, H, device=device).to(dtype)
    gates, room = r.vals, torch.zeros(T * k, H, dtype=dtype, device=device)
    a, d = torch.randn(T, 2 * N, device=device).to(dtype), torch.randn(T, N, device=device).to(dtype)
    pc = PrecisionConfig(limit=7.0)
    _, values, scales = swiglu_checkpoint(a, 1.702, pc)
    offs = r.ragged_metadata
    wide = torch.randn(T * k, 2 * H, device=device).to(dtype)[:, 8:8 + H]
    yield "dispatch", lambda: dispatch(x, p)
    yield "dispatch", lambda: dispatch(x, p, gates=gates, out=room).clone()
    yield "combine", lambda: combine(rows, p, gates=gates)
    yield "combine", lambda: combine(wide, p)
    yield "dispatch_backward", lambda: dispatch_backward(rows, p, x=x, gates=gates)
    yield "dispatch_backward", lambda: dispatch_backward(rows, p)
    yield "combine_backward", lambda: combine_backward(x, p, rows=rows, gates=gates)
    yield "combine_backward", lambda: combine_backward(x, p, gates=gates, out=room)
    yield "swiglu_checkpoint", lambda: swiglu_checkpoint(a, 1.702, pc)
    yield "swiglu_checkpoint", lambda: swiglu_checkpoint(a, 1, PrecisionConfig(limit=None))
    yield "swiglu_backward", lambda: swiglu_backward(d, values, scales, 1.702, pc, return_out=True)
    yield "swiglu_backward", lambda: swiglu_backward(d, values, scales, 1.702, pc)
    yield "topk_backward", lambda: topk_backward(logits, r.indx, gates)
    yield "topk_backward", lambda: topk_backward(logits, r.indx, gates.float(), apply_softmax=False)
    if dtype != torch.float32:
        yield "matmul_ragged_k", lambda: matmul(rows.t(), wide, None, offs, offs)
        yield "matmul_ragged_k", lambda: matmul(rows.t(), wide, None, None, offs, precision_config=Precision(out_dtype=torch.float32))


def flat(v):
    return [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (v if isinstance(v, tuple) else (v,)) if t is not None]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_same_results(dtype, device, monkeypatch):
    _native.load()
    for name, call in list(calls(device, dtype)):
        native, taken = getattr(_native, name), []
        monkeypatch.setattr(_native, name, lambda *args: taken.append(native(*args)) or taken[-1])
        fast = call()
        assert len(taken) == 1 and taken[0] is not None, name
        monkeypatch.setattr(_native, name, lambda *args: None)
        slow = call()
        monkeypatch.setattr(_native, name, native)
        assert type(fast) is type(slow) and len(flat(fast)) == len(flat(slow))
        for x, y in zip(flat(fast), flat(slow)):
            assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and torch.equal(x, y), name


def test_misuse_is_reported_by_the_general_path(device):
    """What the native path does not take raises as if it were not there."""
    _native.load()
    x, p, gates = torch.randn(6, 32, device=device), torch.zeros(6, 2, dtype=torch.int32, device=device), torch.rand(6, 2, device=device)
    md = make_ragged_tensor_metadata(torch.tensor([2, 4], dtype=torch.int32, device=device), 6)
    for call in (lambda: dispatch(x, p.long()), lambda: dispatch(x, p.cpu()), lambda: combine(x, p, gates=gates[:, :1]), lambda: combine_backward(x, p, rows=x, gates=gates),
                 lambda: dispatch_backward(x, p, x=x.half(), gates=gates), lambda: swiglu_checkpoint(x[:, :31], 1.0, PrecisionConfig(limit=None)),
                 lambda: topk_backward(x, p, gates), lambda: matmul(x.half(), x.half(), None, md, md)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: dispatch(x.double(), p), lambda: combine(x, p, gates=gates.double()), lambda: swiglu_checkpoint(x.double(), 1.0, PrecisionConfig(limit=None)),
                 lambda: matmul(x.t(), x, None, md, md)):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(ValueError):
        swiglu_checkpoint(x, 1.0, PrecisionConfig(limit=-1.0))
