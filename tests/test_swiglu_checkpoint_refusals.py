"""What `swiglu_checkpoint`, `swiglu_backward` and their C entry points refuse before anything is launched (no GPU needed)."""
import pytest
import torch

from triton_amd import _lib
from triton_amd.numerics import InFlexData, OutFlexData
from triton_amd.swiglu import FlexCtx, PrecisionConfig, swiglu_backward, swiglu_checkpoint


def forward(a=0x1000, dtype=_lib.BF16, M=0, N=16, sa=32, out=0x2000, so=16, v=0x3000, sv=32, s=0x4000, ss=1, alpha=1.0, limit=7.0, has=1):
    return _lib.lib().tamd_swiglu_checkpoint(a, dtype, M, N, sa, out, so, v, sv, s, ss, alpha, limit, has, None)


def backward(d=0x1000, dtype=_lib.BF16, M=0, N=16, sd=16, v=0x3000, sv=32, s=0x4000, ss=1, da=0x5000, sda=32, out=None, so=16, alpha=1.0, limit=7.0, has=1):
    return _lib.lib().tamd_swiglu_backward(d, dtype, M, N, sd, v, sv, s, ss, da, sda, out, so, alpha, limit, has, None)


@pytest.mark.parametrize("call,strides,pointers", [(forward, ("sa", "so", "sv", "ss"), ("a", "out", "v", "s")), (backward, ("sd", "sv", "ss", "sda", "so"), ("d", "v", "s", "da"))])
def test_c_entry_points(call, strides, pointers):
    assert call() == 0 and call(M=3, N=0) == 0
    for name in ("M", "N", *strides):
        assert call(**{name: -1}) == _lib.E_INVALID, name
    assert call(limit=-1.0) == _lib.E_INVALID and call(limit=float("nan")) == _lib.E_INVALID and call(limit=-1.0, has=0) == 0
    for dtype in (_lib.FP8_E4M3, _lib.MXFP4, -1):
        assert call(dtype=dtype) == _lib.E_UNSUPPORTED
    for name in pointers:
        assert call(M=3, **{name: None}) == _lib.E_INVALID, name
    for name in pointers:
        if name not in "vs":
            assert call(M=3, **{name: 0x1001}) == _lib.E_ALIGNMENT, name
    assert call(M=1 << 29, N=64) == _lib.E_TOO_LARGE      # more threads than a launch has
    assert call(M=1 << 31) == _lib.E_TOO_LARGE and call(M=1, N=1 << 30) == _lib.E_TOO_LARGE and call(M=(1 << 31) - 1, N=(1 << 30) - 1) == _lib.E_TOO_LARGE


def test_cpu_tensors_are_refused():
    pc = PrecisionConfig(limit=7.0)
    with pytest.raises(RuntimeError, match="GPU"):
        swiglu_checkpoint(torch.zeros(2, 32), 1.0, pc)
    with pytest.raises(RuntimeError, match="GPU"):
        swiglu_backward(torch.zeros(2, 16), torch.zeros(2, 32).to(torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8), 1.0, pc)


def test_shapes_types_and_options(monkeypatch):
    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    for entry in ("tamd_swiglu_checkpoint", "tamd_swiglu_backward"):
        monkeypatch.setattr(_lib.lib(), entry, lambda *a: pytest.fail("launched"))
    pc, a, d = PrecisionConfig(limit=7.0), torch.zeros(2, 40), torch.zeros(2, 20)
    v, s = a.to(torch.float8_e4m3fn), torch.zeros(2, 2, dtype=torch.uint8)
    for call in (lambda: swiglu_checkpoint(a[:, :39], 1.0, pc), lambda: swiglu_backward(d, v[:, :38], s, 1.0, pc), lambda: swiglu_backward(d, v, s[:, :1], 1.0, pc),
                 lambda: swiglu_backward(d, v[:1], s, 1.0, pc), lambda: swiglu_backward(d, a, s, 1.0, pc), lambda: swiglu_backward(d, v, s.float(), 1.0, pc),
                 lambda: swiglu_backward(d[0], v, s, 1.0, pc)):
        with pytest.raises(AssertionError):
            call()
    flex = PrecisionConfig(limit=7.0, flex_ctx=FlexCtx(inp_data=InFlexData(scale=torch.ones(1))))
    for call in (lambda: swiglu_checkpoint(a.double(), 1.0, pc), lambda: swiglu_checkpoint(v, 1.0, pc), lambda: swiglu_backward(d.long(), v, s, 1.0, pc),
                 lambda: swiglu_checkpoint(a, 1.0, flex), lambda: swiglu_backward(d, v, s, 1.0, flex)):
        with pytest.raises(NotImplementedError):
            call()
    for limit in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            swiglu_checkpoint(a, 1.0, PrecisionConfig(limit=limit))
        with pytest.raises(ValueError):
            swiglu_backward(d, v, s, 1.0, PrecisionConfig(limit=limit))


@pytest.mark.parametrize("name", ["expected_scale", "actual_scale", "checksum_scale"])
def test_scales_of_the_result_are_not_dropped(name, monkeypatch):
    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    for entry in ("tamd_swiglu_checkpoint", "tamd_swiglu_backward"):
        monkeypatch.setattr(_lib.lib(), entry, lambda *a: pytest.fail("launched"))
    pc = PrecisionConfig(limit=7.0, flex_ctx=FlexCtx(out_data=OutFlexData(**{name: torch.ones(1)})))
    with pytest.raises(NotImplementedError):
        swiglu_checkpoint(torch.zeros(2, 32), 1.0, pc)
    with pytest.raises(NotImplementedError):
        swiglu_backward(torch.zeros(2, 16), torch.zeros(2, 32).to(torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8), 1.0, pc)
