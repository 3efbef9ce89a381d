"""What `topk_backward` and its C entry point refuse before anything is launched (no GPU needed)."""
import pytest
import torch

from triton_amd import _lib
from triton_amd.topk import topk_backward


def call(x=0x1000, dtype=_lib.F32, sx=8, rows=0, live=0, cols=8, k=2, softmax=1, indx=0x2000, si=2, d=0x3000, dd=_lib.F32, sd=2, dx=0x4000, sdx=8):
    return _lib.lib().tamd_topk_backward(x, dtype, sx, rows, live, cols, k, softmax, indx, si, d, dd, sd, dx, sdx, None)


def test_c_entry_point():
    assert call() == 0 and call(rows=3, cols=0) == 0
    for name in ("sx", "rows", "live", "cols", "k", "si", "sd", "sdx"):
        assert call(**{name: -1}) == _lib.E_INVALID, name
    assert call(dtype=_lib.FP8_E4M3) == call(dd=_lib.FP8_E5M2) == _lib.E_UNSUPPORTED
    assert call(cols=32768) == call(k=65) == call(rows=1 << 32) == call(rows=1 << 28, live=0) == call(rows=1 << 26, live=0, k=17) == _lib.E_TOO_LARGE
    for name in ("x", "indx", "d", "dx"):
        assert call(rows=3, live=3, **{name: None}) == _lib.E_INVALID, name
        assert call(rows=3, live=3, **{name: 0x1001}) == _lib.E_ALIGNMENT, name


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        topk_backward(torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int16), torch.zeros(2, 1))


def test_shapes_and_types(monkeypatch):
    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    monkeypatch.setattr(_lib.lib(), "tamd_topk_backward", lambda *a: pytest.fail("launched"))
    x, i, d = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int16), torch.zeros(3, 2)
    for bad in (lambda: topk_backward(x[0], i, d), lambda: topk_backward(x, i.int(), d), lambda: topk_backward(x, i[:2], d[:2]), lambda: topk_backward(x, i, d[:, :1]),
                lambda: topk_backward(x, i, d, n_rows=4), lambda: topk_backward(x, i, d, n_rows=-1), lambda: topk_backward(torch.zeros(1, 32768), i[:1], d[:1])):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: topk_backward(x.double(), i, d), lambda: topk_backward(x, i, d.double()),
                lambda: topk_backward(x, torch.zeros(3, 65, dtype=torch.int16), torch.zeros(3, 65))):
        with pytest.raises(NotImplementedError):
            bad()
