"""What the product over ragged rows and its C entry point refuse before anything is launched (no GPU needed)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from triton_amd import _lib
from triton_amd.matmul import FlexCtx, FnSpecs, FusedActivation, PrecisionConfig, matmul
from triton_amd.numerics import InFlexData, OutFlexData
from triton_amd.tensor import RaggedTensorMetadata


def good(**more):
    return _lib.RaggedKArgs(**{**dict(x=0x1000, x_stride=64, d=0x2000, d_stride=64, slice_offs=0x3000, slice_sizes=0x3800, y=0x4000, y_stride_e=4096, y_stride_m=64, K=100, dtype=_lib.BF16,
                                      y_dtype=_lib.BF16, M=0, N=64, E=2), **more})


def test_c_entry_point():
    L = _lib.lib()
    code = lambda a, size=C.sizeof(_lib.RaggedKArgs): L.tamd_ragged_k_matmul(C.byref(a), size, None)  # noqa: E731
    room_of = lambda a: L.tamd_ragged_k_matmul_workspace(C.byref(a), C.sizeof(_lib.RaggedKArgs))  # noqa: E731
    assert L.tamd_ragged_k_matmul(None, C.sizeof(_lib.RaggedKArgs), None) == _lib.E_INVALID
    assert code(good()) == 0 and code(good(), C.sizeof(_lib.RaggedKArgs) - 8) == _lib.E_INVALID
    for field in ("M", "N", "E", "K", "x_stride", "d_stride", "y_stride_e", "y_stride_m"):
        assert code(good(**{field: -1})) == _lib.E_INVALID, field
    for dtype in (_lib.F32, _lib.FP8_E4M3):
        assert code(good(dtype=dtype)) == _lib.E_UNSUPPORTED
    assert code(good(y_dtype=_lib.FP8_E4M3)) == _lib.E_UNSUPPORTED
    for field in ("x", "d", "y", "slice_offs", "slice_sizes"):
        assert code(good(M=64, **{field: None})) == _lib.E_INVALID, field
        assert code(good(M=64, **{field: 0x1001})) == _lib.E_ALIGNMENT, field
    assert code(good(M=64, y_dtype=_lib.F32, y=0x4002)) == _lib.E_ALIGNMENT
    assert code(good(M=64, K=1 << 31)) == _lib.E_TOO_LARGE and code(good(M=2 ** 31 - 1, N=2 ** 31 - 1)) == _lib.E_TOO_LARGE
    # rows that would have to be laid out first, by more threads than a launch has
    assert code(good(M=2047, K=1 << 28, x_stride=2047)) == room_of(good(M=2047, K=1 << 28, x_stride=2047)) == _lib.E_TOO_LARGE
    assert room_of(good(M=2048, K=1 << 28, x_stride=2048)) >= 0
    # long slices of few tiles are cut: their partial sums need room; so do rows that are not whole pieces of 16 bytes
    room = lambda a, size=C.sizeof(_lib.RaggedKArgs): L.tamd_ragged_k_matmul_workspace(C.byref(a), size)  # noqa: E731
    n = room(good(M=64, K=10000))
    assert n > 0 and n % (2 * 64 * 64 * 4) == 0 and room(good(M=64)) == room(good()) == 0
    assert code(good(M=64, K=10000)) == _lib.E_INVALID and code(good(M=64, K=10000, workspace=0x5004)) == _lib.E_ALIGNMENT
    assert room(good(M=64, x=0x1002)) == 100 * 64 * 2 and room(good(M=63, d_stride=65)) == 100 * 64 * 2 * 2 and code(good(M=63)) == _lib.E_INVALID
    assert room(good(M=-1)) == room(good(), 8) == L.tamd_ragged_k_matmul_workspace(None, C.sizeof(_lib.RaggedKArgs)) == _lib.E_INVALID
    assert room(good(M=64, K=1 << 31)) == room(good(M=1 << 24)) == _lib.E_TOO_LARGE


@pytest.mark.parametrize("pitch", [0, 8, 56])
@pytest.mark.parametrize("K", [1, 5, 100])
def test_rows_that_overlap_are_laid_out_first(pitch, K):
    """A pitch below the columns: the copies' bounds would let rows behind a slice in, so there has to be room for rows of their own."""
    room = lambda **more: _lib.lib().tamd_ragged_k_matmul_workspace(C.byref(good(M=64, K=K, **more)), C.sizeof(_lib.RaggedKArgs))  # noqa: E731
    assert room(x_stride=pitch) == room(d_stride=pitch) == K * 64 * 2 and room(x_stride=pitch, d_stride=pitch) == 2 * K * 64 * 2
    assert room() == room(x_stride=72, d_stride=80) == 0


def test_structure_matches_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.RaggedKArgs._fields_]
    (tmp_path / "at.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "triton_amd.h"\nint main(void){printf("%zu\\n", sizeof(tamd_ragged_k_args));\n'
                                   + "".join(f'printf("%zu\\n", offsetof(tamd_ragged_k_args, {n}));\n' for n in names) + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "at.c"), "-o", str(tmp_path / "at")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "at")]).split()]
    assert sizes == [C.sizeof(_lib.RaggedKArgs)] + [getattr(_lib.RaggedKArgs, n).offset for n in names]


def metadata(E):
    table = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return RaggedTensorMetadata(table(E), table(E + 1), table(5, E + 1), table(5, 4))


def test_python_calls(monkeypatch):
    x, d, md = torch.zeros(10, 16).bfloat16(), torch.zeros(10, 24).bfloat16(), metadata(3)
    with pytest.raises(RuntimeError, match="GPU"):
        matmul(x.t(), d, None, md, md)
    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    monkeypatch.setattr(_lib.lib(), "tamd_ragged_k_matmul", lambda *a: pytest.fail("launched"))
    rows = torch.zeros(10, dtype=torch.int32)
    act = FusedActivation(FnSpecs("swiglu", None, ("alpha", "limit"), reduction_n=2), (1.0, 1.0))
    for call in (lambda: matmul(x.t(), d, torch.zeros(3, 24), md, md), lambda: matmul(x.t(), d, None, md, md, gather_indx=rows),
                 lambda: matmul(x.t(), d, None, md, md, scatter_indx=rows), lambda: matmul(x.t(), d, None, md, md, gammas=torch.zeros(10)),
                 lambda: matmul(x.t(), d, None, md, md, betas=torch.zeros(10)), lambda: matmul(x.t(), d, None, md, md, out_alpha=2.0),
                 lambda: matmul(x.t(), d, None, md, md, c_acc_in=torch.zeros(3, 16, 24)), lambda: matmul(x.t(), d, None, md, md, fused_activation=act),
                 lambda: matmul(x.t().float(), d.float(), None, md, md), lambda: matmul(x.t(), d.half(), None, md, md),
                 lambda: matmul(x.t(), d, None, md, md, precision_config=PrecisionConfig(out_dtype=torch.float64)),
                 lambda: matmul(x.t(), d, None, md, md, precision_config=PrecisionConfig(acc_scale=2.0)),
                 lambda: matmul(x.t(), d, None, md, md, precision_config=PrecisionConfig(b_mx_scale=rows))):
        with pytest.raises(NotImplementedError):
            call()
    for call in (lambda: matmul(x, d, None, md, md), lambda: matmul(x.t()[:, :9], d, None, md, md), lambda: matmul(x.t(), d, None, metadata(2), md),
                 lambda: matmul(x.t(), d, None, md, md, c=torch.zeros(3, 16, 23)), lambda: matmul(x.t(), d, None, md, md, c=torch.zeros(3, 24, 16).transpose(1, 2)),
                 lambda: matmul(x.t(), d, None, md, md, c=torch.zeros(3, 1, 24).expand(3, 16, 24)),
                 lambda: matmul(x.t()[None], d[None], None, md, md)):
        with pytest.raises(AssertionError):
            call()


@pytest.mark.parametrize("settings", [dict(c_value_pack_factor=2), *(dict(flex_ctx=FlexCtx(out_data=OutFlexData(**{name: torch.ones(1)}))) for name in ("checksum_scale", "expected_scale", "actual_scale")),
                                      dict(flex_ctx=FlexCtx(acc_data=InFlexData(scale=torch.ones(1)))), dict(a_mx_tensor_scale=torch.ones(1)), dict(c_mx_scale=torch.zeros(1, dtype=torch.uint8))],
                         ids=["packed", "checksum", "expected", "actual", "accumulator", "per tensor", "results' scales"])
@pytest.mark.parametrize("given", [False, True])
def test_settings_that_change_the_result_are_not_dropped(settings, given, monkeypatch):
    """What has no kernel here is refused before the native call as behind it, whether the caller has results of their own or not."""
    from triton_amd import _native
    x, d, md = torch.zeros(10, 16).bfloat16(), torch.zeros(10, 24).bfloat16(), metadata(3)
    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    for holder, name in ((_native, "matmul_ragged_k"), (_lib.lib(), "tamd_ragged_k_matmul")):
        monkeypatch.setattr(holder, name, lambda *a: pytest.fail("called"))
    with pytest.raises(NotImplementedError):
        matmul(x.t(), d, None, md, md, c=torch.zeros(3, 16, 24).bfloat16() if given else None, precision_config=PrecisionConfig(**settings))
