"""What `dispatch`, `combine`, their gradients and the C entry points refuse before anything is launched (no GPU needed)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from triton_amd import _lib
from triton_amd.dispatch import combine, combine_backward, dispatch, dispatch_backward

ENTRIES = ("tamd_dispatch", "tamd_combine")


def good(**more):
    return _lib.TokenRowsArgs(**{**dict(src=0x1000, src_stride=64, dst=0x2000, dst_stride=64, row_indx=0x3000, row_indx_stride=4, dtype=_lib.BF16, T=0, k=4, H=64, n_rows=8),
                                 **more})


@pytest.mark.parametrize("entry", ENTRIES)
def test_c_entry_points(entry):
    f = getattr(_lib.lib(), entry)
    code = lambda a, size=C.sizeof(_lib.TokenRowsArgs): f(C.byref(a), size, None)  # noqa: E731
    assert f(None, C.sizeof(_lib.TokenRowsArgs), None) == _lib.E_INVALID
    assert code(good()) == 0 and code(good(), C.sizeof(_lib.TokenRowsArgs) + 8) == _lib.E_INVALID
    assert code(good(T=3, H=0)) == 0
    for field in ("T", "k", "H", "n_rows", "src_stride", "dst_stride", "row_indx_stride", "gates_stride", "other_stride", "dots_stride"):
        assert code(good(**{field: -1})) == _lib.E_INVALID, field
    for dtype in (_lib.FP8_E4M3, _lib.MXFP4, 17):
        assert code(good(dtype=dtype)) == _lib.E_UNSUPPORTED
        assert code(good(gates=0x4000, gates_dtype=dtype)) == _lib.E_UNSUPPORTED
    for field in ("src", "dst", "row_indx"):
        assert code(good(T=3, **{field: None})) == _lib.E_INVALID, field
        if field != "row_indx":
            assert code(good(T=3, **{field: 0x1001})) == _lib.E_ALIGNMENT, field
    assert code(good(T=3, row_indx=0x3002)) == _lib.E_ALIGNMENT
    assert code(good(T=3, gates=0x4002, gates_dtype=_lib.F32)) == code(good(T=3, gates=0x4001, gates_dtype=_lib.BF16)) == _lib.E_ALIGNMENT
    assert code(good(T=1 << 28)) == code(good(T=1 << 26, H=1000)) == _lib.E_TOO_LARGE     # more threads than a launch has
    assert code(good(T=3, dots=0x5000, dots_stride=4)) == _lib.E_INVALID        # (without the other operand)
    assert code(good(T=3, dots=0x5000, dots_stride=4, other=0x6001)) == _lib.E_ALIGNMENT


def test_structure_matches_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.TokenRowsArgs._fields_]
    (tmp_path / "at.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "triton_amd.h"\nint main(void){printf("%zu\\n", sizeof(tamd_token_rows_args));\n'
                                   + "".join(f'printf("%zu\\n", offsetof(tamd_token_rows_args, {n}));\n' for n in names) + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "at.c"), "-o", str(tmp_path / "at")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "at")]).split()]
    assert sizes == [C.sizeof(_lib.TokenRowsArgs)] + [getattr(_lib.TokenRowsArgs, n).offset for n in names]


def test_cpu_tensors_are_refused():
    p = torch.zeros(2, 1, dtype=torch.int32)
    for f in (dispatch, combine, combine_backward, dispatch_backward):
        with pytest.raises(RuntimeError, match="GPU"):
            f(torch.zeros(2, 8), p)


@pytest.fixture
def as_if_on_the_gpu(monkeypatch):
    """The checks behind the first one, on the CPU; nothing is launched."""
    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    for entry in ENTRIES:
        monkeypatch.setattr(_lib.lib(), entry, lambda *a: pytest.fail("launched"))


def test_shapes_and_types(as_if_on_the_gpu):
    x, p, gates = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    rows = torch.zeros(6, 8)
    for call in (lambda: dispatch(x[0], p), lambda: dispatch(x, p[0]), lambda: dispatch(x, p.long()), lambda: dispatch(x[:2], p),
                 lambda: dispatch(x, p, gates=gates[:2]), lambda: dispatch(x, p, out=rows.double()), lambda: dispatch(x, p, out=rows[:, :4]),
                 lambda: dispatch(x, p, out=torch.zeros(8, 6).t()), lambda: dispatch(x, p, out=rows[:1].expand(6, 8)),
                 lambda: combine(rows, p, out=rows), lambda: combine(rows, p, out=x.half()), lambda: combine(rows, p, gates=gates.t()),
                 lambda: combine_backward(x, p, rows=rows[:5], gates=gates), lambda: combine_backward(x, p, rows=rows.half(), gates=gates),
                 lambda: combine_backward(x, p, rows=rows, gates=gates, out=torch.zeros(5, 8)), lambda: dispatch_backward(rows, p, x=x[:2], gates=gates),
                 lambda: dispatch_backward(rows, p, x=rows, gates=gates)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: dispatch(x.double(), p), lambda: combine(rows.to(torch.float8_e4m3fn), p), lambda: dispatch(x, p, gates=gates.double()),
                 lambda: dispatch_backward(rows.long(), p)):
        with pytest.raises(NotImplementedError):
            call()
