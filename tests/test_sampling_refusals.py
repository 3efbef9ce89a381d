"""What `sample` and `tamd_sample` refuse before anything is launched (no GPU needed)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from triton_amd import _lib
from triton_amd.sampling import sample


def good():
    return _lib.SampleArgs(logits=0x1000, logits_stride=100, u=0x2000, tokens=0x3000, workspace=0x4000, logits_dtype=_lib.F32, R=0, V=100, temperature_value=1.0,
                           top_p_value=1.0)


def code(a, size=None):
    return _lib.lib().tamd_sample(C.byref(a), C.sizeof(a) if size is None else size, None)


def test_c_entry_point():
    assert _lib.lib().tamd_sample(None, C.sizeof(_lib.SampleArgs), None) == _lib.E_INVALID
    assert code(good()) == 0 and code(good(), C.sizeof(_lib.SampleArgs) + 8) == _lib.E_INVALID
    for field, value, want in (("R", -1, _lib.E_INVALID), ("V", 0, _lib.E_INVALID), ("V", (1 << 20) + 1, _lib.E_TOO_LARGE), ("R", (1 << 20) + 1, _lib.E_TOO_LARGE),
                               ("logits_dtype", _lib.FP8_E4M3, _lib.E_UNSUPPORTED)):
        a = good()
        setattr(a, field, value)
        assert code(a) == want, field
    for field in ("logits", "u", "tokens", "workspace"):
        a = good()
        a.R = 1
        setattr(a, field, None)
        assert code(a) == _lib.E_INVALID, field
    a = good()
    a.R, a.logits_stride = 2, -100
    assert code(a) == _lib.E_INVALID
    assert _lib.lib().tamd_sample_workspace(3, 1000) > 0 and _lib.lib().tamd_sample_workspace(-1, 5) == _lib.E_INVALID


def test_structure_matches_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.SampleArgs._fields_]
    (tmp_path / "at.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "triton_amd.h"\nint main(void){printf("%zu\\n", sizeof(tamd_sample_args));\n'
                                   + "".join(f'printf("%zu\\n", offsetof(tamd_sample_args, {n}));\n' for n in names) + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "at.c"), "-o", str(tmp_path / "at")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "at")]).split()]
    assert sizes == [C.sizeof(_lib.SampleArgs)] + [getattr(_lib.SampleArgs, n).offset for n in names]


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        sample(torch.zeros(1, 8), torch.zeros(1))
