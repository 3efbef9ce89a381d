"""`moe_layer` and `tamd_moe_layer` refuse what the kernels do not take, before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

from triton_amd import _lib
from triton_amd.moe_layer import moe_layer


def good():
    a = _lib.MoeLayerArgs(x=0x1000, x_stride_m=64, logits=0x2000, logits_stride=8, y=0x3000, y_stride_m=64, workspace=0x4000, x_dtype=_lib.BF16,
                          logits_dtype=_lib.F32, n_tokens=65, n_experts=8, n_picks=2, hidden=64, inter=32)
    for w, K in ((a.up, 64), (a.down, 32)):
        w.w, w.w_stride_e, w.w_stride_n, w.scale, w.scale_stride_e, w.scale_stride_n = 0x5000, 64 * K, K // 2, 0x6000, 2 * K, K // 32
    return a


def code(a, size=None):
    return _lib.lib().tamd_moe_layer(C.byref(a), C.sizeof(a) if size is None else size, None)


def test_c_entry_point():
    assert _lib.lib().tamd_moe_layer(None, C.sizeof(_lib.MoeLayerArgs), None) == _lib.E_INVALID
    assert code(good()) == _lib.E_TOO_LARGE   # 65 tokens
    for field, value, want in (("n_tokens", -1, _lib.E_INVALID), ("n_experts", 0, _lib.E_INVALID), ("n_picks", 0, _lib.E_INVALID),
                               ("n_picks", 9, _lib.E_INVALID), ("hidden", 48, _lib.E_INVALID), ("inter", 0, _lib.E_INVALID), ("inter", 33, _lib.E_INVALID),
                               ("x_dtype", _lib.F32, _lib.E_UNSUPPORTED), ("logits_dtype", _lib.FP8_E4M3, _lib.E_INVALID),
                               ("n_experts", 513, _lib.E_TOO_LARGE)):
        a = good()
        setattr(a, field, value)
        assert code(a) == want, field
    for field, value, want in (("x", 0, _lib.E_INVALID), ("workspace", 0, _lib.E_INVALID), ("y", None, _lib.E_INVALID), ("x", 0x1008, _lib.E_ALIGNMENT),
                               ("x_stride_m", 68, _lib.E_ALIGNMENT), ("x_stride_m", 1 << 25, _lib.E_UNSUPPORTED), ("x_stride_m", -64, _lib.E_INVALID),
                               ("workspace", 0x4004, _lib.E_ALIGNMENT), ("hidden", 1 << 21, _lib.E_UNSUPPORTED)):
        a = good()
        a.n_tokens = 4
        setattr(a, field, value)
        assert code(a) == want, (field, value)
    for field, value, want in (("w", 0, _lib.E_INVALID), ("scale", 0, _lib.E_INVALID), ("w", 0x5004, _lib.E_ALIGNMENT), ("w_stride_n", 40, _lib.E_ALIGNMENT),
                               ("w_stride_e", 8, _lib.E_ALIGNMENT), ("w_stride_e", -16, _lib.E_INVALID), ("w_layout", 2, _lib.E_INVALID),
                               ("scale_layout", 7, _lib.E_INVALID), ("w_stride_n", 1 << 26, _lib.E_UNSUPPORTED), ("scale_stride_n", 1 << 30, _lib.E_UNSUPPORTED)):
        for part in ("up", "down"):
            a = good()
            a.n_tokens = 4
            setattr(getattr(a, part), field, value)
            assert code(a) == want, (part, field, value)
    a = good()
    a.n_tokens, a.up.bias, a.up.bias_dtype = 4, 0x7000, _lib.FP8_E5M2
    assert code(a) == _lib.E_INVALID
    a = good()
    assert code(a, C.sizeof(a) - 8) == _lib.E_INVALID and code(a, C.sizeof(a) + 8) == _lib.E_INVALID
    a.n_tokens = 0
    assert code(a) == 0
    assert _lib.lib().tamd_moe_layer_workspace(4, 2, 32) > 4 * 2 * 32 * 4 and _lib.lib().tamd_moe_layer_workspace(-1, 2, 32) == _lib.E_INVALID


def test_structure_matches_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [("tamd_moe_layer_args", n, getattr(_lib.MoeLayerArgs, n).offset) for n, _ in _lib.MoeLayerArgs._fields_]
    fields += [("tamd_moe_weights", n, getattr(_lib.MoeWeights, n).offset) for n, _ in _lib.MoeWeights._fields_]
    src = tmp_path / "at.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "triton_amd.h"\nint main(void){printf("%zu\\n", sizeof(tamd_moe_layer_args));\n'
                   + "".join(f'printf("%zu\\n", offsetof({s}, {n}));\n' for s, n, _ in fields) + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "at")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "at")]).split()]
    assert sizes == [C.sizeof(_lib.MoeLayerArgs)] + [at for _, _, at in fields]


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        moe_layer(torch.zeros(1, 32, dtype=torch.bfloat16), torch.zeros(1, 8), 2, None, None, None, None, None, None, None)
