"""`pack_int4`'s layout and refusals, and what `tamd_matvec` refuses before anything is launched (no GPU needed)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from triton_amd import _lib
from triton_amd.matvec import matvec, pack_int4


def good():
    return _lib.MatvecArgs(x=0x1000, x_stride_m=128, codes=0x2000, scales=0x3000, y=0x4000, y_stride_m=16, x_dtype=_lib.BF16, scale_dtype=_lib.F16,
                           bias_dtype=_lib.F32, y_dtype=_lib.F32, M=0, N=16, K=128, group=64)


def code(a, size=None):
    return _lib.lib().tamd_matvec(C.byref(a), C.sizeof(a) if size is None else size, None)


def test_c_entry_point():
    assert _lib.lib().tamd_matvec(None, C.sizeof(_lib.MatvecArgs), None) == _lib.E_INVALID
    assert code(good()) == 0   # no rows
    assert code(good(), C.sizeof(_lib.MatvecArgs) - 4) == _lib.E_INVALID
    for field, value, want in (("M", -1, _lib.E_INVALID), ("K", 0, _lib.E_INVALID), ("K", 96, _lib.E_INVALID), ("group", 16, _lib.E_UNSUPPORTED),
                               ("x_dtype", _lib.F32, _lib.E_UNSUPPORTED), ("scale_dtype", _lib.F32, _lib.E_UNSUPPORTED), ("y_dtype", _lib.FP8_E4M3, _lib.E_INVALID)):
        a = good()
        setattr(a, field, value)
        assert code(a) == want, field
    for field, value, want in (("x", 0, _lib.E_INVALID), ("codes", 0, _lib.E_INVALID), ("scales", 0, _lib.E_INVALID), ("y", 0, _lib.E_INVALID),
                               ("x", 0x1008, _lib.E_ALIGNMENT), ("codes", 0x2008, _lib.E_ALIGNMENT), ("zeros", 0x5001, _lib.E_ALIGNMENT),
                               ("x_stride_m", 100, _lib.E_ALIGNMENT), ("x_stride_m", -128, _lib.E_INVALID), ("x_stride_m", 1 << 25, _lib.E_UNSUPPORTED),
                               ("K", 1 << 21, _lib.E_UNSUPPORTED), ("M", 1 << 30, _lib.E_UNSUPPORTED)):
        a = good()
        a.M = 2
        setattr(a, field, value)
        assert code(a) == want, field
    a = good()
    a.bias, a.bias_dtype = 0x6000, _lib.MXFP4
    assert code(a) == _lib.E_INVALID


def test_structure_matches_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in _lib.MatvecArgs._fields_]
    (tmp_path / "at.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "triton_amd.h"\nint main(void){printf("%zu\\n", sizeof(tamd_matvec_args));\n'
                                   + "".join(f'printf("%zu\\n", offsetof(tamd_matvec_args, {n}));\n' for n in names) + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "at.c"), "-o", str(tmp_path / "at")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "at")]).split()]
    assert sizes == [C.sizeof(_lib.MatvecArgs)] + [getattr(_lib.MatvecArgs, n).offset for n in names]


@pytest.mark.parametrize("K,N,group", [(32, 1, 32), (96, 5, 32), (128, 16, 128), (448, 33, 64), (1056, 40, 32)])
def test_layout(K, N, group):
    """Every code where the header says, and back."""
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 256, (K // 2, N), dtype=torch.uint8, generator=g)
    scales = torch.randn(K // group, N, generator=g).to(torch.bfloat16)
    zeros = torch.randint(0, 16, (K // group, N), dtype=torch.uint8, generator=g)
    w = pack_int4(codes, scales, zeros, group)
    dwords = w.data.contiguous().numpy().view("uint32").reshape(*w.data.shape[:2], 4, 16, 4)
    for k in range(0, K, 3):
        for n in range(N):
            b, t, h, i = k // 128, k % 128 // 32, k % 32 // 8, k % 8
            assert int(dwords[n // 16, b, h, n % 16, t]) >> (4 * (i // 2) + 16 * (i % 2)) & 15 == int(codes[k // 2, n]) >> (4 * (k % 2)) & 15
            at = (n // 16, b, n % 16, k % 128 // group)
            assert w.scales[at] == scales[k // group, n] and w.zeros[at] == zeros[k // group, n]
    c, s, z = w.unpack()
    assert torch.equal(c, codes) and torch.equal(s, scales) and torch.equal(z, zeros)


def test_pack_refusals():
    codes, scales = torch.zeros(64, 8, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.bfloat16)
    for bad in (lambda: pack_int4(codes.int(), scales, None, 64), lambda: pack_int4(codes, scales, None, 128), lambda: pack_int4(codes[:60], scales, None, 64),
                lambda: pack_int4(codes, scales, scales, 64), lambda: pack_int4(codes, scales, torch.zeros(2, 7, dtype=torch.uint8), 64),
                lambda: pack_int4(codes[:0], scales[:0], None, 64)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: pack_int4(codes, scales, None, 16), lambda: pack_int4(codes, scales.float(), None, 64)):
        with pytest.raises(NotImplementedError):
            bad()
    with pytest.raises(RuntimeError, match="GPU"):
        matvec(torch.zeros(1, 128, dtype=torch.bfloat16), pack_int4(codes, scales, None, 64))
