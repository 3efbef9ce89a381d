"""Kernels' sources, read as text: where the lanes of one wave exchange data through a part of LDS that is theirs, without a barrier, the place that
a lane reads is one that the compiler cannot tell from the places that it writes (wave_lds_offset in common.h), so that it leaves them in order."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_amd", "csrc")
OF_A_WAVE = re.compile(r"uint8_t \*const (\w+) = lds[^;]*\bwave \*")


def reads(text):
    """(name of a wave's part of LDS, what is added to it where it is read) in every kernel that has one."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in OF_A_WAVE.finditer(text):
        end = text.find("__global__", m.end())
        body = text[m.end():end if end >= 0 else len(text)]
        hidden = re.findall(r"const uint32_t (\w+) = wave_lds_offset\(", body)
        for at in re.findall(rf"\*\(const u32x4_t \*\)\({m.group(1)} \+ ([^;]*);", body):
            yield m.group(1), any(at.startswith(name + " ") for name in hidden)


def test_the_check_finds_them():
    plain = "uint8_t *const r = lds + wave * 5;\n *(u32x4_t *)(r + 1) = x; y = *(const u32x4_t *)(r + at + 2);"
    assert list(reads(plain)) == [("r", False)]
    assert list(reads(plain.replace("y =", "const uint32_t at = wave_lds_offset(3); y ="))) == [("r", True)]
    found = {os.path.basename(p): {n for n, _ in reads(open(p).read())} for p in glob.glob(os.path.join(CSRC, "*.h"))}
    assert found["matvec.h"] == {"x_lds"} and found["moe_layer.h"] == {"rows_lds"}


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip"))), ids=os.path.basename)
def test_reads_of_a_waves_part(path):
    with open(path) as f:
        assert all(hidden for _, hidden in reads(f.read()))
