"""The bench line's measured HBM traffic is reported while the sources of its kernels are those it was measured on, whatever else changes."""
import os
import shutil

import pytest

import bench

CSRC = os.path.join("triton_amd", "csrc")


@pytest.fixture
def tree(tmp_path, monkeypatch):
    shutil.copytree(os.path.join(bench.ROOT, CSRC), tmp_path / CSRC)
    shutil.copytree(os.path.join(bench.ROOT, "include"), tmp_path / "include")
    (tmp_path / "profiles").mkdir()
    shutil.copy(os.path.join(bench.ROOT, "profiles", "hbm_traffic.txt"), tmp_path / "profiles")
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    return tmp_path


def append(path):
    with open(path, "a") as f:
        f.write("// another line\n")


@pytest.mark.parametrize("name", ["sampling.hip", "matvec.h", "moe_layer.h", "routing.hip", "host.cpp", "../../include/triton_amd.h"])
def test_other_operators_do_not_count(tree, name):
    before = bench.kernel_sources_digest()
    append(tree / CSRC / name)
    assert bench.kernel_sources_digest() == before


@pytest.mark.parametrize("name", ["moe_matmul.hip", "moe_matmul_impl.h", "moe_matmul_stream.h", "moe_matmul_kkring.h", "common.h", "tile_rules.h", "moe_matmul_fp8.hip"])
def test_the_kernels_sources_do(tree, name):
    before = bench.kernel_sources_digest()
    append(tree / CSRC / name)
    assert bench.kernel_sources_digest() != before


def test_figures_of_other_sources_are_not_reported(tree):
    text = (tree / "profiles" / "hbm_traffic.txt").read_text()
    (tree / "profiles" / "hbm_traffic.txt").write_text(bench.re.sub(r"(digest:\s*)[0-9a-f]+", r"\g<1>" + bench.kernel_sources_digest(), text))
    for workload in ("fc1_prefill", "fc1_decode", "fc2_combine"):
        assert bench.measured_traffic(workload)[0] > 1e8
    append(tree / CSRC / "common.h")
    value, why = bench.measured_traffic("fc1_prefill")
    assert value is None and "stale" in why
