"""Sizes of `sample`'s workspace (no GPU needed), and that a call of a large batch does not allocate what it does not use (GPU)."""
import pytest
import torch

from triton_amd import _lib, _native


def exact(R, V):
    return _lib.lib().tamd_sample_workspace_exact(R, V)


def test_sizes():
    most = _lib.lib().tamd_sample_workspace
    assert exact(256, 100003) == 16 and exact(4096, 1 << 20) == 16 and exact(1000, 2000) == 16   # a workgroup does a row alone
    assert exact(1, 131072) == most(1, 131072) > 10000 and exact(64, 131072) == most(64, 131072) > 60 * most(1, 131072)
    assert exact(-1, 5) == most(5, -1) == exact(5, -1) == _lib.E_INVALID
    for V in (1, 24000, 24001, 30000, 50001, 100003, 1 << 20):
        before = 0
        for R in (0, 1, 7, 60, 143, 144, 160, 200, 255, 256, 257, 300, 512, 600, 1000, 3000, 4095, 4096, 5000, 1 << 20):
            assert before <= most(R, V) and exact(R, V) <= most(R, V)   # what serves R rows serves fewer
            before = most(R, V)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_what_a_call_allocates(native, device, monkeypatch):
    from triton_amd.sampling import sample
    z, u = torch.randn(256, 100003, device=device), torch.rand(256, device=device)
    want = sample(z, u, top_p=0.9)
    if not native:
        monkeypatch.setattr(_native, "sample", lambda *args: None)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(device)
    before = torch.cuda.memory_allocated(device)
    got = sample(z, u, top_p=0.9)
    assert torch.cuda.max_memory_allocated(device) - before < 1 << 16
    few = sample(z[:3], u[:3], top_p=0.9)
    assert torch.equal(got, want) and torch.equal(few, want[:3])
