"""The stream that kernels are launched on, with torch's shortcut to its handle and without."""
import types

import pytest
import torch


@pytest.mark.parametrize("shortcut", [True, False])
def test_the_handle_comes_from_the_shortcut_or_from_the_public_stream(shortcut, monkeypatch):
    from mqgan_amd import _lib
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(cuda_stream=0x5000))
    monkeypatch.setattr(_lib, "_raw_stream", (lambda device: 0x4000 + device) if shortcut else None)
    assert _lib.stream().value == (0x4003 if shortcut else 0x5000)


@pytest.mark.gpu
@pytest.mark.parametrize("shortcut", [True, False])
def test_kernels_run_on_the_current_stream(shortcut, monkeypatch):
    from mqgan_amd import _lib, ops
    if not shortcut:
        monkeypatch.setattr(_lib, "_raw_stream", None)
    side = torch.cuda.Stream()
    assert (_lib.stream().value or 0) == torch.cuda.current_stream().cuda_stream
    z, u = torch.randn(50, 100, device="cuda"), torch.rand(50, device="cuda")
    want = ops.sample_codes(z, u)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert _lib.stream().value == side.cuda_stream != 0
        got = ops.sample_codes(z, u)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
