"""Which device's stream _lib.stream_ptr hands to a launch (no GPU needed)."""
import pytest
import torch

from home_seek_amd import _lib


@pytest.fixture()
def streams(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)


@pytest.mark.parametrize("device,want", [(None, 1003), (torch.device("cuda"), 1003), (torch.device("cuda", 1), 1001),
                                         ("cuda:2", 1002), ("cuda", 1003), (0, 1000)])
def test_a_device_in_any_form_that_torch_takes(streams, device, want):
    assert _lib.stream_ptr(device) == want


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu")])
def test_no_stream_of_a_cpu(streams, device):
    with pytest.raises(ValueError, match="cpu"):
        _lib.stream_ptr(device)
