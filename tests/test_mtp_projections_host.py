"""load_engine(mtp_projections=True): both projections under their keys, or an error (no GPU needed)."""
import pytest
import torch
from safetensors.torch import load_file, save_file

from home_seek_amd import checkpoint
from test_checkpoint import D, ckpt  # noqa: F401  (the fixture)


def _with(tmp_path, path, more):
    import os
    for f in os.listdir(path):
        if f.endswith(".safetensors"):
            save_file(load_file(os.path.join(path, f)), str(tmp_path / f))
    save_file(more, str(tmp_path / "proj.safetensors"))
    return str(tmp_path)


def test_projections_are_loaded_when_asked_for(ckpt, tmp_path):  # noqa: F811
    g = torch.Generator().manual_seed(3)
    e8 = torch.randint(0, 126, (D, D), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.full((D // 128, D // 128), 126, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    h = torch.randn(D, D, generator=g).to(torch.bfloat16)
    path = _with(tmp_path, ckpt[0], {"mtp.0.e_proj.weight": e8, "mtp.0.e_proj.scale": scale, "mtp.0.h_proj.weight": h})
    mw = checkpoint.load_engine(path, device="cpu", mtp_projections=True)._mtp_weights
    assert torch.equal(mw["h_proj.weight"], h)
    assert torch.equal(mw["e_proj.weight"], (e8.to(torch.float32) * 0.5).to(torch.bfloat16))
    assert "h_proj.weight" not in checkpoint.load_engine(path, device="cpu")._mtp_weights  # as before unless asked for


def test_missing_projection_is_an_error(ckpt):  # noqa: F811
    with pytest.raises(KeyError, match="e_proj"):
        checkpoint.load_engine(ckpt[0], device="cpu", mtp_projections=True)
