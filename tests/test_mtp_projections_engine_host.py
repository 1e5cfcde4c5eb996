"""The engine takes the draft block's projections as its drafts use them, or says so at once (no GPU needed)."""
import pytest
import torch

from home_seek_amd import checkpoint
from test_checkpoint import D, ckpt  # noqa: F401  (the fixture)


def engine_with(path, e, h):
    eng = checkpoint.load_engine(path, device="cpu")
    mw = {**eng._mtp_weights, "e_proj.weight": e, "h_proj.weight": h}
    return type(eng)(eng.config, eng.store, eng._layer_weights, eng.lm_head, eng.norm_weight, eng.embed, mw)


def test_bf16_projections_are_taken(ckpt):  # noqa: F811
    e, h = torch.randn(D, D).to(torch.bfloat16), torch.randn(D, D).to(torch.bfloat16)
    assert engine_with(ckpt[0], e, h)._mtp_weights["h_proj.weight"] is h


@pytest.mark.parametrize("bad", [torch.zeros(D, D, dtype=torch.float8_e4m3fn), torch.zeros(D, D),
                                 torch.zeros(D, D // 2, dtype=torch.bfloat16), torch.zeros(D * D, dtype=torch.bfloat16)])
def test_others_are_refused_before_the_first_draft(ckpt, bad):  # noqa: F811
    good = torch.zeros(D, D, dtype=torch.bfloat16)
    for e, h in ((bad, good), (good, bad)):
        with pytest.raises(ValueError, match=f"bf16 \\[{D}, {D}\\]"):
            engine_with(ckpt[0], e, h)
