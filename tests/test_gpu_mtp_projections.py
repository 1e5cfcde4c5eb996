"""The draft block's projections (h_proj(hnorm(h)) + e_proj(enorm(e))) in the engine's draft loop."""
import pytest
import torch

from home_seek_amd import ops, stack
from home_seek_amd.engine import rms_norm

pytestmark = pytest.mark.gpu

D, V = 512, 1000


@pytest.fixture()
def eng(dev):
    e = stack.build_stack(3, n_layers=2, n_experts=16, d=D, i=512, vocab=V, top_k=4, n_hash=1, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    for n in ("e_proj", "h_proj"):
        e._mtp_weights[f"{n}.weight"] = (torch.randn((D, D), generator=g, device=dev) * D ** -0.5).to(torch.bfloat16)
    return e


def test_drafts_go_through_the_projections(eng, dev):
    mw, eps = eng._mtp_weights, eng.config.rms_norm_eps
    h = eng._forward_stack(torch.tensor([[5]], device=dev))[0]
    tok = torch.tensor([7], device=dev)
    drafts, n = eng._mtp_generate_draft(h, 2, last_token_id=tok)
    prev, want = h.reshape(1, D), []
    for _ in range(2):
        e = rms_norm(eng.embed[tok].reshape(1, D), mw["enorm.weight"], eps)
        g = rms_norm(prev.reshape(1, D), mw["hnorm.weight"], eps)
        proj = e.double() @ mw["e_proj.weight"].double().T
        h_in = (g.double() @ mw["h_proj.weight"].double().T + proj.to(torch.bfloat16).double())
        # within one bf16 step of the sum (the projection's fp32 sums may round its bf16 value the other way)
        got = ops.linear(g, mw["h_proj.weight"], residual=ops.linear(e, mw["e_proj.weight"]))
        assert bool(((got.double() - h_in).abs() <= 2.0 ** -8 * (h_in.abs() + proj.abs()) + 1e-5).all())
        prev, hf = eng._forward_layer_norm(got.reshape(1, 1, D), mw["layer"], mw["layer_idx"], tok.reshape(1, 1), mw["norm.weight"])
        tok = ops.lm_head_accept(hf, eng.lm_head, None, want_logits=False)[1]
        want.append(int(tok))
    assert n == 2 and drafts.reshape(-1).tolist() == want


def test_greedy_stream_is_the_same_with_other_drafts(eng, dev):
    """Drafts change how many tokens a step brings, never which."""
    with_proj = eng.generate_greedy(3, 6)[0]
    plain = stack.build_stack(3, n_layers=2, n_experts=16, d=D, i=512, vocab=V, top_k=4, n_hash=1, device=dev)
    without = plain.generate_greedy(3, 6)[0]
    n = min(len(with_proj), len(without))
    assert n >= 6 and with_proj[:n] == without[:n]


def test_one_projection_alone_is_refused(eng):
    mw = dict(eng._mtp_weights)
    del mw["h_proj.weight"]
    with pytest.raises(ValueError, match="projections"):
        type(eng)(eng.config, eng.store, eng._layer_weights, eng.lm_head, eng.norm_weight, eng.embed, mw)
