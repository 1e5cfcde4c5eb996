"""Argument checks of the block norm's entry points, before anything is launched (no GPU needed)."""
import ctypes

from home_seek_amd import _lib

A = 4096  # an aligned address that is never read


def spec(**kw):
    base = dict(post_w_dev=A, pre_w_dev=A, gate_dev=A, row_kind=1, stream_kind=1, weight_kind=1, gate_kind=1, gate_form=1)
    return _lib.BlockNormSpec(**{**base, **kw})


def forward(f=A, h=A, m=4, d=64, sp=None, eps=1e-6, out=A, n=A, null_spec=False):
    sp = spec() if sp is None else sp
    return _lib.lib().hsmoe_block_norm(f, h, m, d, None if null_spec else ctypes.addressof(sp), 1.0, eps, out, n, None)


def grad(d_h=A, d_n=A, f=A, h=A, m=4, d=64, sp=None, eps=1e-6, d_f=A, d_x=A, d_post=A, d_gate=A, d_pre=A, ws=A, nws=1 << 30):
    sp = spec() if sp is None else sp
    return _lib.lib().hsmoe_block_norm_grad(d_h, d_n, f, h, m, d, ctypes.addressof(sp), 1.0, eps, d_f, d_x, d_post, d_gate, d_pre, ws,
                                            nws, None)


def test_forward_rejects_bad_arguments():
    for kw in (dict(f=None), dict(h=None), dict(out=None), dict(n=None), dict(m=-1), dict(d=0), dict(eps=-1.0), dict(eps=float("nan")),
               dict(null_spec=True), dict(sp=spec(pre_w_dev=None)), dict(sp=spec(gate_dev=None)), dict(sp=spec(gate_form=0)),
               dict(sp=spec(gate_form=4)), dict(sp=spec(row_kind=2)), dict(sp=spec(stream_kind=3)), dict(sp=spec(weight_kind=2)),
               dict(sp=spec(gate_kind=-1))):
        assert forward(**kw) == -1, kw
    for kw in (dict(d=60), dict(d=16392), dict(f=A + 8), dict(h=A + 2), dict(out=A + 4), dict(n=A + 8), dict(m=1 << 31),
               dict(sp=spec(post_w_dev=A + 2)), dict(sp=spec(gate_dev=A + 8)), dict(sp=spec(pre_w_dev=A + 4))):
        assert forward(**kw) == -2, kw
    assert forward(f=None, h=None, out=None, n=None, m=0) == 0


def test_gradient_rejects_bad_arguments():
    for kw in (dict(d_h=None, d_n=None), dict(f=None), dict(h=None), dict(m=-1), dict(sp=spec(post_w_dev=None)), dict(sp=spec(pre_w_dev=None)),
               dict(sp=spec(gate_dev=None, gate_form=0))):
        assert grad(**kw) == -1, kw
    for kw in (dict(d=60), dict(d_h=A + 8), dict(d_n=A + 8), dict(d_f=A + 8), dict(d_x=A + 8), dict(d_gate=A + 2), dict(d_post=A + 2),
               dict(ws=A + 4), dict(sp=spec(gate_form=3), d_gate=A + 8)):
        assert grad(**kw) == -2, kw
    need = _lib.lib().hsmoe_block_norm_grad_workspace_size(4, 64)
    assert need == 3 * 64 * 4 and grad(nws=need - 1) == -4 and grad(ws=None) == -4


def test_refuses_what_one_launch_does_not_hold():
    assert forward(m=1 << 24, d=4096) == -2 and forward(m=1 << 29, d=64) == -2
