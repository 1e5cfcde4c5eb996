"""Argument checks of the linear entry points, before anything is launched (no GPU needed)."""
from home_seek_amd import _lib

A = 4096  # an aligned address that is never read


def linear(x=A, ldx=64, m=4, k=64, w=A, w_up=None, ldw=64, wg=0, n=32, off=None, g=1, b=None, bu=None, res=None, ldr=32,
           act=0, limit=1.0, kind=1, out=A, pre=None, ws=None, nws=0):
    return _lib.lib().hsmoe_linear(x, ldx, m, k, w, w_up, ldw, wg, n, off, g, b, bu, res, ldr, act, limit, kind, out, pre,
                                   ws, nws, None)


def test_linear_rejects_bad_arguments():
    for kw in (dict(x=None), dict(w=None), dict(out=None), dict(m=-1), dict(n=0), dict(k=0), dict(g=0), dict(g=2),
               dict(act=3), dict(kind=2), dict(act=2), dict(w_up=A), dict(act=2, w_up=A, limit=0.0),
               dict(act=2, w_up=A, limit=float("nan")), dict(bu=A), dict(ldx=56), dict(ldw=56), dict(res=A, ldr=24)):
        assert linear(**kw) == -1, kw
    for kw in (dict(n=30), dict(k=60), dict(x=A + 2), dict(ldx=65), dict(w=A + 8), dict(ldw=68), dict(out=A + 4),
               dict(b=A + 2), dict(pre=A + 8), dict(res=A + 2), dict(off=A + 2, g=2), dict(off=A, g=2, wg=4),
               dict(off=A, g=1025), dict(m=1 << 31), dict(m=(1 << 31) - 1000), dict(ldx=1 << 22), dict(m=(1 << 31) - 1025, n=1 << 20)):
        assert linear(**kw) == -2, kw
    assert linear(x=None, m=0) == 0
    big = dict(m=64, k=4096, ldx=4096, ldw=4096, n=4096)
    need = _lib.lib().hsmoe_linear_workspace_size(64, 4096, 4096, 1, 0)
    assert need > 0 and linear(**big) == -4 and linear(**big, ws=A, nws=need - 1) == -4
    assert linear(**big, ws=A + 4, nws=need) == -2


def test_gradient_entry_points_reject_bad_arguments():
    L = _lib.lib()
    need = L.hsmoe_linear_act_grad_workspace_size(4096, 4096, 1, 0)
    assert need > 0 and need % (4096 * 4) == 0
    assert L.hsmoe_linear_act_grad_workspace_size(4096, 4096, 1, 2) == 2 * need
    act = lambda *a: L.hsmoe_linear_act_grad(*a, None)
    assert act(A, 4096, None, 4096, 4096, 0, 1.0, None, 1, None, A, None, A, need - 1) == -4
    assert act(A, 4096, None, 4096, 4096, 1, 1.0, None, 1, A, None, None, None, 0) == -1   # pre missing
    assert act(A, 4096, None, 4096, 4096, 0, 1.0, None, 1, None, A, A, A, need) == -1      # an up bias without swiglu
    assert act(A, 4096, A, 4096, 4096, 2, -1.0, None, 1, A, None, None, None, 0) == -1
    assert act(A, 4090, None, 4096, 4096, 0, 1.0, None, 1, None, A, None, A, need) == -2
    assert act(None, 4096, None, 4096, 4096, 0, 1.0, None, 1, None, None, None, None, 0) == 0
    inp = lambda *a: L.hsmoe_linear_grad_input(*a, None, 0, None)
    assert inp(A, 32, 4, 32, A, None, 64, 0, 64, None, 1, None) == -1
    assert inp(A, 32, 4, 32, A, A, 64, 0, 64, None, 1, A) == -1       # dz has two matrices' columns
    assert inp(A, 32, 4, 32, A + 2, None, 64, 0, 64, None, 1, A) == -2
    assert inp(None, 32, 0, 32, None, None, 64, 0, 64, None, 1, None) == 0
    wgt = lambda *a: L.hsmoe_linear_grad_weight(*a, None, 0, None)
    assert wgt(A, 32, A, 64, 4, 32, 64, None, 1, 5, A, None) == -1
    assert wgt(A, 32, None, 64, 4, 32, 64, None, 1, 1, A, None) == -1
    assert wgt(A, 32, A, 64, 4, 32, 60, None, 1, 1, A, None) == -2
    assert L.hsmoe_linear_grad_workspace_size(64, 4096, 4096, 1, 0) > 0
    assert inp(A, 4096, 64, 4096, A, None, 4096, 0, 4096, None, 1, A) == -4
