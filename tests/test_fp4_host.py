"""Argument checks of the 4-bit entry points, before anything is launched (no GPU needed)."""
from home_seek_amd import _lib

A = 4096  # an aligned address that is never read


def quant(x=A, ld=64, kind=1, m=4, k=64, codes=A, scale=A):
    return _lib.lib().hsmoe_fp4_quant(x, ld, kind, m, k, codes, scale, None)


def linear(x=A, kind=1, ld=64, xs=None, m=4, k=64, w=A, ws=A, n=32, out_kind=1, out=A, work=A, nwork=1 << 30):
    return _lib.lib().hsmoe_fp4_linear(x, kind, ld, xs, m, k, w, ws, n, out_kind, out, work, nwork, None)


def test_quant_rejects_bad_arguments():
    for kw in (dict(x=None), dict(codes=None), dict(scale=None), dict(m=-1), dict(k=0), dict(kind=2)):
        assert quant(**kw) == -1, kw
    for kw in (dict(k=40), dict(k=1 << 22, ld=1 << 22), dict(x=A + 8), dict(ld=63), dict(ld=68), dict(ld=66, kind=0), dict(codes=A + 2),
               dict(k=128, ld=128, scale=A + 1), dict(m=1 << 31)):
        assert quant(**kw) == -2, kw
    assert quant(x=None, m=0) == 0


def test_linear_rejects_bad_arguments():
    for kw in (dict(x=None), dict(w=None), dict(ws=None), dict(out=None), dict(kind=3), dict(kind=2), dict(out_kind=2), dict(m=-1),
               dict(n=0), dict(k=0)):
        assert linear(**kw) == -1, kw
    for kw in (dict(n=12), dict(k=48), dict(x=A + 8), dict(ld=32), dict(w=A + 8), dict(out=A + 8), dict(n=1 << 31),
               dict(k=512, ld=512, ws=A + 4), dict(m=1 << 20, k=1 << 21, ld=1 << 21, nwork=1 << 50)):
        assert linear(**kw) == -2, kw
    assert linear(m=0, x=None) == 0
    size = _lib.lib().hsmoe_fp4_linear_workspace_size
    assert size(1, 4096, 4096, 1) == 0 and size(40, 4096, 4096, 2) == 0 and size(40, 4096, 4096, 1) > 0
    need = size(500, 2048, 4096, 1)
    big = dict(m=500, n=2048, k=4096, ld=4096)
    assert need >= 500 * 2048 + 128 * 512 + 128 * 2048
    assert linear(**big, nwork=need - 1) == -4 and linear(**big, work=None) == -4 and linear(**big, work=A + 8) == -2


def test_refuses_what_one_launch_does_not_hold():
    assert quant(m=1 << 28, k=32, ld=32) == -2
    assert linear(m=1, n=1 << 28, k=32, ld=32) == -2
