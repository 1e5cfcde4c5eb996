"""Argument checks of the embedding's entry points, before anything is launched (no GPU needed)."""
from home_seek_amd import _lib

A = 4096  # an aligned address that is never read


def embed(ids=A, ik=1, m=4, table=A, ld=64, tk=1, vocab=100, d=64, ok=1, out=A):
    return _lib.lib().hsmoe_embed(ids, ik, m, table, ld, tk, vocab, d, 1.0, ok, out, None)


def grad(d_out=A, ldd=64, dk=1, ids=A, ik=1, m=4, vocab=100, d=64, add=0, table=A, ld=64, tk=1, ws=A, nws=1 << 30):
    return _lib.lib().hsmoe_embed_grad(d_out, ldd, dk, ids, ik, m, vocab, d, 1.0, add, table, ld, tk, ws, nws, None)


def test_lookup_rejects_bad_arguments():
    for kw in (dict(ids=None), dict(table=None), dict(out=None), dict(m=-1), dict(vocab=0), dict(d=0), dict(ld=63), dict(tk=2), dict(ok=-1),
               dict(ik=2)):
        assert embed(**kw) == -1, kw
    for kw in (dict(m=1 << 31), dict(vocab=1 << 30), dict(d=1 << 23, ld=1 << 23), dict(ld=1 << 31), dict(ids=A + 4), dict(ids=A + 2, ik=0),
               dict(table=A + 1), dict(out=A + 2, ok=0)):
        assert embed(**kw) == -2, kw
    assert embed(ids=None, table=None, out=None, m=0) == 0


def test_gradient_rejects_bad_arguments():
    for kw in (dict(d_out=None), dict(ids=None), dict(table=None), dict(ldd=60), dict(add=2), dict(ld=72), dict(tk=3), dict(dk=2), dict(m=-1)):
        assert grad(**kw) == -1, kw
    for kw in (dict(m=1 << 24), dict(vocab=1 << 30), dict(d_out=A + 1), dict(table=A + 2, tk=0), dict(ws=A + 8)):
        assert grad(**kw) == -2, kw
    need = _lib.lib().hsmoe_embed_grad_workspace_size(4, 64)
    assert need >= 2 * 64 * 4 and grad(nws=need - 1) == -4 and grad(ws=None) == -4
    assert _lib.lib().hsmoe_embed_grad_workspace_size(0, 64) == 0 and grad(m=0, add=1, ws=None, nws=0, d_out=None, ids=None) == 0


def test_refuses_what_one_launch_does_not_hold():
    # threads of a launch are counted in 32 bits: 2^24 rows by workgroups of 256, 2^22 pieces of 16 KB by 1024
    wide = dict(d=4096, ld=4096)
    assert embed(m=1 << 24, **wide) == -2
    for kw in (dict(vocab=1 << 23, **wide), dict(vocab=(1 << 23) - 1, **wide), dict(m=0, vocab=1 << 23, **wide),
               dict(m=(1 << 24) - 1, add=1, d=65536, ld=65536, vocab=100)):
        assert grad(**{"ldd": kw["d"], "nws": 1 << 60, **kw}) == -2, kw
