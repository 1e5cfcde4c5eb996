"""Argument checks of the gradient norm's entry points, before anything is launched (no GPU needed)."""
import ctypes
import math

from home_seek_amd import _lib

A = 1 << 20  # an aligned address that is never read


def clip(ins=(A, 2 * A), counts=(100, 50), kinds=(1, 0), outs=None, out_kinds=None, norm_type=2.0, max_norm=1.0, norm=A // 2, ws=A // 4,
         nws=1 << 30, n=None):
    c = lambda t, v: (t * len(v))(*v)
    outs, out_kinds = ins if outs is None else outs, kinds if out_kinds is None else out_kinds
    arrays = [c(ctypes.c_uint64, ins), c(ctypes.c_int64, counts), c(ctypes.c_int32, kinds), c(ctypes.c_uint64, outs), c(ctypes.c_int32, out_kinds)]
    return _lib.lib().hsmoe_clip_grads(len(ins) if n is None else n, *[ctypes.addressof(a) for a in arrays], norm_type, max_norm, norm, ws, nws,
                                       None)


def test_rejects_bad_arguments():
    for kw in (dict(n=-1), dict(norm=None), dict(counts=(100, -1)), dict(kinds=(1, 2)), dict(out_kinds=(1, 3)), dict(ins=(A, 0)),
               dict(outs=(0, 2 * A)), dict(norm_type=1.0), dict(norm_type=-math.inf), dict(norm_type=math.nan), dict(max_norm=-0.5),
               dict(max_norm=math.nan)):
        assert clip(**kw) == -1, kw
    for kw in (dict(ins=(A + 1, 2 * A)), dict(ins=(A, 2 * A + 2)), dict(outs=(A, 3 * A + 2)), dict(norm=A + 2), dict(ws=A + 4),
               dict(counts=(1 << 40, 1))):
        assert clip(**kw) == -2, kw
    assert clip(nws=8) == -4 and clip(ws=None) == -4


def test_rejects_tensors_that_overlap():
    for kw in (dict(ins=(A, A)), dict(ins=(A, A + 196)), dict(outs=(A, A + 100)), dict(outs=(2 * A, A), kinds=(1, 1)),
               dict(outs=(4 * A, A)), dict(outs=(A, 2 * A), out_kinds=(0, 0)), dict(outs=(A + 16, 2 * A)), dict(outs=(4 * A, 4 * A + 196))):
        assert clip(**kw) == -1, kw
        assert b"overlap" in _lib.lib().hsmoe_last_error()
