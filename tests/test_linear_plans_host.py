"""hsmoe_linear_plan: its arguments, and that the GPU tests' shapes reach every way of doing a product that the rule
takes over the range of sizes (no GPU needed: the rule is the host's, for 256 CUs)."""
import ctypes
import math
import random

import test_gpu_linear as first
import test_gpu_linear_plans as more
from home_seek_amd import _lib

OUT, DX, DW = _lib.LINEAR_OUT, _lib.LINEAR_DX, _lib.LINEAR_DW


def plan(product, m, n, k, groups=1, act=_lib.ACT_NONE):
    """(rows, columns, workgroups per CU, parts)"""
    p = (ctypes.c_int32 * 4)()
    assert _lib.lib().hsmoe_linear_plan(product, m, n, k, groups, act, p) == 0
    return tuple(p)


def way(product, m, n, k, groups, grouped, act):
    rows, cols, per_cu, parts = plan(product, m, n, k, groups, act)
    return product, (rows, cols, per_cu), parts > 1, grouped, act == _lib.ACT_SWIGLU


def test_arguments():
    call, p = _lib.lib().hsmoe_linear_plan, (ctypes.c_int32 * 4)()
    for bad in ((3, 1, 8, 8, 1, 0), (OUT, 0, 8, 8, 1, 0), (OUT, 1, 0, 8, 1, 0), (OUT, 1, 8, 0, 1, 0), (OUT, 1, 8, 8, 0, 0),
                (OUT, 1, 8, 8, 1, 3)):
        assert call(*bad, p) == -1, bad
    assert call(OUT, 1, 8, 8, 1, 0, None) == -1


def test_a_split_reduction_is_what_needs_a_workspace():
    size = _lib.lib().hsmoe_linear_workspace_size
    for m, n, k, g in ((1, 4096, 4096, 1), (64, 4096, 4096, 1), (500, 2048, 4096, 1), (20, 3608, 4096, 4)):
        for act in (_lib.ACT_NONE, _lib.ACT_SWIGLU):
            parts = plan(OUT, m, n, k, g, act)[3]
            assert size(m, n, k, g, act) == (parts > 1) * parts * m * n * (2 if act == _lib.ACT_SWIGLU else 1) * 4


def _parameters(test, names):
    return next(mark.args[1] for mark in test.pytestmark if mark.name == "parametrize" and mark.args[0] == names)


def test_every_way_is_tested():
    acts = (_lib.ACT_NONE, _lib.ACT_SWIGLU)
    tested = set()
    for act in acts:
        for m, n, k in first.SHAPES + more.FORWARD:
            tested.add(way(OUT, m, n, k, 1, False, act))
        for m, n, k in list(_parameters(first.test_dense_gradient, "m,n,k")) + more.GRAD:
            tested |= {way(p, m, n, k, 1, False, act) for p in (DX, DW)}
        for m, top_k, e, n, k, _ in first.GROUPS:
            tested |= {way(p, m * top_k, n, k, e, True, act) for p in (OUT, DX, DW)}
        for m, top_k, e, n, k in more.FORWARD_GROUPS:
            tested.add(way(OUT, m * top_k, n, k, e, True, act))
        for m, top_k, e, n, k in more.GRAD_GROUPS:
            tested |= {way(p, m * top_k, n, k, e, True, act) for p in (DX, DW)}
    rng = random.Random(3)

    def size(top):
        return int(math.exp(rng.uniform(0.0, math.log(top))))

    missing = {}
    for _ in range(200000):
        m, n, k, grouped = size(20000), 8 * size(1100), 8 * size(1100), rng.random() < 0.5
        args = (rng.choice((OUT, DX, DW)), m, n, k, size(512) if grouped else 1, grouped, rng.choice(acts))
        if way(*args) not in tested:
            missing.setdefault(way(*args), args)
    assert not missing, missing


def test_the_weights_gradients_are_tiled_each_for_itself():
    """One expert's columns that end inside a tile leave its rest empty: widths of as many whole tiles of 128 cost
    the same (but for the sums of a split reduction), and so have the same tile."""
    rng = random.Random(5)
    wrong = []
    for _ in range(20000):
        m, n, groups = rng.randint(1, 4000), 8 * rng.randint(1, 512), rng.randint(2, 256)
        k, act = 8 * rng.randint(1, 512), rng.choice((_lib.ACT_NONE, _lib.ACT_SWIGLU))
        a, b = plan(DW, m, n, k, groups, act), plan(DW, m, n, (k + 127) // 128 * 128, groups, act)
        if a[3] == b[3] == 1 and a != b:
            wrong.append((m, n, k, groups, act, a, b))
    assert not wrong, (len(wrong), wrong[:3])
    assert plan(DW, 50, 352, 64, 205)[:2] == (128, 128)  # not 410 tiles of 256 x 256, each three quarters empty


def test_few_rows_of_many_experts_with_short_reductions_take_tiles():
    """The kernel for few rows goes through w in tiles of 16 rows, 2.2 us each however short: 48 of them in a row per
    workgroup take 109 us where 128 x 128 tiles take 39."""
    assert plan(OUT, 49, 4024, 104, 156, _lib.ACT_SWIGLU) == (128, 128, 2, 1)
    assert plan(OUT, 127, 440, 72, 108, _lib.ACT_SWIGLU) == (128, 128, 2, 1)
    for long in ((48, 2048, 4096, 256, _lib.ACT_SWIGLU), (1, 4096, 4096), (6, 2048, 4096, 256), (6, 4352, 664, 86)):
        assert plan(OUT, *long)[:2] == (16, 16), long
