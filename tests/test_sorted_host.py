"""Argument checks of the sort, gather and combine entry points, before anything is launched (no GPU needed)."""
from home_seek_amd import _lib


def test_sort_rejects_bad_arguments():
    L = _lib.lib()
    assert L.hsmoe_moe_sort_workspace_size(341, 6, 256) == 0
    need = L.hsmoe_moe_sort_workspace_size(1 << 16, 6, 256)
    assert need > 0
    assert L.hsmoe_moe_sort(4096, 1 << 16, 6, 256, 4096, 4096, 4096, None, 0, None) == -4
    assert L.hsmoe_moe_sort(4096, 1 << 16, 6, 256, 4096, 4096, 4096, 4096, need - 1, None) == -4
    assert L.hsmoe_moe_sort(None, 4, 6, 256, 4096, 4096, 4096, None, 0, None) == -1
    assert L.hsmoe_moe_sort(4096, 4, 6, 1025, 4096, 4096, 4096, None, 0, None) == -2
    assert L.hsmoe_moe_sort(4096, 4, 0, 256, 4096, 4096, 4096, None, 0, None) == -1
    assert L.hsmoe_moe_sort(4096, 4, 17, 256, 4096, 4096, 4096, None, 0, None) == -2
    assert L.hsmoe_moe_sort(4096, 1 << 24, 2, 256, 4096, 4096, 4096, 4096, 1 << 30, None) == -2
    assert L.hsmoe_moe_sort(4100, 4, 6, 256, 4096, 4096, 4096, None, 0, None) == -2  # ids not 8-byte aligned


def test_rows_entry_points_reject_bad_arguments():
    L = _lib.lib()
    gather = lambda *a: L.hsmoe_moe_gather(*a, None)
    assert gather(4096, 64, 4, 64, 2, 4096, 8, 4096, 2, 4096) == -1       # row kind
    assert gather(4096, 63, 4, 64, 1, 4096, 8, 4096, 2, 4096) == -1       # rows overlap
    assert gather(4097, 64, 4, 64, 1, 4096, 8, 4096, 2, 4096) == -2       # misaligned
    assert gather(None, 64, 4, 64, 1, 4096, 8, 4096, 2, 4096) == -1
    assert gather(None, 64, 0, 64, 1, None, 8, None, 2, None) == 0        # no tokens
    combine = lambda *a: L.hsmoe_moe_combine(*a, None)
    assert combine(4096, 1, 8, 4, 64, 4096, None, 2, None, 7, 4096) == -1
    assert combine(None, 1, 8, 4, 64, 4096, None, 2, None, 1, 4096) == -1
    assert combine(4096, 1, 8, 4, (1 << 23) + 1, 4096, None, 2, None, 1, 4096) == -2
    assert combine(4098, 0, 8, 4, 64, 4096, None, 2, None, 1, 4096) == -2
    assert combine(None, 1, 0, 0, 64, None, None, 2, None, 1, None) == 0
    grad = lambda *a: L.hsmoe_moe_combine_grad(*a, None)
    assert grad(4096, 1, None, 1, 4, 64, 4096, 8, 4096, None, 2, None, 4096) == -1  # d_w needs the rows
    assert grad(4096, 1, None, 1, 4, 64, 4096, 8, 4096, None, 2, None, None) == 0   # nothing asked for
    assert grad(4096, 3, 4096, 1, 4, 64, 4096, 8, 4096, None, 2, 4096, 4096) == -1
