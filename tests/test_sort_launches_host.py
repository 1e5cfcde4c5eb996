"""Where the sort takes a launch of its own for counting (no GPU needed)."""
import pytest

from home_seek_amd import _lib


@pytest.mark.parametrize("m,top_k,experts,counts", [(1, 6, 256, False), (2048, 6, 256, False), (2049, 6, 256, True),
                                                    (4096, 6, 256, True), (4096, 8, 64, True)])
def test_only_few_pairs_are_counted_by_every_workgroup(m, top_k, experts, counts):
    """24576 pairs counted by each of 24 workgroups take 13.7 us, a launch that counts and one that places 9."""
    nbytes = _lib.lib().hsmoe_moe_sort_workspace_size(m, top_k, experts)
    chunks = -(-m * top_k // 1024)
    assert nbytes == (4 * experts * chunks if counts else 0)
