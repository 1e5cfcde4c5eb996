"""The sort on both sides of the size from which counting is a launch of its own: the stable sort, eager and replayed,
two captured ones at once."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

SIZES = [(2047, 6, 256), (2048, 6, 256), (2049, 6, 256), (12288, 1, 1024), (12289, 1, 1024), (1600, 8, 7)]


def ids(dev, m, k, e, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    u = torch.rand((m, k), generator=g, device=dev)
    return torch.where(u < 0.2, -1, (u * u * e).long())  # skewed, a fifth dropped


def check(order, idx, e):
    key = torch.where(idx < 0, e, idx).reshape(-1)
    perm = torch.sort(key, stable=True).indices
    n = int((key < e).sum())
    assert torch.equal(order.pairs[:n].long(), perm[:n]) and bool((order.pairs[n:] == -1).all())
    assert torch.equal(order.offsets.long(), torch.searchsorted(key[perm], torch.arange(e + 1, device=idx.device)))
    rows = torch.empty_like(key).scatter_(0, perm, torch.arange(key.numel(), device=idx.device))
    assert torch.equal(order.rows.reshape(-1).long(), torch.where(key < e, rows, -1))


@pytest.mark.parametrize("m,k,e", SIZES)
def test_both_ways_of_counting(dev, m, k, e):
    idx = ids(dev, m, k, e, m)
    check(ops.moe_sort(idx, e), idx, e)


def test_two_captured_sorts_that_count_at_once(dev):
    m, k, e = 4096, 6, 256
    runs = []
    for seed in (1, 2):
        idx, stream = ids(dev, m, k, e, seed), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.moe_sort(idx, e)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                orders = [ops.moe_sort(idx, e) for _ in range(4)]
        runs.append((stream, graph, orders, idx))
    torch.cuda.synchronize()
    for seed in range(4):
        for i, (stream, graph, _, idx) in enumerate(runs):
            with torch.cuda.stream(stream):
                idx.copy_(ids(dev, m, k, e, 10 * seed + i))
                graph.replay()
        torch.cuda.synchronize()
        for _, _, orders, idx in runs:
            for order in orders:
                check(order, idx, e)
