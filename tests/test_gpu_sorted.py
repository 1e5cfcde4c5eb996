"""Pairs sorted by expert, rows gathered to that order and combined back, and
the gradients, against plain restatements: the sort and the gather exactly, the
sums in 64 bits within a bound of fp32 summation (n terms in any order are off
by at most n 2^-24 of the sum of their magnitudes) plus half a step of the
output's type."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make_idx(dev, m, k, e, seed, drop=0.0, one=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    idx = torch.randint(0, e, (m, k), generator=g, device=dev)  # ids may repeat within a token
    if one:
        idx.fill_(e - 1)
    if drop:
        away = torch.rand((m, k), generator=g, device=dev) < drop
        idx = torch.where(away, torch.randint(0, 2, (m, k), generator=g, device=dev) * (e + 7) - 1, idx)  # -1 or e + 6
    return idx


def plain_order(idx, e):
    """offsets, pairs, rows on the host, by a stable sort of the valid pairs."""
    flat = idx.reshape(-1).cpu().tolist()
    pairs = sorted((q for q, v in enumerate(flat) if 0 <= v < e), key=lambda q: (flat[q], q))
    rows = [-1] * len(flat)
    for r, q in enumerate(pairs):
        rows[q] = r
    counts = [0] * e
    for q in pairs:
        counts[flat[q]] += 1
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    return offsets, pairs + [-1] * (len(flat) - len(pairs)), rows


SORTS = [
    (0, 6, 256, 0.0), (1, 1, 1, 0.0), (1, 6, 256, 0.0), (3, 16, 5, 0.3), (37, 6, 256, 0.5), (341, 6, 256, 0.0),
    (342, 6, 256, 0.1), (1000, 8, 1024, 0.2), (4096, 6, 256, 0.25), (2048, 1, 2, 0.0), (2049, 1, 1, 0.0),
    (700, 3, 64, 1.0), (50001, 6, 129, 0.1),
    (4096, 8, 64, 0.1), (4097, 8, 1000, 0.1),
]


@pytest.mark.parametrize("m,k,e,drop", SORTS)
def test_sort_is_the_stable_sort(dev, m, k, e, drop):
    idx = make_idx(dev, m, k, e, m + k, drop)
    order = ops.moe_sort(idx, e)
    offsets, pairs, rows = plain_order(idx, e)
    assert order.offsets.tolist() == offsets
    assert order.pairs.tolist() == pairs
    assert order.rows.reshape(-1).tolist() == rows


def test_sort_many_pairs_takes_larger_chunks(dev):
    """More than 256 x 1024 pairs: a workgroup places several thousand."""
    idx = make_idx(dev, 70001, 8, 200, 5, 0.05)
    order = ops.moe_sort(idx, 200)
    flat = idx.reshape(-1)
    key = torch.where((flat >= 0) & (flat < 200), flat, 200)
    perm = torch.sort(key, stable=True).indices
    n = int((key < 200).sum())
    assert torch.equal(order.pairs[:n].long(), perm[:n]) and bool((order.pairs[n:] == -1).all())
    assert torch.equal(order.offsets.long(), torch.searchsorted(key[perm], torch.arange(201, device=dev)))
    rows = torch.empty_like(flat).scatter_(0, perm, torch.arange(flat.numel(), device=dev))
    assert torch.equal(order.rows.reshape(-1).long(), torch.where(key < 200, rows, -1))


def test_sort_of_one_expert_and_int32_ids(dev):
    idx = make_idx(dev, 900, 4, 256, 1, one=True)
    a, b = ops.moe_sort(idx, 256), ops.moe_sort(idx.to(torch.int32), 256)
    assert a.offsets.tolist() == [0] * 256 + [3600] and a.pairs.tolist() == list(range(3600))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_ids_of_any_size_are_no_experts(dev):
    idx = torch.tensor([[1 << 40, 0], [-(1 << 40), (1 << 32) + 1], [1, -1]], device=dev)
    order = ops.moe_sort(idx, 2)
    assert order.offsets.tolist() == [0, 1, 2] and order.pairs.tolist() == [1, 4, -1, -1, -1, -1]
    assert order.rows.tolist() == [[-1, 0], [-1, -1], [1, -1]]


def test_a_row_number_that_is_none_counts_as_dropped(dev):
    order = ops.moe_sort(torch.tensor([[0, 1], [1, 0]], device=dev), 2)
    wild = order._replace(rows=torch.tensor([[0, 1 << 30], [-5, 1]], dtype=torch.int32, device=dev))
    rows, w = torch.randn(4, 64, device=dev), torch.ones(2, 2, device=dev)
    assert torch.equal(ops.moe_combine(rows, wild, w), rows[:2])
    assert ops.moe_combine_grad(rows[:2], rows, wild, w)[1][0, 1] == 0


ROWS = [(1, 6, 256, 4096, 0.0), (5, 6, 256, 4096, 0.4), (37, 3, 9, 72, 0.2), (33, 16, 40, 1001, 0.5), (200, 9, 64, 520, 0.1),
        (3, 2, 4, 1, 0.0), (700, 6, 64, 2048, 1.0), (2, 1, 3, 16392, 0.0)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k,e,d,drop", ROWS)
def test_gather(dev, m, k, e, d, drop, dtype):
    idx = make_idx(dev, m, k, e, d, drop)
    order = ops.moe_sort(idx, e)
    x = torch.randn(m, d, device=dev).to(dtype)
    got = ops.moe_gather(x, order)
    pairs = order.pairs.long()
    want = torch.where((pairs >= 0)[:, None], x[pairs.clamp(min=0) // k], 0)
    assert torch.equal(got, want)


def test_gather_takes_strided_rows_and_leaves_the_rest(dev):
    base = torch.randn(40, 3, 520, device=dev).to(BF16)
    idx = make_idx(dev, 40, 4, 7, 3, 0.3)
    order = ops.moe_sort(idx, 7)
    for x in (base[:, 1], base[:, 1, 1:], base[:, 2, ::2], base[::2].expand(20, 3, 520).repeat(2, 1, 1)[:, 0],
              base[0, 0].expand(40, 520)):
        assert torch.equal(ops.moe_gather(x, order), ops.moe_gather(x.clone(memory_format=torch.contiguous_format), order))


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k,e,d,drop", ROWS)
def test_combine(dev, m, k, e, d, drop, dtype, out_dtype):
    idx = make_idx(dev, m, k, e, d + 1, drop)
    order = ops.moe_sort(idx, e)
    rows = torch.randn(m * k, d, device=dev).to(dtype)
    n = int(order.offsets[-1])
    rows[n:] = float("nan")  # behind the last row nothing is read
    w = torch.randn(m, k, device=dev)
    w[order.rows < 0] = float("nan")  # nor is a dropped pair's weight
    res = torch.randn(m, d, device=dev).to(out_dtype)
    at, live = order.rows.clamp(min=0).long(), (order.rows >= 0)[:, :, None]
    for weights, residual in ((w, res), (w, None), (None, None)):
        got = ops.moe_combine(rows, order, weights, residual, out_dtype=out_dtype)
        terms = rows[at].double() * (1.0 if weights is None else weights.double()[:, :, None])
        terms = torch.where(live, terms, 0.0)
        if residual is not None:
            terms = torch.cat((terms, residual.double()[:, None]), dim=1)
        want, size = terms.sum(dim=1), terms.abs().sum(dim=1)
        bound = (k + 1) * 2.0 ** -24 * size
        bound = bound + half_step(out_dtype) * (want.abs() + bound)
        assert got.dtype == out_dtype and bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k,e,d,drop", ROWS)
def test_combine_grad(dev, m, k, e, d, drop, dtype, out_dtype):
    idx = make_idx(dev, m, k, e, d + 2, drop)
    order = ops.moe_sort(idx, e)
    n = int(order.offsets[-1])
    rows = torch.randn(m * k, d, device=dev).to(dtype)
    rows[n:] = float("nan")
    w = torch.randn(m, k, device=dev)
    g = torch.randn(m, d, device=dev).to(out_dtype)
    for weights in (w, None):
        d_rows, d_w = ops.moe_combine_grad(g, rows, order, weights)
        at, live = order.rows.clamp(min=0).long(), order.rows >= 0
        want = g.double()[:, None].expand(m, k, d) * (1.0 if weights is None else weights.double()[:, :, None])
        want_rows = torch.zeros(m * k, d, dtype=torch.float64, device=dev)
        want_rows[at[live]] = want[live]
        # one fp32 product, one rounding
        assert bool(((d_rows.double() - want_rows).abs() <=
                     want_rows.abs() * (2.0 ** -24 + half_step(dtype) * (1 + 2.0 ** -24))).all())
        dots = torch.where(live[:, :, None], rows[at].double() * g.double()[:, None], 0.0)
        assert bool(((d_w.double() - dots.sum(dim=2)).abs() <= d * 2.0 ** -24 * dots.abs().sum(dim=2)).all())
    only_w = ops.moe_combine_grad(g, rows, order, w, need_rows=False)
    only_rows = ops.moe_combine_grad(g, rows, order, w, need_w=False)
    both = ops.moe_combine_grad(g, rows, order, w)
    assert only_w[0] is None and torch.equal(only_w[1], both[1])
    assert only_rows[1] is None and torch.equal(only_rows[0], both[0])


def test_gradient_against_differences(dev):
    """fp32 rows: the function is linear in the rows and in the weights, so a step of
    size 1 gives the gradient's product with the step up to the sums' rounding."""
    m, k, e, d = 9, 4, 5, 64
    order = ops.moe_sort(make_idx(dev, m, k, e, 2, 0.2), e)
    rows, w, g = torch.randn(m * k, d, device=dev), torch.rand(m, k, device=dev), torch.randn(m, d, device=dev)
    d_rows, d_w = ops.moe_combine_grad(g, rows, order, w)
    base = (ops.moe_combine(rows, order, w).double() * g.double()).sum()
    step = torch.randn_like(rows)
    moved = (ops.moe_combine(rows + step, order, w).double() * g.double()).sum()
    tol = 2.0 ** -24 * 4 * (k + 2) * float((rows.abs() + step.abs()).sum() * g.abs().max() * w.max())
    assert abs(float(moved - base - (d_rows.double() * step.double()).sum())) <= tol
    step_w = torch.rand_like(w)
    moved = (ops.moe_combine(rows, order, w + step_w).double() * g.double()).sum()
    assert abs(float(moved - base - (d_w.double() * step_w.double()).sum())) <= 2 * d * tol


def test_gather_then_its_gradient(dev):
    """The gradient of the gather is the combine without weights."""
    m, k, e, d = 50, 6, 16, 512
    order = ops.moe_sort(make_idx(dev, m, k, e, 3, 0.3), e)
    x = torch.randn(m, d, device=dev)
    g = torch.randn(m * k, d, device=dev)
    lhs = (ops.moe_gather(x, order).double() * g.double()).sum()
    rhs = (x.double() * ops.moe_combine(g, order).double()).sum()
    assert abs(float(lhs - rhs)) <= 2.0 ** -24 * (k + 1) * float((g.abs().sum() * x.abs().max()))


def test_infinite_rows_and_zero_weights_follow_the_formula(dev):
    idx = torch.tensor([[0, 1], [1, -1]], device=dev)
    order = ops.moe_sort(idx, 2)
    rows = torch.ones(4, 8, device=dev)
    rows[0, 0] = float("inf")
    w = torch.tensor([[0.0, 1.0], [2.0, 3.0]], device=dev)
    out = ops.moe_combine(rows, order, w)
    assert bool(out[0, 0].isnan()) and out[0, 1:].tolist() == [1.0] * 7 and out[1].tolist() == [2.0] * 8


def test_many_rows_pass_32_bit_offsets(dev):
    """Rows beyond 2^31 elements (and 2^32 bytes): the last ones are the right ones."""
    m, k, d = 70000, 8, 4096
    idx = torch.arange(k, device=dev).expand(m, k).contiguous()
    order = ops.moe_sort(idx, k)
    x = torch.randn(m, 1, device=dev).to(BF16).expand(m, d).contiguous()
    rows = ops.moe_gather(x, order)
    assert rows.numel() > 1 << 31
    assert torch.equal(rows.reshape(k, m, d)[-1, -100:], x[-100:]) and torch.equal(rows[:100], x[:100])
    out = ops.moe_combine(rows, order)
    assert torch.equal(out[-100:], x[-100:] * 8) and torch.equal(out[:100], x[:100] * 8)
    d_rows, d_w = ops.moe_combine_grad(out, rows, order, need_w=True)
    assert torch.equal(d_rows.reshape(k, m, d)[-1, -100:], out[-100:])
    assert bool((d_w > 0).all())


def test_replayed_graph_and_side_stream(dev):
    m, k, e, d = 600, 6, 64, 1024
    idx, x, w = make_idx(dev, m, k, e, 4, 0.1), torch.randn(m, d, device=dev).to(BF16), torch.rand(m, k, device=dev)

    def step():
        order = ops.moe_sort(idx, e)
        rows = ops.moe_gather(x, order)
        out = ops.moe_combine(rows, order, w)
        return (*order, rows, out, *ops.moe_combine_grad(out, rows, order, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        idx.copy_(make_idx(dev, m, k, e, 50 + seed, 0.1 * seed))
        x.copy_(torch.randn(m, d, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_refusals(dev):
    idx = make_idx(dev, 4, 2, 8, 0)
    order = ops.moe_sort(idx, 8)
    x = torch.randn(4, 64, device=dev)
    rows = ops.moe_gather(x, order)
    with pytest.raises(TypeError, match="integers"):
        ops.moe_sort(idx.float(), 8)
    with pytest.raises(ValueError, match="top_k"):
        ops.moe_sort(idx.reshape(-1), 8)
    for n in (0, -1, 1025):
        with pytest.raises(ops._lib.HsmoeError, match="experts"):
            ops.moe_sort(idx, n)
    with pytest.raises(ops._lib.HsmoeError, match="top_k"):
        ops.moe_sort(torch.zeros(2, 17, dtype=torch.int64, device=dev), 8)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.moe_gather(x.half(), order)
    with pytest.raises(ValueError, match="tokens"):
        ops.moe_gather(x[:3], order)
    with pytest.raises(TypeError, match="int32"):
        ops.moe_gather(x, order._replace(rows=order.rows.long()))
    with pytest.raises(ValueError, match="expert order"):
        ops.moe_gather(x, order._replace(pairs=order.pairs[:-1]))
    with pytest.raises(ValueError, match="pairs"):
        ops.moe_combine(rows[:-1], order)
    with pytest.raises(ValueError, match="weights"):
        ops.moe_combine(rows, order, torch.ones(4, 3, device=dev))
    with pytest.raises(ValueError, match="residual"):
        ops.moe_combine(rows, order, None, x.to(BF16), out_dtype=F32)
    with pytest.raises(ValueError, match="pairs"):
        ops.moe_combine_grad(x[:, :32], rows, order)
    with pytest.raises(ops._lib.HsmoeError, match="CPU|cpu"):
        ops.moe_gather(x.cpu(), order)
