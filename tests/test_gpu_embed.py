"""The embedding lookup with its scale, and the table's gradient, against plain
restatements: the lookup exactly (one product, one rounding), the gradient's sums in
64 bits.  Bound: n terms in any order and the product with the scale are off by at
most (n + 1) 2^-24 of the sum of their magnitudes, then half a step of the type;
where they are added to what is there, one more rounding of the sum."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E = 2.0 ** -24


def normal(dev, seed, shape, dtype=BF16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(shape, generator=g, device=dev).to(dtype)


def make_ids(dev, m, vocab, seed, outside=0.2, hot=0.3, dtype=torch.int64):
    """Some of them outside the table on both sides, a share of them one word."""
    g = torch.Generator(device=dev).manual_seed(seed)
    ids = torch.randint(0, vocab, (m,), generator=g, device=dev)
    u = torch.rand(m, generator=g, device=dev)
    ids = torch.where(u < hot, vocab // 2, ids)
    far = torch.tensor([-1, vocab, -2 ** 31, 2 ** 31 - 1], device=dev)[torch.randint(0, 4, (m,), generator=g, device=dev)]
    return torch.where(u > 1 - outside, far, ids).to(dtype)


def plain_grad(d_out, ids, vocab):
    """Sums and sums of magnitudes [vocab, D] in 64 bits, and the terms of each row, on the host."""
    ids, d_out = ids.cpu().long(), d_out.cpu().double()
    keep = (ids >= 0) & (ids < vocab)
    s = torch.zeros(vocab, d_out.shape[1], dtype=F64).index_add_(0, ids[keep], d_out[keep])
    a = torch.zeros_like(s).index_add_(0, ids[keep], d_out[keep].abs())
    n = torch.zeros(vocab, dtype=F64).index_add_(0, ids[keep], torch.ones(int(keep.sum()), dtype=F64))
    return s, a, n[:, None]


SIZES = [(1, 1, 1), (1, 5, 8), (3, 7, 33), (31, 2, 64), (32, 3, 7), (33, 50, 72), (64, 1, 16), (65, 1, 9), (500, 40, 520), (1000, 1, 24),
         (1024, 3000, 4096), (2049, 129280, 8), (4097, 300, 100), (16384, 97, 40), (5000, 2000, 1001)]


@pytest.mark.parametrize("t", (BF16, F32))
@pytest.mark.parametrize("m,vocab,d", SIZES)
def test_lookup_and_gradient(dev, m, vocab, d, t):
    ids = make_ids(dev, m, vocab, m + d, dtype=torch.int32 if m % 2 else torch.int64)
    table = normal(dev, 1, (vocab, d), t)
    inside = ((ids >= 0) & (ids < vocab))[:, None]
    rows = table.float()[ids.long().clamp(0, vocab - 1)]
    for scale, o in ((1.0, None), (0.3, F32), (64.0, BF16)):
        out = ops.embed(ids, table, scale, o)
        want = torch.where(inside, rows * torch.tensor(scale, dtype=F32, device=dev), 0.0).to(o or t)
        assert out.dtype == (o or t) and torch.equal(out, want)
    d_out = normal(dev, 2, (m, d), t)
    s, a, n = plain_grad(d_out, ids, vocab)
    for scale, o in ((1.0, None), (-2.5, F32 if t == BF16 else BF16)):
        o_t = o or t
        got = ops.embed_grad(d_out, ids, vocab, scale, o)
        assert got.dtype == o_t and got.shape == (vocab, d)
        tol = (n + 1) * E * abs(scale) * a + torch.finfo(o_t).eps / 2 * abs(scale) * s.abs() + 1e-38
        assert ((got.cpu().double() - scale * s).abs() <= tol).all()
        assert (got.cpu()[(n == 0)[:, 0]] == 0).all()
        base = normal(dev, 3, (vocab, d), o_t)
        out = base.clone()
        assert ops.embed_grad(d_out, ids, vocab, scale, out=out) is out
        want = base.cpu().double() + scale * s
        tol = (n + 2) * E * (abs(scale) * a + base.cpu().double().abs()) + torch.finfo(o_t).eps / 2 * want.abs()
        assert ((out.cpu().double() - want).abs() <= tol).all()
        untouched = (n == 0)[:, 0].to(dev)
        assert torch.equal(out[untouched], base[untouched])


@pytest.mark.parametrize("m,vocab", ((16385, 1), (20000, 700), (65536, 5000), (65537, 5000), (70001, 1 << 20), (70000, (1 << 20) + 1), (66000, 1), (50001, 129280), (40000, 3000000), (17000, 1 << 20), (17001, (1 << 20) + 1)))
def test_many_tokens(dev, m, vocab):
    ids, d_out = make_ids(dev, m, vocab, m, hot=0.4), normal(dev, 2, (m, 16))
    s, a, n = plain_grad(d_out, ids, vocab)
    got = ops.embed_grad(d_out, ids, vocab, 1.0, F32)
    assert ((got.cpu().double() - s).abs() <= (n + 2) * E * a).all()
    assert torch.equal(ops.embed_grad(d_out, ids, vocab, 1.0, F32), got)


def test_all_tokens_one_word_and_none(dev):
    for m in (1, 32, 33, 64, 1000, 16384, 20000):
        d_out = normal(dev, m, (m, 136))
        ids = torch.full((m,), 3, device=dev)
        s, a, n = plain_grad(d_out, ids, 5)
        got = ops.embed_grad(d_out, ids, 5, 1.0, F32)
        assert ((got.cpu().double() - s).abs() <= (n + 1) * E * a).all() and (got[[0, 1, 2, 4]] == 0).all()
        for far in (-1, 5):
            assert (ops.embed_grad(d_out, torch.full((m,), far, device=dev), 5) == 0).all()
            assert (ops.embed(torch.full((m,), far, device=dev), normal(dev, 1, (5, 136))) == 0).all()


def test_terms_are_added_in_the_order_of_the_tokens(dev):
    """2^24, then ones, in fp32: what the first chunk of 32 adds after it is lost, what it adds before is not."""
    d_out = torch.ones(40, 8, device=dev)
    ids = torch.zeros(40, dtype=torch.int64, device=dev)
    for at in (0, 31):
        d = d_out.clone()
        d[at] = 2.0 ** 24
        first = 2.0 ** 24 if at == 0 else 2.0 ** 24 + 30  # 31 + 2^24 rounds to even
        first = float(torch.tensor(31.0 + 2.0 ** 24, dtype=F32)) if at == 31 else first
        assert (ops.embed_grad(d, ids, 2)[0] == first + 8).all()


def test_values_outside_the_table_count_for_nothing(dev):
    """Not-a-number in a padding token's gradient, and in table rows that no id names, stays there."""
    ids = torch.tensor([2, -1, 4, 9, 2], device=dev)
    d_out = normal(dev, 1, (5, 64))
    d_out[1] = float("nan")
    d_out[3] = float("inf")
    got = ops.embed_grad(d_out, ids, 9)
    assert torch.isfinite(got).all()
    table = normal(dev, 2, (9, 64))
    table[0] = float("nan")
    assert (ops.embed(ids, table, float("inf"))[[1, 3]] == 0).all()
    assert torch.isfinite(ops.embed(ids, table)).all()


def test_shapes_strides_and_kinds_of_ids(dev):
    table = normal(dev, 1, (50, 96))
    ids = make_ids(dev, 24, 50, 3, outside=0.0).reshape(2, 3, 4)
    want = table[ids]
    for i in (ids, ids.to(torch.int32), ids.to(torch.uint8), ids.transpose(0, 2).contiguous().transpose(0, 2)):
        assert torch.equal(ops.embed(i, table), want)
    wide = normal(dev, 4, (50, 200))
    for view in (wide[:, :96], wide[:, 1:98], wide[::2, 8:72], wide.t()[:96]):
        v = view if view.shape[0] == 50 else view
        i = ids % v.shape[0]
        assert torch.equal(ops.embed(i, v), v[i])
    d_out = normal(dev, 5, (2, 3, 4, 96))
    g = ops.embed_grad(d_out, ids, 50)
    assert torch.equal(ops.embed_grad(d_out.transpose(0, 1).contiguous().transpose(0, 1), ids, 50), g)
    assert torch.equal(ops.embed_grad(normal(dev, 6, (24, 200))[:, 3:99], ids.reshape(-1), 50),
                       ops.embed_grad(normal(dev, 6, (24, 200))[:, 3:99].contiguous(), ids.reshape(-1), 50))
    one = ops.embed_grad(torch.ones(1, 1, device=dev).expand(24, 96), ids.reshape(-1), 50)
    assert float(one.sum()) == 24 * 96
    base = torch.zeros(50, 208, dtype=F32, device=dev)
    ops.embed_grad(d_out, ids, 50, out=base[:, 5:101])  # rows that are apart, not 16-byte aligned
    assert torch.equal(base[:, 5:101].to(BF16), g) and (base[:, :5] == 0).all() and (base[:, 101:] == 0).all()
    far = torch.tensor([2 ** 32 + 3, -2 ** 40, 3, 2 ** 63 - 1], device=dev)  # beyond 32 bits: no row of the table
    assert torch.equal(ops.embed(far, table), torch.where((far == 3)[:, None], table[3], 0))
    assert torch.equal(ops.embed_grad(torch.ones(4, 96, device=dev), far, 50)[:, 0], (torch.arange(50, device=dev) == 3).float())
    assert ops.embed(ids[:0], table).shape == (0, 3, 4, 96)
    assert (ops.embed_grad(d_out[:0], ids[:0], 50) == 0).all()
    assert ops.embed(ids[0, 0, 0], table).shape == (96,)
    kept = base.clone()
    ops.embed_grad(d_out[:0], ids[:0], 50, out=base[:, 5:101])
    assert torch.equal(base, kept)


def test_table_beyond_32_bits(dev):
    vocab, d = 2 ** 20 + 5, 4104  # 8.6 GB
    table = torch.empty(vocab, d, dtype=BF16, device=dev)
    ids = torch.tensor([0, vocab - 1, vocab - 2, 7, vocab - 1, vocab], device=dev)
    for i in ids[:-1].tolist():
        table[i] = float(i % 97)
    out = ops.embed(ids, table, 2.0)
    assert torch.equal(out[:, 0].float().cpu(), torch.tensor([2.0 * (i % 97) for i in ids[:-1].tolist()] + [0.0]))
    table[vocab - 3:] = 1
    got = ops.embed_grad(torch.ones(6, d, dtype=BF16, device=dev), ids, vocab, out=table)
    assert (got[vocab - 1] == 3).all() and (got[vocab - 2] == 2).all() and (got[vocab - 3] == 1).all()
    del got, table
    got = ops.embed_grad(torch.ones(6, d, dtype=BF16, device=dev), ids, vocab)
    assert (got[vocab - 1] == 2).all() and (got[vocab - 2] == 1).all() and (got[vocab - 3] == 0).all() and float(got[8:16].abs().sum()) == 0


def test_deterministic_and_replayed(dev):
    for m in (3000, 17000):
        ids, d_out, table = make_ids(dev, m, 500, 1), normal(dev, 2, (m, 264)), normal(dev, 3, (500, 264))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.embed_grad(d_out, ids, 500)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out, g = ops.embed(ids, table, 0.5), ops.embed_grad(d_out, ids, 500, 0.5)
        torch.cuda.synchronize()
        for seed in range(3):
            ids.copy_(make_ids(dev, m, 500, 10 + seed))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.embed(ids, table, 0.5)) and torch.equal(g, ops.embed_grad(d_out, ids, 500, 0.5))


def test_refusals(dev):
    ids, table, d_out = torch.tensor([1, 2], device=dev), normal(dev, 1, (4, 16)), normal(dev, 2, (2, 16))
    for bad, exc in ((lambda: ops.embed(ids.float(), table), TypeError), (lambda: ops.embed(ids > 1, table), TypeError),
                     (lambda: ops.embed(ids, table.half()), TypeError), (lambda: ops.embed(ids, table[0]), ValueError),
                     (lambda: ops.embed(ids, table, out_dtype=torch.float16), TypeError), (lambda: ops.embed(ids.cpu(), table), RuntimeError),
                     (lambda: ops.embed_grad(d_out[:1], ids, 4), ValueError), (lambda: ops.embed_grad(d_out, ids, 0), ValueError),
                     (lambda: ops.embed_grad(d_out, ids, 4, out=table[:3]), ValueError), (lambda: ops.embed_grad(d_out, ids, 4, out=table.half()), TypeError),
                     (lambda: ops.embed_grad(d_out, ids, 4, out=normal(dev, 1, (16, 4)).t()), ValueError),
                     (lambda: ops.embed_grad(d_out, ids, 4, out_dtype=F32, out=table), TypeError),
                     (lambda: ops.embed_grad(d_out, ids, 4, out=table[:1].expand(4, 16)), ValueError)):
        with pytest.raises(exc):
            bad()


@pytest.mark.parametrize("d", (8, 15, 520, 4104))
def test_runs_of_every_length(dev, d):
    """Runs that begin and end anywhere in the chunks and in their parts: sums of small integers, which are exact."""
    for seed in range(8):
        g = torch.Generator().manual_seed(seed)
        lengths = torch.randint(1, (2, 5, 9, 17, 40, 70, 100, 12)[seed], (120,), generator=g)
        ids = torch.repeat_interleave(torch.randperm(500, generator=g)[:120], lengths)
        ids = ids[torch.randperm(len(ids), generator=g)].to(dev)
        if seed % 2:
            ids[::7] = -1
        d_out = torch.randint(-8, 9, (len(ids), d), generator=g).to(dev, BF16)
        want = torch.zeros(501, d, device=dev).index_add_(0, torch.where(ids < 0, 500, ids), d_out.float())[:500]
        assert torch.equal(ops.embed_grad(d_out, ids, 500, 2.0, F32), 2 * want)
        base = torch.full((500, d), 3.0, device=dev)
        assert torch.equal(ops.embed_grad(d_out, ids, 500, 1.0, out=base), want + 3)
