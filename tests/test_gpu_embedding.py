"""embedding_lookup and embedding_grad against plain sums in 64 bits.

Tolerances.  A lookup is one 32-bit product, rounded to the type: off by at
most 2^-24 and half a step of the type, relative; float16 has an absolute half
step of 2^-25 below its smallest normal number.  A gradient adds n rows, the
scale and what was there before in 32 bits: each of the at most n + 2
operations is off by 2^-24 of a partial result, which is no larger than the
sum of the absolute values; then the rounding to the type."""
import pytest
import torch

import moderngpu_amd as m

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES}


def near(got, want, slack, dtype):
    """|got - want| <= slack, plus the rounding of a value that is itself up
    to slack off."""
    step = HALF_STEP[dtype] * (want.abs() + slack) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -149)
    off = (got.double().cpu() - want).abs()
    assert got.dtype == dtype
    assert bool((off <= slack + step).all()), (off - slack - step).max().item()


def make_ids(kind, count, rows, gen):
    if kind == "same":
        return torch.full((count,), rows // 2, dtype=torch.int32)
    if kind == "distinct":
        return torch.arange(count, dtype=torch.int32) % rows
    if kind == "padding":
        return torch.where(torch.arange(count) % 2 == 0, -1, rows).to(torch.int32)
    if kind == "mixed":            # a frequent token, padding, extremes of int
        ids = torch.randint(0, rows, (count,), generator=gen)
        pick = torch.randint(0, 8, (count,), generator=gen)
        ids[pick < 3] = rows - 1
        ids[pick == 3] = -1
        ids[pick == 4] = 2 ** 31 - 1
        ids[pick == 5] = -2 ** 31
        return ids.to(torch.int32)
    return torch.randint(0, rows, (count,), generator=gen).to(torch.int32)


def lookup_want(table, ids, scale):
    ids = ids.long()
    ok = (ids >= 0) & (ids < table.shape[0])
    if not table.shape[0]:
        return torch.zeros(ids.numel(), table.shape[1], dtype=torch.float64)
    return torch.where(ok[:, None], table.double()[ids.clamp(0, table.shape[0] - 1)] * scale, 0.0)


def grad_want(grad, ids, rows):
    """Sums and sums of absolute values per row, and the rows' counts."""
    ids = ids.long()
    ok = (ids >= 0) & (ids < rows)
    g = grad.double()[ok]
    at = ids[ok]
    return (torch.zeros(rows, grad.shape[1], dtype=torch.float64).index_add_(0, at, g),
            torch.zeros(rows, grad.shape[1], dtype=torch.float64).index_add_(0, at, g.abs()),
            torch.bincount(at, minlength=rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,rows,dim", [(1, 1, 1), (3, 7, 8), (17, 5, 3), (64, 1000, 129), (257, 33, 515),
                                            (1, 100, 4096), (5, 64, 2055), (1000, 77, 64), (0, 5, 8), (4, 3, 0)])
def test_lookup(dev, dtype, count, rows, dim):
    gen = torch.Generator().manual_seed(count * 31 + dim)
    table = torch.randn(rows, dim, generator=gen).to(dtype)
    ids = make_ids("mixed", count, rows, gen)
    out = m.embedding_lookup(table.to(dev), ids.to(dev), scale=1.75)
    assert out.shape == (count, dim)
    want = lookup_want(table, ids, 1.75)
    near(out, want, want.abs() * 2.0 ** -24, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_strides_and_alignment(dev, dtype):
    """Rows that begin off every vector boundary, a repeated row, an output
    inside a wider tensor whose other values stay."""
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(50, 301, generator=gen).to(dtype)
    ids = make_ids("random", 90, 50, gen)
    for table in (wide[:, 1:], wide[:, 3:200], wide[::2, 5:6], wide[:1].expand(50, 301)):
        on_dev = wide.to(dev)
        view = torch.as_strided(on_dev, table.shape, table.stride(), table.storage_offset())
        outer = torch.full((90, table.shape[1] + 7), 5.0, dtype=dtype, device=dev)
        out = outer[:, 3:3 + table.shape[1]]
        assert m.embedding_lookup(view, ids.to(dev), scale=0.5, out=out) is out
        want = lookup_want(table, ids, 0.5)
        near(out, want, want.abs() * 2.0 ** -24, dtype)
        assert bool((outer[:, :3] == 5).all()) and bool((outer[:, 3 + table.shape[1]:] == 5).all())


def test_lookup_shapes_nan_and_empty_table(dev):
    table = torch.tensor([[1.0, float("inf")], [float("nan"), -2.0]], device=dev)
    ids = torch.tensor([[0, 1, -1], [2, 1, 0]], dtype=torch.int32, device=dev)
    out = m.embedding_lookup(table, ids, scale=2.0)
    assert out.shape == (2, 3, 2)
    want = torch.tensor([[[2, float("inf")], [float("nan"), -4], [0, 0]], [[0, 0], [float("nan"), -4], [2, float("inf")]]])
    assert torch.equal(torch.nan_to_num(out.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))
    none = m.embedding_lookup(torch.empty(0, 5, device=dev), ids)
    assert none.shape == (2, 3, 5) and not none.any()


GRAD_SIZES = [(1, 1, 1), (3, 7, 8), (17, 5, 3), (64, 100, 129), (257, 33, 515), (1, 100, 4096), (5, 64, 2055),
              (1000, 77, 64), (1025, 300, 17), (0, 5, 8), (6, 3, 0), (5000, 2000, 40), (9001, 50, 72), (20000, 4099, 8)]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("types", [(t, t) for t in TYPES] + [(torch.float16, torch.float32), (torch.bfloat16, torch.float32)],
                         ids=lambda t: "%s-%s" % t)
@pytest.mark.parametrize("count,rows,dim", GRAD_SIZES)
def test_grad(dev, count, rows, dim, types, accumulate):
    gtype, otype = types
    gen = torch.Generator().manual_seed(count + dim)
    for kind in ("mixed", "same", "distinct", "padding"):
        ids = make_ids(kind, count, rows, gen)
        grad = torch.randn(count, dim, generator=gen).to(gtype)
        before = torch.randn(rows, dim, generator=gen).to(otype)
        out = before.to(dev)
        m.embedding_grad(grad.to(dev), ids.to(dev), num_rows=rows, scale=0.75, out=out, accumulate=accumulate)
        total, size, n = grad_want(grad, ids, rows)
        base = before.double() if accumulate else torch.zeros(rows, dim, dtype=torch.float64)
        want = base + 0.75 * total
        slack = (n[:, None] + 2) * 2.0 ** -24 * (base.abs() + 0.75 * size)
        if accumulate:
            untouched = n == 0
            assert torch.equal(out.cpu()[untouched], before[untouched])
        near(out, want, slack, otype)


@pytest.mark.parametrize("accumulate", [False, True])
def test_grad_strides(dev, accumulate):
    """Gradient rows off every boundary, one row for all tokens (a broadcast
    gradient), and a gradient buffer inside a wider tensor."""
    gen = torch.Generator().manual_seed(5)
    for dtype in TYPES:
        wide = torch.randn(700, 133, generator=gen).to(dtype)
        ids = make_ids("mixed", 700, 90, gen)
        on_dev = wide.to(dev)
        for view in (lambda t: t[:, 1:], lambda t: t[:, 5:70], lambda t: t[:1, 2:101].expand(700, 99)):
            grad = view(wide)
            dim = grad.shape[1]
            outer = torch.full((90, dim + 5), 2.0, dtype=dtype, device=dev)
            out = outer[:, 2:2 + dim]
            m.embedding_grad(view(on_dev), ids.to(dev), out=out, accumulate=accumulate)
            total, size, n = grad_want(grad, ids, 90)
            base = 2.0 if accumulate else 0.0
            near(out, total + base, (n[:, None] + 2) * 2.0 ** -24 * (size + base), dtype)
            assert bool((outer[:, :2] == 2).all()) and bool((outer[:, 2 + dim:] == 2).all())


def test_grad_nan_stays_in_its_row(dev):
    grad = torch.ones(300, 16, device=dev)
    ids = (torch.arange(300, device=dev) % 30).to(torch.int32)
    grad[7, 3] = float("nan")
    grad[8, 4] = float("inf")
    ids[9] = -1
    grad[9] = float("nan")                       # padding: never in any sum
    out = m.embedding_grad(grad, ids, num_rows=40)
    want = torch.zeros(40, 16, dtype=torch.float64)
    want[:30] = 10
    want[9] = 9
    want[7, 3], want[8, 4] = float("nan"), float("inf")
    assert torch.equal(torch.nan_to_num(out.double().cpu(), nan=-5.0), torch.nan_to_num(want, nan=-5.0))


def test_grad_is_the_same_every_time(dev):
    gen = torch.Generator().manual_seed(8)
    for count, dim in ((900, 70), (30000, 24)):
        grad = torch.randn(count, dim, generator=gen).to(dev)
        ids = make_ids("mixed", count, 500, gen).to(dev)
        first = m.embedding_grad(grad, ids, num_rows=500)
        for _ in range(3):
            assert torch.equal(m.embedding_grad(grad, ids, num_rows=500), first)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("count,rows,dim", [(2047, 40, 300), (2048, 7, 520), (2049, 7, 520), (2049, 9000, 130),
                                            (100, 20000, 1100), (2048, 4100, 2063)])
def test_grad_of_few_tokens_and_of_more(dev, count, rows, dim, accumulate):
    """Around 2048 tokens, where one launch gives way to three; several blocks
    of columns, side by side and one after the other; several rows of many
    tokens next to each other; strides and padding for both."""
    gen = torch.Generator().manual_seed(count + rows)
    for gtype, otype in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)):
        ids = make_ids("mixed", count, rows, gen)
        hot = torch.rand(count, generator=gen) < 0.5
        ids[hot] = torch.randint(0, min(rows, 5), (int(hot.sum()),), generator=gen).to(torch.int32)
        wide = torch.randn(count, dim + 3, generator=gen).to(gtype)
        outer = torch.full((rows, dim + 5), 2.0, dtype=otype, device=dev)
        out = outer[:, 1:1 + dim]
        m.embedding_grad(wide.to(dev)[:, 3:], ids.to(dev), out=out, accumulate=accumulate)
        total, size, n = grad_want(wide[:, 3:], ids, rows)
        base = 2.0 if accumulate else 0.0
        near(out, total + base, (n[:, None] + 2) * 2.0 ** -24 * (size + base), otype)
        assert bool((outer[:, :1] == 2).all()) and bool((outer[:, 1 + dim:] == 2).all())


@pytest.mark.parametrize("count", [300, 2100])
def test_grad_in_a_graph(dev, count):
    gen = torch.Generator().manual_seed(count)
    grad, ids = torch.randn(count, 70, generator=gen).to(dev), make_ids("mixed", count, 90, gen).to(dev)
    out = torch.zeros(90, 70, device=dev)
    m.embedding_grad(grad, ids, out=out)                         # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.embedding_grad(grad, ids, out=out)
        m.embedding_grad(grad, ids, out=out, accumulate=True)
    for seed in (1, 2, 3):
        new = make_ids("mixed", count, 90, torch.Generator().manual_seed(seed)).to(dev)
        ids.copy_(new)
        grad.mul_(-0.5)
        graph.replay()
        want = m.embedding_grad(grad, ids, num_rows=90)
        m.embedding_grad(grad, ids, out=want, accumulate=True)
        assert torch.equal(out, want)


def test_gradient_against_differences(dev):
    """Moving one table value by h moves the weighted sum of the lookups by h
    times its gradient (the map is linear: exact up to the 64-bit reference's
    rounding and the 32-bit sums)."""
    gen = torch.Generator().manual_seed(9)
    table = torch.randn(20, 12, generator=gen, dtype=torch.float64)
    ids = make_ids("mixed", 80, 20, gen)
    weight = torch.randn(80, 12, generator=gen)
    grad = m.embedding_grad(weight.to(dev), ids.to(dev), num_rows=20, scale=1.5).double().cpu()
    _, size, n = grad_want(weight, ids, 20)
    f = lambda t: (lookup_want(t, ids, 1.5) * weight.double()).sum()  # noqa: E731
    for v, c in ((0, 0), (19, 3), (7, 11), (12, 5)):
        step = torch.zeros_like(table)
        step[v, c] = 0.5
        difference = f(table + step) - f(table - step)
        slack = (n[v] + 2) * 2.0 ** -23 * 1.5 * size[v, c] + 1e-10
        assert abs(difference - grad[v, c]) <= slack


def test_offsets_past_32_bits(dev):
    """A table, and a gradient, of more than 2^31 values."""
    rows, dim = (1 << 20) + 3, 2056
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device=dev)
    table[-1] = 3.0
    table[rows // 2] = 2.0
    ids = torch.tensor([rows - 1, 0, rows // 2, rows - 1], dtype=torch.int32, device=dev)
    out = m.embedding_lookup(table, ids)
    assert out.float().cpu().unique(dim=1).squeeze(1).tolist() == [3, 0, 2, 3]
    m.embedding_grad(out, ids, out=table, accumulate=True)
    assert bool((table[-1] == 9).all()) and bool((table[rows // 2] == 4).all()) and not bool(table[1:rows // 2].any())
    m.embedding_grad(out, ids, out=table)
    assert bool((table[-1] == 6).all()) and bool((table[rows // 2] == 2).all())
    assert not bool(table[rows // 2 + 1:rows - 1].any()) and not bool(table[:rows // 2].any())


def test_refusals(dev):
    t = torch.zeros(4, 6, device=dev)
    ids = torch.zeros(4, dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        m.embedding_lookup(t.double(), ids)
    with pytest.raises(TypeError):
        m.embedding_lookup(t.t(), ids)
    with pytest.raises(TypeError):
        m.embedding_lookup(t, ids.long())
    with pytest.raises(ValueError):
        m.embedding_lookup(t, ids.cpu().to(dev), out=torch.zeros(4, 5, device=dev))
    with pytest.raises(m.MgpuError):
        m.embedding_lookup(t, ids, out=t)
    with pytest.raises(ValueError):
        m.embedding_grad(t, ids)
    with pytest.raises(ValueError):
        m.embedding_grad(t, ids, num_rows=4, accumulate=True)
    with pytest.raises(ValueError):
        m.embedding_grad(t, ids[:3], num_rows=4)
    with pytest.raises(TypeError):
        m.embedding_grad(t, ids, out=torch.zeros(4, 6, dtype=torch.float16, device=dev))
    with pytest.raises(TypeError):
        m.embedding_grad(t, ids, out=torch.zeros(1, 6, device=dev).expand(4, 6))
    with pytest.raises(m.MgpuError):
        m.embedding_grad(t, ids, out=t)


# ---- sizes at which other kernels, or more launches, take over ----------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,dim", [(16501, 1021), (17003, 2051), (8195, 4099), (140001, 33)])
def test_lookup_of_many_tokens(dev, dtype, count, dim):
    """Four tokens a thread, results below 64 MB and streamed ones, rows that
    begin off every boundary."""
    gen = torch.Generator().manual_seed(count)
    table = torch.randn(777, dim + 1, generator=gen).to(dtype)
    ids = make_ids("mixed", count, 777, gen)
    ids[::3] = torch.randint(0, 777, ids[::3].shape, generator=gen).to(torch.int32)
    out = torch.full((count, dim + 3), 5.0, dtype=dtype, device=dev)
    m.embedding_lookup(table.to(dev)[:, 1:], ids.to(dev), scale=1.75, out=out[:, 1:1 + dim])
    near(out[:, 1:1 + dim], *(lambda w: (w, w.abs() * 2.0 ** -24))(lookup_want(table[:, 1:], ids, 1.75)), dtype)
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 1 + dim:] == 5).all())


def test_lookup_in_several_launches(dev):
    """Tokens past one launch of 2^18 CTAs, by their number and by the length
    of their rows.  Every value is compared, on the device (the products are
    exact)."""
    for count, dim, rows in ((2 ** 25 + 77, 3, 1000), (2051, 2 ** 20 + 8, 5)):
        gen = torch.Generator(device=dev).manual_seed(dim)
        table = torch.randn(rows, dim, generator=gen, device=dev).to(torch.bfloat16)
        ids = torch.randint(-1, rows, (count,), generator=gen, device=dev, dtype=torch.int32)
        out = m.embedding_lookup(table, ids, scale=2.0)
        want = torch.cat([table * 2, torch.zeros(1, dim, dtype=table.dtype, device=dev)])
        for begin in range(0, count, 2 ** 22 if dim == 3 else 512):
            part = ids[begin:begin + (2 ** 22 if dim == 3 else 512)].long()
            assert torch.equal(out[begin:begin + part.numel()], want[part])


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("types", [(t, t) for t in TYPES] + [(torch.bfloat16, torch.float32)], ids=lambda t: "%s-%s" % t)
@pytest.mark.parametrize("count,rows,dim", [(2501, 16411, 2051), (1501, 16411, 2051), (20011, 9001, 130)])
def test_grad_of_large_tables(dev, count, rows, dim, types, accumulate):
    """Results of 64 MB and more, from few tokens and from many; more tokens
    than the sort keeps between its passes.  Rows of many tokens among them."""
    gtype, otype = types
    gen = torch.Generator().manual_seed(count)
    ids = make_ids("mixed", count, rows, gen)
    ids[::5] = torch.randint(0, rows, ids[::5].shape, generator=gen).to(torch.int32)
    ids[1::5] = 7
    grad = torch.randn(count, dim, generator=gen).to(gtype)
    out = torch.full((rows, dim), 2.0, dtype=otype, device=dev)
    m.embedding_grad(grad.to(dev), ids.to(dev), scale=0.75, out=out, accumulate=accumulate)
    # what occurs, in 64 bits; the other rows hold zeros, or what they held
    used = torch.unique(ids[(ids >= 0) & (ids < rows)])
    place = torch.full((rows,), -1, dtype=torch.int64)
    place[used.long()] = torch.arange(used.numel())
    inside = (ids >= 0) & (ids < rows)
    local = torch.where(inside, place[ids.long().clamp(0, rows - 1)], -1)
    total, size, n = grad_want(grad, local, used.numel())
    base = 2.0 if accumulate else 0.0
    near(out[used.long().to(dev)], base + 0.75 * total, (n[:, None] + 2) * 2.0 ** -24 * (base + 0.75 * size), otype)
    rest = torch.ones(rows, dtype=torch.bool, device=dev)
    rest[used.long().to(dev)] = False
    assert bool((out[rest] == base).all())


def test_grad_in_several_launches(dev):
    """Rows and blocks of tokens past one launch of 2^18 CTAs: of few tokens by
    the rows, of many by the rows, the blocks and the length of a row.  Whole
    numbers, whose sums are exact; every value is compared, on the device."""
    for count, rows, dim, repeat in ((1500, 2 ** 23 + 999, 2, False),            # one launch's kernel
                                     (5000, 2 ** 26 + 5000, 1, False),           # sums, by rows
                                     (2 ** 23 + 12345, 50, 1, False),            # joins, by blocks
                                     (20000, 40, 2 ** 19 + 4, True)):            # both, by columns
        gen = torch.Generator(device=dev).manual_seed(count)
        ids = torch.randint(-1, rows, (count,), generator=gen, device=dev, dtype=torch.int32)
        ids[::3] = rows - 1
        grad = torch.randint(-4, 5, (1 if repeat else count, dim), generator=gen, device=dev).float()
        ok = ids >= 0
        at = ids[ok].long()
        if repeat:                  # one gradient row for all tokens
            want = torch.bincount(at, minlength=rows).float()[:, None] * grad
            grad = grad.expand(count, dim)
        else:
            want = torch.stack([torch.bincount(at, weights=grad[ok, j].double(), minlength=rows) for j in range(dim)], 1).float()
        out = m.embedding_grad(grad, ids, num_rows=rows)
        assert torch.equal(out, want), (count, rows, dim)
        m.embedding_grad(grad, ids, out=out, accumulate=True)
        assert torch.equal(out, 2 * want), (count, rows, dim)
