"""sample() against the definition in 64 bits, token for token.

The tokens have to be equal: the sums that decide are exact to 2^-38 of the
largest probability or better, and the random numbers drawn here do not come
that near to a border.  A log probability is a 64-bit result rounded to 32
bits: off by 2^-24 relative, and by 1e-9 through the sums."""
import math

import numpy as np
import pytest
import torch

import moderngpu_amd as m

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def draw(z, u, t, k, p, least):
    """One row by the definition."""
    z = np.where(np.isnan(z), -np.inf, np.minimum(z.astype(np.float64), np.float64(np.finfo(np.float32).max)))
    if np.isneginf(z).all():
        return -1, -math.inf
    if not t > 0:
        t, k = 1.0, 1
    order = np.lexsort((np.arange(z.size), -z))
    if 0 < k < z.size:
        order = order[:k]
    with np.errstate(under="ignore", over="ignore"):
        w = np.exp((z[order] - z.max()) / np.float64(np.float32(t)))
    w[np.isneginf(z[order])] = 0
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep = before < max(np.float64(np.float32(p)), 0) * w.sum()
        keep[0] = True
        order, w = order[keep], w[keep]
    keep = w >= min(np.float64(np.float32(least)), 1.0)
    order, w = order[keep], w[keep]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    sums = np.cumsum(w)
    at = int(np.searchsorted(sums, np.float64(np.float32(u)) * sums[-1], side="right"))
    at = min(at, int(np.nonzero(w)[0][-1]))
    return int(order[at]), math.log(w[at] / sums[-1]) if w[at] > 1e-290 else (z[order[at]] - z.max()) / t - math.log(sums[-1])


def check(dev, z, u, t=1.0, k=0, p=1.0, least=0.0, view=None):
    """z: logits on the CPU; settings: numbers or CPU tensors."""
    put = lambda v: v.to(dev) if isinstance(v, torch.Tensor) else v  # noqa: E731
    token, logprob = m.sample(z.to(dev) if view is None else view, u.to(dev), temperature=put(t), top_k=put(k),
                              top_p=put(p), min_p=put(least))
    assert token.dtype == torch.int32 and logprob.dtype == torch.float32
    token, logprob = token.cpu().tolist(), logprob.double().cpu().tolist()
    at = lambda v, r: v[r].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    for r in range(z.shape[0]):
        want, log = draw(z[r].float().numpy(), u[r].item(), at(t, r), at(k, r), at(p, r), at(least, r))
        assert token[r] == want, (r, token[r], want)
        assert logprob[r] == log or abs(logprob[r] - log) <= 2.0 ** -24 * abs(log) + 1e-9, (r, logprob[r], log)
    return token


def logits(rows, vocab, dtype, seed=0, std=2.5):
    gen = torch.Generator().manual_seed(seed * 7919 + rows * 131 + vocab)
    return (torch.randn(rows, vocab, generator=gen) * std).to(dtype), torch.rand(rows, generator=gen)


SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=5), dict(k=40, t=1.3), dict(k=1000), dict(k=2500, p=0.97), dict(p=0.9),
            dict(p=0.3, t=0.5), dict(p=0.999, t=2.0), dict(least=0.05), dict(least=0.3, p=0.8), dict(k=50, p=0.95, least=0.02),
            dict(t=0.0), dict(p=0.0), dict(least=1.0), dict(t=100.0, p=0.7), dict(t=0.01)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "-".join("%s%s" % i for i in s.items()) or "plain")
def test_settings(dev, dtype, settings):
    for rows, vocab in ((3, 1), (2, 2), (4, 63), (5, 1000), (3, 4099), (2, 20011)):
        z, u = logits(rows, vocab, dtype)
        check(dev, z, u, **settings)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 131072), (2, 140003), (70, 9000), (300, 2049), (1, 300007), (0, 10)])
def test_sizes(dev, dtype, rows, vocab):
    z, u = logits(rows, vocab, dtype, seed=2)
    for settings in (dict(), dict(k=50, p=0.9), dict(p=0.95), dict(least=0.01), dict(k=3000)):
        check(dev, z, u, **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_its_own_settings(dev, dtype):
    rows = 64
    z, u = logits(rows, 3001, dtype, seed=4)
    gen = torch.Generator().manual_seed(6)
    pick = lambda values, t: torch.tensor(values, dtype=t)[torch.randint(0, len(values), (rows,), generator=gen)]  # noqa: E731
    check(dev, z, u, t=pick([0.0, 0.5, 1.0, 1.7, -1.0], torch.float32), k=pick([0, -3, 1, 7, 400, 3001, 9999], torch.int32),
          p=pick([1.0, 0.5, 0.9, 0.99, 2.0, 0.0], torch.float32), least=pick([0.0, 0.1, 0.001, -1.0, 3.0], torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_go_to_the_lowest_index(dev, dtype):
    """Few distinct values: every border falls into a group of equal logits,
    over many tiles of the row; and rows of one value only."""
    gen = torch.Generator().manual_seed(10)
    for vocab in (100, 5000, 40000):
        z = torch.randint(-2, 3, (6, vocab), generator=gen).to(dtype)
        z[5] = 1.5
        u = torch.tensor([0.0, 0.1, 0.5, 0.9, 0.99999994, 0.7])
        for settings in (dict(), dict(k=1), dict(k=vocab // 3), dict(k=vocab // 2, p=0.6), dict(p=0.25), dict(p=0.7), dict(p=0.97),
                         dict(least=0.2), dict(t=0.0)):
            check(dev, z, u, **settings)


def test_zero_signs_are_equal(dev):
    z = torch.tensor([[-0.0, 0.0, -0.0, 0.0]]).expand(4, 4).contiguous()
    assert check(dev, z, torch.tensor([0.0, 0.3, 0.6, 0.9]), k=2) == [0, 0, 1, 1]


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows(dev, dtype):
    """-inf, NaN, +inf and the type's lowest value; rows with one token left,
    and with none."""
    z, _ = logits(9, 2500, dtype, seed=12)
    u = torch.linspace(0, 0.99, 9)
    lowest = torch.finfo(dtype).min
    z[0, 10:] = -math.inf
    z[1] = -math.inf
    z[2] = -math.inf
    z[2, 2400] = -5.0
    z[3] = math.nan
    z[4, ::2] = math.nan
    z[5] = lowest
    z[6, 1:] = lowest
    z[7, [3, 99, 2222]] = math.inf
    z[8, 1200:] = -math.inf
    z[8, 7] = math.inf
    for settings in (dict(), dict(k=3), dict(k=2000), dict(p=0.9), dict(least=0.1), dict(k=20, p=0.5, least=0.01), dict(t=0.0),
                     dict(t=50.0, p=0.99)):
        got = check(dev, z, u, **settings)
        assert got[1] == got[3] == -1 and got[2] == 2400 and got[7] in (3, 99, 2222) and got[8] == 7


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dev, dtype):
    """Rows at odd offsets of a wider tensor, with larger values beside them;
    one row for all requests."""
    z, u = logits(5, 1001, dtype, seed=14)
    wide = torch.full((5, 1010), 100.0, dtype=dtype)
    for left in (1, 3, 8):
        wide[:] = 100.0
        wide[:, left:left + 1001] = z
        for settings in (dict(), dict(k=9), dict(p=0.9)):
            check(dev, z, u, view=wide.to(dev)[:, left:left + 1001], **settings)
    one = z[:1].to(dev).expand(5, 1001)
    check(dev, z[:1].expand(5, 1001), u, view=one, p=0.8)


def test_more_rows_than_go_together(dev):
    """Rows past one round of launches, each with its own settings."""
    rows = 20_011
    z, u = logits(rows, 33, torch.float32, seed=16)
    gen = torch.Generator().manual_seed(17)
    k = torch.randint(0, 6, (rows,), generator=gen).to(torch.int32)
    p = torch.rand(rows, generator=gen) * 1.2
    t = torch.rand(rows, generator=gen) * 2
    check(dev, z, u, t=t, k=k, p=p)
    check(dev, z, u, least=torch.rand(rows, generator=gen) * 0.3)


def test_ends_of_the_random_range(dev):
    """u = 0 takes the first kept token with a probability, the largest u
    below 1 the last; numbers outside [0, 1) count as the ends."""
    z = torch.tensor([[-math.inf, 1.0, 0.0, 1.0, -math.inf]]).expand(5, 5).contiguous()
    u = torch.tensor([0.0, 0.99999994, 1.0, -3.0, math.nan], device=dev)
    token, _ = m.sample(z.to(dev), u)
    assert token.tolist() == [1, 3, 3, 1, 1]
    # a token far below the others has no probability and is not the last one
    z[:, 3], z[:, 4] = 1.0, -3000.0
    token, _ = m.sample(z.to(dev), u)
    assert token.tolist() == [1, 3, 3, 1, 1]


def test_shares_follow_the_probabilities(dev):
    """Evenly spread random numbers draw each token as often as its share
    says, to one count either side."""
    n = 4096
    z = torch.tensor([0.5, -1.0, 2.0, 0.0, 1.0])
    u = (torch.arange(n) + 0.5) / n
    token, _ = m.sample(z.to(dev).expand(n, 5), u.to(dev), temperature=1.5)
    counts = torch.bincount(token.long().cpu(), minlength=5)
    assert bool(((counts - n * torch.softmax(z.double() / 1.5, 0)).abs() <= 1).all())


def test_refusals(dev):
    z, u = torch.zeros(3, 8, device=dev), torch.zeros(3, device=dev)
    with pytest.raises(TypeError):
        m.sample(z.double(), u)
    with pytest.raises(TypeError):
        m.sample(z[0], u[:1])
    with pytest.raises(TypeError):
        m.sample(z, u.double())
    with pytest.raises(ValueError):
        m.sample(z, u[:2].contiguous())
    with pytest.raises(TypeError):
        m.sample(z, u, top_k=torch.ones(3, device=dev))
    with pytest.raises(ValueError):
        m.sample(z, u, temperature=torch.ones(2, device=dev))
    with pytest.raises(ValueError):
        m.sample(z, u, top_k=1 << 40)
    with pytest.raises(m.MgpuError):
        m.sample(z[:, :0], u)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_settings(dev, dtype):
    """NaN, one for all rows or a row's own: the temperature counts as 0,
    top_p and min_p as not given."""
    z, u = logits(5, 3001, dtype, seed=18)
    for given, meant in ((dict(t=math.nan), dict(t=0.0)), (dict(p=math.nan), dict()), (dict(least=math.nan), dict()),
                         (dict(p=math.nan, least=math.nan), dict()), (dict(p=0.8, least=math.nan), dict(p=0.8)),
                         (dict(k=40, least=math.nan), dict(k=40)), (dict(p=math.nan, least=0.1), dict(least=0.1)),
                         (dict(t=math.nan, p=0.9, least=math.nan), dict(t=0.0))):
        want = check(dev, z, u, **meant)
        for value in (lambda v: v, lambda v: torch.full((5,), v, device=dev)):
            token, _ = m.sample(z.to(dev), u.to(dev), temperature=value(given.get("t", 1.0)), top_k=given.get("k", 0),
                                top_p=value(given.get("p", 1.0)), min_p=value(given.get("least", 0.0)))
            assert token.tolist() == want, given


@pytest.mark.parametrize("dtype", TYPES)
def test_logits_many_temperatures_from_zero(dev, dtype):
    """Logits a few steps of the type apart that lie 10^7 temperatures and more
    from zero: the products logit / temperature are further apart than 1."""
    step = lambda a: 2.0 ** (math.frexp(a)[1]) * torch.finfo(dtype).eps / 2  # noqa: E731
    for vocab in (8192, 20011):
        for a in (23300014.0, 15.1, 2000000.0, -15.1, 1.7):
            a = torch.tensor(a).clamp(max=60000.0 if dtype == torch.float16 else 1e9).to(dtype).item()
            for steps, share in ((3, 1 / 6), (4, 0.17), (2, 0.3), (1, 1.0)):
                z = torch.full((3, vocab), a - steps * step(a)).to(dtype)
                z[:, 0] = a
                z[1, ::3] = a - (steps + 1) * step(a)
                z[2, ::7] = -math.inf
                u = torch.tensor([0.9871234, 0.31, 0.6])
                t = float(np.float32(steps * step(a) * share))
                for settings in (dict(p=0.5), dict(p=0.9), dict(least=0.001), dict(p=0.9, least=0.001), dict()):
                    check(dev, z, u, t=t, **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_temperatures_next_to_zero(dev, dtype):
    """Temperatures that leave a few tokens; logits among the smallest numbers
    with a temperature among them."""
    z, u = logits(4, 20011, dtype, seed=20)
    for t in (1e-3, 1e-5, 1e-6, 1e-8, 1e-20, 1e-38, 1e-45):
        for settings in (dict(p=0.95), dict(p=0.5, least=0.1), dict(least=0.3), dict(k=50, p=0.9), dict()):
            check(dev, z, u, t=t, **settings)
    if dtype != torch.float16:
        small = (z.double() * 4e-39).to(dtype)
        for t in (1e-38, 1.8e-38, 1.2e-38):
            for settings in (dict(p=0.3), dict(p=0.95), dict(least=0.01, p=0.7), dict(k=30), dict()):
                check(dev, small, u, t=t, **settings)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [270001, 600001])
def test_wide_vocabularies(dev, dtype, vocab):
    """More than 64 pieces, and runs of more than 64 chunks; candidates for a k
    of 256 that outdo each other across pieces."""
    z, u = logits(2, vocab, dtype, seed=22)
    z[1, ::5] = -math.inf
    for settings in (dict(), dict(p=0.95), dict(p=0.9, least=0.001), dict(least=0.01), dict(k=256), dict(k=256, p=0.9),
                     dict(k=1536), dict(k=5000, p=0.99), dict(t=2.0, p=0.999), dict(t=0.0)):
        check(dev, z, u, **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_in_a_wide_vocabulary(dev, dtype):
    """One value all through, and few values: a border is an index of three
    digits."""
    gen = torch.Generator().manual_seed(23)
    z = torch.randint(-2, 3, (2, 600001), generator=gen).to(dtype)
    z[0] = 0.5
    u = torch.tensor([0.77, 0.99])
    for settings in (dict(), dict(k=256), dict(k=450001), dict(p=0.7), dict(k=500000, p=0.4), dict(p=0.3, least=0.1), dict(t=0.0)):
        check(dev, z, u, **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_widest_vocabulary(dev, dtype):
    """2048 pieces, in two rounds of a CTA's threads; masses of 38 bits."""
    z, u = logits(1, 1 << 24, dtype, seed=24)
    assert m.lib().mgpu_hip_sample_workspace_bytes(1, 1 << 24) > 0
    for settings in (dict(), dict(p=0.9), dict(k=300, p=0.8)):
        check(dev, z, u, **settings)
    ties = torch.full_like(z, 3.0)
    ties[0, :100] = -math.inf
    for settings in (dict(), dict(p=0.6), dict(k=(1 << 24) - 5000)):
        check(dev, ties, u, **settings)
