"""distill_loss, distill_grad and distill_loss_and_grad against the formulas in
64 bits.

Tolerances, with u = 2^-24 (half a step of a 32-bit float).  An exponential
2^y, y = (z - max) * c, is off by 3 u |y| ln 2 through its argument (difference,
c and product are each rounded) and 2 u through itself; a sum of such terms, all
positive, by as much again plus u for each addition that follows another.  A
thread adds vocab / 64 of them at most, and the joining of threads a few dozen.
So a share q or p is off by E(y) = u (6 |y| + 2 vocab / 64 + 128) relative.
Below 2^-126 an exponential may be 0.  log q is off by E(y) too, log p
likewise, and each by u for its own value; products and sums of `top` terms
add u each."""
import math

import pytest
import torch

import moderngpu_amd as m

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


class Want:
    """Loss, gradient and how far 32-bit arithmetic may be off them."""

    def __init__(self, z, ids, teacher, tau, weights, arriving=None):
        if not ids.shape[1]:                    # no entries: one that does not count
            ids, teacher = torch.full((z.shape[0], 1), -1), torch.zeros(z.shape[0], 1)
        z, a, w = z.double(), teacher.double() / tau, weights.double()
        rows, vocab = z.shape
        top = ids.shape[1]
        ids = ids.long()
        ok = (ids >= 0) & (ids < vocab)
        at = ids.clamp(0, max(vocab - 1, 0))
        a = torch.where(ok, a, torch.full_like(a, -math.inf))
        self.live = (w != 0) & (a > -math.inf).any(1)
        live = self.live[:, None]
        a = torch.where(live, a, torch.zeros_like(a))
        log_p = a - torch.logsumexp(a, 1, keepdim=True)
        p = torch.where(ok, log_p.exp(), 0.0)
        none = torch.isneginf(z).all(1, keepdim=True)
        y = torch.where(none, -math.inf, z / tau - z.amax(1, keepdim=True) / tau)
        log_q = torch.where(none, -math.inf, y - torch.log(y.exp().sum(1, keepdim=True)))
        q = torch.where(none, 0.0, log_q.exp())
        picked = log_q.gather(1, at)
        term = torch.where(p > 0, p * (log_p - picked), 0.0)
        clip = lambda t: t.abs().clamp(max=150 * math.log(2))  # noqa: E731
        add = 2 * vocab / 64 + 128
        e_q = U * (6 / math.log(2) * clip(y) + add)
        e_p = U * (6 / math.log(2) * clip(a - a.amax(1, keepdim=True)) + 2 * top + 128)
        scale = (w * tau * tau)
        self.loss = torch.where(self.live, scale * term.sum(1), 0.0)
        finite = torch.where(torch.isfinite(picked), picked, 0.0)
        lp = torch.where(torch.isfinite(log_p), log_p, 0.0)
        slack = (p * (e_q.gather(1, at) + e_p + U * 4 * (lp.abs() + finite.abs())) + term.abs() * (e_p + U * (top + 8))).sum(1)
        self.loss_slack = scale.abs() * torch.where(torch.isfinite(slack), slack, 0.0) + 1e-30
        target = torch.zeros_like(q).scatter_add(1, at, torch.where(live, p, 0.0))
        target_slack = torch.zeros_like(q).scatter_add(1, at, torch.where(live, p * e_p, 0.0))
        c = ((w if arriving is None else w * arriving.double()) * tau)[:, None]
        self.grad = torch.where(live, c * (q - target), 0.0)
        self.grad_slack = torch.where(live, c.abs() * (q * (e_q + 8 * U) + target_slack + target * 8 * U + 2.0 ** -125), 0.0)
        self.max, self.log_sum = z.amax(1), torch.log(y.exp().sum(1))

    def check_loss(self, got):
        got = got.double().cpu()
        inf = torch.isinf(self.loss)
        assert torch.equal(got[inf], self.loss[inf])
        assert bool(((got - self.loss).abs()[~inf] <= (self.loss_slack + U * self.loss.abs())[~inf]).all())
        assert not got[~self.live].any()

    def check_grad(self, got, dtype):
        assert got.dtype == dtype
        got = got.double().cpu()
        step = torch.finfo(dtype).eps / 2 * (self.grad.abs() + self.grad_slack) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)
        over = (got - self.grad).abs() - self.grad_slack - step
        assert bool((over <= 0).all()), over.max().item()
        assert not got[~self.live].any()


def make(rows, vocab, top, dtype, teacher_type=torch.float32, seed=0, distinct=True):
    gen = torch.Generator().manual_seed(seed + rows * 1009 + vocab)
    z = (torch.randn(rows, vocab, generator=gen) * 3).to(dtype)
    if distinct and rows and top <= vocab:
        ids = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(rows)])
    else:
        ids = torch.randint(0, max(1, min(vocab, top // 3 + 1)), (rows, top), generator=gen)
    ids = ids.reshape(rows, top)
    ids[torch.rand(rows, top, generator=gen) < 0.2] = -1
    ids[torch.rand(rows, top, generator=gen) < 0.05] = vocab
    teacher = (torch.randn(rows, top, generator=gen) * 3).to(teacher_type)
    weights = torch.rand(rows, generator=gen) + 0.25
    weights[torch.rand(rows, generator=gen) < 0.2] = 0
    return z, ids.to(torch.int32), teacher, weights


def run_all(dev, z, ids, teacher, weights, tau, dtype):
    """All three entry points on the same rows."""
    args = [t.to(dev) for t in (z, ids, teacher)]
    w = weights.to(dev)
    want = Want(z, ids, teacher, tau, weights)
    loss, grad = m.distill_loss_and_grad(*args, temperature=tau, weights=w)
    want.check_loss(loss)
    want.check_grad(grad, dtype)
    loss2, norms = m.distill_loss(*args, temperature=tau, weights=w)
    want.check_loss(loss2)
    gen = torch.Generator().manual_seed(77)
    arriving = torch.rand(z.shape[0], generator=gen) - 0.3
    later = Want(z, ids, teacher, tau, weights, arriving)
    grad2 = m.distill_grad(args[0], norms, args[1], args[2], w * arriving.to(dev), temperature=tau)
    later.check_grad(grad2, dtype)
    return loss, grad, norms


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (2, 3, 2), (5, 64, 7), (3, 1000, 64), (4, 1001, 1), (2, 4099, 257),
                                            (7, 515, 515), (1, 9001, 1024), (3, 33000, 40), (2, 70001, 3), (2, 131072, 33),
                                            (1, 140001, 5), (2, 300007, 5), (600, 130, 9), (0, 100, 4), (3, 50, 0)])
def test_distill(dev, rows, vocab, top, dtype):
    z, ids, teacher, weights = make(rows, vocab, top, dtype)
    run_all(dev, z, ids, teacher, weights, 1.5, dtype)


@pytest.mark.parametrize("teacher_type", TYPES)
@pytest.mark.parametrize("tau", [0.25, 1.0, 8.0])
def test_teacher_types_and_temperatures(dev, teacher_type, tau):
    for dtype in TYPES:
        z, ids, teacher, weights = make(6, 777, 20, dtype, teacher_type, seed=3)
        run_all(dev, z, ids, teacher, weights, tau, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_index_many_times(dev, dtype):
    z, ids, teacher, weights = make(9, 400, 100, dtype, distinct=False)
    ids[4] = 7
    weights[4] = 1
    run_all(dev, z, ids, teacher, weights, 2.0, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits_and_rows(dev, dtype):
    """-inf and the type's lowest value among the logits, rows of nothing else,
    rows without a teacher, teacher entries of -inf, and rows of weight 0 that
    hold NaN and infinities."""
    z, ids, teacher, weights = make(12, 300, 10, dtype, seed=5)
    weights[:] = 1.0
    lowest = torch.finfo(dtype).min
    ids[:] = torch.arange(10, dtype=torch.int32)[None] * 7
    z[0, 100:] = -math.inf
    z[1, 100:] = lowest
    z[2] = -math.inf                      # nothing left: q = 0, infinite loss
    z[3] = lowest                         # all equal: q = 1 / 300
    ids[4] = -1
    ids[5] = 2 ** 31 - 1
    teacher[6, 3:] = -math.inf
    teacher[7] = -math.inf
    weights[8] = 0
    z[8, 5], z[8, 6], teacher[8, 1] = math.nan, math.inf, math.nan
    z[9, 7] = -math.inf                   # a teacher's token that the student rules out: infinite loss
    teacher[10, 2], ids[10, 2] = math.nan, -1
    z[11, :] = -math.inf
    z[11, 0] = 2.0                        # one token left
    ids[11, 1:] = -1
    loss, _, norms = run_all(dev, z, ids, teacher, weights, 1.0, dtype)
    assert math.isinf(loss[2]) and math.isinf(loss[9]) and loss[11] == 0
    assert norms[8].tolist() == [0, 0]


def test_lowest_values_with_a_small_temperature(dev):
    """The largest logit times 1 / temperature lies past the largest float."""
    z = torch.full((2, 130), torch.finfo(torch.float32).min)
    z[1, 64:] = torch.finfo(torch.float32).max
    ids = torch.tensor([[3], [70]], dtype=torch.int32)
    run_all(dev, z, ids, torch.zeros(2, 1), torch.ones(2), 0.5, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_inf_reach_loss_and_gradient(dev, dtype):
    z, ids, teacher, weights = make(4, 700, 6, dtype)
    weights[:] = 1
    ids[:] = torch.arange(6, dtype=torch.int32)
    z[0, 650] = math.nan
    z[1, 3] = math.inf
    z[2] = -math.inf
    z[2, 699] = math.nan
    args = [t.to(dev) for t in (z, ids, teacher)]
    loss, grad = m.distill_loss_and_grad(*args, weights=weights.to(dev))
    loss2, norms = m.distill_loss(*args, weights=weights.to(dev))
    grad2 = m.distill_grad(args[0], norms, *args[1:], weights=weights.to(dev))
    for l in (loss, loss2):
        assert bool(torch.isnan(l[:3]).all()) and bool(torch.isfinite(l[3]))
    for g in (grad, grad2):
        assert bool(torch.isnan(g[:2]).all()) and bool(torch.isfinite(g[3]).all())
    teacher[3, 2] = math.nan
    loss, _ = m.distill_loss_and_grad(args[0], args[1], teacher.to(dev))
    assert bool(torch.isnan(loss[3]))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_in_place_and_no_weights(dev, dtype):
    """Logits and gradients inside wider tensors, at odd offsets; gradients
    written over the logits; an expanded row."""
    z, ids, teacher, _ = make(5, 1003, 12, dtype, seed=11)
    ones = torch.ones(5)
    want = Want(z, ids, teacher, 1.0, ones)
    ids_d, teacher_d = ids.to(dev), teacher.to(dev)
    for left, right in ((1, 4), (0, 5), (3, 0)):
        outer = torch.full((5, left + 1003 + right), 9.0, dtype=dtype, device=dev)
        view = outer[:, left:left + 1003]
        view.copy_(z.to(dev))
        loss, grad = m.distill_loss_and_grad(view, ids_d, teacher_d)
        want.check_loss(loss)
        want.check_grad(grad, dtype)
        into = torch.full((5, 1003 + 2), 4.0, dtype=dtype, device=dev)
        loss, norms = m.distill_loss(view, ids_d, teacher_d)
        m.distill_grad(view, norms, ids_d, teacher_d, out=into[:, 1:1004])
        want.check_grad(into[:, 1:1004], dtype)
        assert bool((into[:, 0] == 4).all()) and bool((into[:, 1004] == 4).all())
        loss, grad = m.distill_loss_and_grad(view, ids_d, teacher_d, out=view)
        want.check_loss(loss)
        want.check_grad(view, dtype)
        assert bool((outer[:, :left] == 9).all()) and bool((outer[:, left + 1003:] == 9).all())
    one = z[:1].expand(5, 1003)
    want = Want(one, ids, teacher, 1.0, ones)
    loss, grad = m.distill_loss_and_grad(z[:1].to(dev).expand(5, 1003), ids_d, teacher_d)
    want.check_loss(loss)
    want.check_grad(grad, dtype)


def test_gradient_leaves_the_norms(dev):
    """One loss, two gradients: a row that counts for nothing in the first
    does in the second."""
    gen = torch.Generator().manual_seed(21)
    z = torch.randn(4, 300, generator=gen).to(dev)
    ids = torch.randint(0, 300, (4, 5), generator=gen).to(torch.int32).to(dev)
    a = torch.randn(4, 5, generator=gen).to(dev)
    loss, norms = m.distill_loss(z, ids, a)
    kept = norms.clone()
    want = m.distill_grad(z, norms, ids, a)
    none = m.distill_grad(z, norms, ids, a, weights=torch.tensor([0.0, 1, 0, 1], device=dev))
    assert torch.equal(norms, kept)
    assert not none[0].any() and not none[2].any()
    assert torch.equal(m.distill_grad(z, norms, ids, a), want)


def test_entries_without_dimensions_are_refused(dev):
    z = torch.zeros(8, device=dev)
    with pytest.raises(ValueError):
        m.distill_loss(z, torch.tensor(1, dtype=torch.int32, device=dev), torch.tensor(0.0, device=dev))
    loss, _ = m.distill_loss(z, torch.ones(1, dtype=torch.int32, device=dev), torch.zeros(1, device=dev))
    assert abs(loss.item() - math.log(8)) < 1e-5


def test_empty_rows(dev):
    """No logits at all: no teacher entry is usable."""
    z = torch.empty(3, 0, device=dev)
    ids, a = torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.zeros(3, 2, device=dev)
    loss, grad = m.distill_loss_and_grad(z, ids, a)
    assert loss.tolist() == [0, 0, 0] and grad.shape == (3, 0)
    loss, norms = m.distill_loss(z, ids, a)
    assert loss.tolist() == [0, 0, 0] and not norms.any()


def test_more_rows_than_one_launch(dev):
    rows = (1 << 20) + 3
    z = torch.zeros(rows, 4, device=dev)
    z[-2, 1] = 2.0
    ids = torch.ones(rows, 1, dtype=torch.int32, device=dev)
    loss, grad = m.distill_loss_and_grad(z, ids, torch.zeros(rows, 1, device=dev))
    flat, peak = math.log(4), math.log(3 + math.exp(2)) - 2
    assert abs(loss[-1].item() - flat) < 1e-5 and abs(loss[-2].item() - peak) < 1e-5 and abs(loss[1 << 19].item() - flat) < 1e-5
    assert (grad[-1].cpu() - torch.tensor([0.25, -0.75, 0.25, 0.25])).abs().max() < 1e-6
    assert bool((loss[:-2] == loss[0]).all()) and bool((grad[:-2] == grad[0]).all())


def test_leading_dimensions(dev):
    z, ids, teacher, weights = make(6, 100, 5, torch.float32)
    shape = lambda t: t.reshape((2, 3) + t.shape[1:]).to(dev)  # noqa: E731
    loss, grad = m.distill_loss_and_grad(shape(z), shape(ids), shape(teacher), weights=shape(weights))
    want = Want(z, ids, teacher, 1.0, weights)
    assert loss.shape == (2, 3) and grad.shape == (2, 3, 100)
    want.check_loss(loss.reshape(6))
    want.check_grad(grad.reshape(6, 100), torch.float32)


def test_gradient_against_differences(dev):
    """Central differences of the 64-bit loss: off by h^2 / 6 times its third
    derivative, which is below weight * tau^2 / tau^3 for a softmax."""
    z, ids, teacher, weights = make(3, 40, 6, torch.float32, seed=21)
    weights[:] = torch.tensor([1.0, 0.5, 2.0])
    tau, h = 2.0, 1e-3
    ids[:, 0] = torch.tensor([1, 2, 3])
    _, grad = m.distill_loss_and_grad(z.to(dev), ids.to(dev), teacher.to(dev), temperature=tau, weights=weights.to(dev))
    base = Want(z, ids, teacher, tau, weights)
    for r in range(3):
        for v in (0, 1, 2, 3, 17, 39):
            step = torch.zeros(3, 40, dtype=torch.float64)
            step[r, v] = h
            f = lambda s: Want(z.double() + s, ids, teacher, tau, weights).loss[r]  # noqa: E731
            difference = (f(step) - f(-step)) / (2 * h)
            slack = base.grad_slack[r, v] + U * base.grad[r, v].abs() + h * h / 6 * weights[r] / tau + 1e-11 / h
            assert abs(difference - grad[r, v].double().cpu()) <= slack


def test_large_rows_past_32_bit_offsets(dev):
    """More than 2^31 logits in one call; the last rows are looked at."""
    rows, vocab = 16500, 131072
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=dev)
    z[-1, 5] = 4.0
    ids = torch.full((rows, 1), 5, dtype=torch.int32, device=dev)
    teacher = torch.zeros(rows, 1, device=dev)
    loss, _ = m.distill_loss_and_grad(z, ids, teacher, out=z)
    flat = math.log(vocab)
    last = math.log(vocab - 1 + math.exp(4)) - 4
    assert abs(loss[0].item() - flat) < 1e-4 and abs(loss[-2].item() - flat) < 1e-4 and abs(loss[-1].item() - last) < 1e-4
    tail = z[-2:].double().cpu()
    assert tail[0, 5] == -1 and tail[0, 6] == 2.0 ** -17
    assert abs(tail[1, 5] - (math.exp(-last) - 1)) < 2.0 ** -8 and tail[1].sum().abs() < 0.01


def test_refusals(dev):
    z = torch.zeros(3, 8, device=dev)
    ids = torch.zeros(3, 2, dtype=torch.int32, device=dev)
    a = torch.zeros(3, 2, device=dev)
    with pytest.raises(TypeError):
        m.distill_loss(z.double(), ids, a)
    with pytest.raises(TypeError):
        m.distill_loss(z, ids.long(), a)
    with pytest.raises(ValueError):
        m.distill_loss(z, ids, a[:, :1].contiguous())
    with pytest.raises(ValueError):
        m.distill_loss(z, ids, a, weights=torch.ones(2, device=dev))
    with pytest.raises(m.MgpuError):
        m.distill_loss(z, ids, a, temperature=0.0)
    with pytest.raises(m.MgpuError):
        m.distill_loss(z, torch.zeros(3, 1025, dtype=torch.int32, device=dev), torch.zeros(3, 1025, device=dev))
    with pytest.raises(ValueError):
        m.distill_grad(z, torch.zeros(3, device=dev), ids, a)
    wide = torch.zeros(3, 9, device=dev)
    with pytest.raises(m.MgpuError):
        m.distill_loss_and_grad(wide[:, :8], ids, a, out=wide[:, 1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau", [0.5, 1.0, 2.0])
def test_teachers_tokens_that_hold_the_lowest_value(dev, dtype, tau):
    """A student that masks with its type's lowest value rules out tokens of
    the teacher's: log q lies near or past the lowest float, the loss is
    finite.  Weights of a mean over rows; a row that holds the largest value
    as well."""
    z, ids, teacher, weights = make(4, 900, 8, dtype, seed=25)
    lowest = torch.finfo(dtype).min
    ids[:] = torch.arange(8, dtype=torch.int32) * 100
    teacher[:] = torch.linspace(0, 1, 8)
    weights[:] = 2.0 ** -6
    z[0, 100] = lowest
    z[1, ::100] = lowest
    z[2, 1:] = lowest
    z[3, 300], z[3, 5] = lowest, -lowest
    loss, _, _ = run_all(dev, z, ids, teacher, weights, tau, dtype)
    assert bool(torch.isfinite(loss).all())
