"""Refusals of the operators between tokens and rows: bad sizes, types,
pointers and overlapping buffers are turned into errors on the host, before
anything is enqueued (these run without a GPU)."""
import ctypes

import pytest
import torch

import moderngpu_amd as m

INVALID = 1
F32, F64, F16, BF16 = 4, 5, 6, 7


@pytest.fixture(scope="module")
def mem():
    """Addresses to refuse, far enough apart not to overlap by accident."""
    buf = (ctypes.c_char * (1 << 20))()
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    return buf, [base + i * (1 << 16) for i in range(12)]


def test_lookup_refuses(mem):
    _, p = mem
    f = m.lib().mgpu_hip_embedding_lookup
    good = dict(table=p[0], rows=8, dim=4, ts=4, ids=p[1], n=5, scale=1.0, out=p[2], os=4, dt=F32)

    def call(**kw):
        a = dict(good, **kw)
        return f(a["table"], a["rows"], a["dim"], a["ts"], a["ids"], a["n"], a["scale"], a["out"], a["os"], a["dt"], None)
    for bad in (dict(rows=-1), dict(dim=-1), dict(n=-1), dict(ts=-4), dict(os=3), dict(dt=F64), dict(dt=0), dict(dt=9),
                dict(table=None), dict(ids=None), dict(out=None), dict(table=p[0] + 2), dict(ids=p[1] + 1),
                dict(out=p[2] + 1), dict(out=p[0]), dict(out=p[0] + 16 * 7), dict(out=p[1]),
                dict(ts=1 << 61), dict(os=1 << 61), dict(out=p[2] + 1, dt=BF16),
                dict(n=(1 << 31) - 1, dim=1 << 12, os=1 << 12)):
        assert call(**bad) == INVALID, bad
    assert call(n=0, ids=None, out=None) == 0                    # nothing to do
    assert call(dim=0) == 0


def test_grad_refuses(mem):
    _, p = mem
    L = m.lib()
    need = L.mgpu_hip_embedding_grad_workspace_bytes(5, 8, 4)
    assert L.mgpu_hip_embedding_grad_workspace_bytes(-1, 8, 4) == 0
    good = dict(grad=p[0], gs=4, ids=p[1], n=5, rows=8, dim=4, out=p[2], os=4, gt=BF16, ot=BF16, ws=p[3], nb=1 << 16)

    def call(**kw):
        a = dict(good, **kw)
        return L.mgpu_hip_embedding_grad(a["grad"], a["gs"], a["ids"], a["n"], a["rows"], a["dim"], 1.0, 0, a["out"],
                                         a["os"], a["gt"], a["ot"], a["ws"], a["nb"], None)
    for bad in (dict(n=-1), dict(rows=-1), dict(dim=-1), dict(gs=-1), dict(os=3), dict(gt=F64), dict(ot=F16),
                dict(gt=F32, ot=BF16), dict(grad=None), dict(ids=None), dict(out=None), dict(out=p[0]),
                dict(out=p[1]), dict(grad=p[0] + 1), dict(out=p[2] + 2, ot=F32), dict(n=(1 << 31) - 1, dim=1 << 12)):
        assert call(**bad) == INVALID, bad
    if need:
        assert call(nb=need - 1) == INVALID
        assert call(ws=None) == INVALID
    assert call(dim=0) == 0 and call(rows=0, out=None) == 0


def test_distill_refuses(mem):
    _, p = mem
    L = m.lib()
    good = dict(z=p[0], zs=16, rows=3, vocab=16, ids=p[1], a=p[2], top=4, tau=1.0, w=p[3], loss=p[4], norms=p[5],
                grad=p[6], gs=16, dt=F16, tt=F32)

    # Each entry point by itself: a call that is not refused would launch a
    # kernel on these addresses where there is a GPU.
    def args(kw):
        a = dict(good, **kw)
        return (a, (a["z"], a["zs"], a["rows"], a["vocab"]), (a["ids"], a["a"], a["top"], a["tau"], a["w"]),
                (a["dt"], a["tt"], None))

    def loss(**kw):
        a, front, teacher, back = args(kw)
        return L.mgpu_hip_distill_loss(*front, *teacher, a["loss"], a["norms"], *back)

    def grad(**kw):
        a, front, teacher, back = args(kw)
        return L.mgpu_hip_distill_grad(*front, a["norms"], *teacher, a["grad"], a["gs"], *back)

    def both(**kw):
        a, front, teacher, back = args(kw)
        return L.mgpu_hip_distill_loss_and_grad(*front, *teacher, a["loss"], a["grad"], a["gs"], *back)

    for bad in (dict(rows=-1), dict(vocab=-1), dict(top=-1), dict(top=1025), dict(tau=0.0), dict(tau=-1.0),
                dict(tau=float("nan")), dict(tau=float("inf")), dict(tau=1e-39), dict(tau=1e30), dict(zs=-1), dict(dt=F64), dict(tt=F64),
                dict(z=None), dict(ids=None), dict(a=None), dict(z=p[0] + 1), dict(w=p[3] + 2)):
        for call in (loss, grad, both):
            assert call(**bad) == INVALID, bad
    for bad in (dict(gs=15), dict(grad=None), dict(grad=p[0] + 2),      # rows that overlap; neither apart from the logits nor the same
                dict(grad=p[0], gs=17), dict(grad=p[1])):
        for call in (grad, both):
            assert call(**bad) == INVALID, bad
    for bad in (dict(loss=None), dict(loss=p[0])):
        for call in (loss, both):
            assert call(**bad) == INVALID, bad
    assert loss(loss=p[5]) == INVALID                             # loss and norms
    assert grad(norms=None) == INVALID
    assert loss(rows=0) == grad(rows=0) == both(rows=0) == 0


def test_sample_refuses(mem):
    _, p = mem
    L = m.lib()
    good = dict(z=p[0], zs=16, rows=3, vocab=16, u=p[1], t=p[2], k=p[3], tp=p[4], mp=p[5], tok=p[6], lp=p[7], dt=BF16,
                ws=p[8], nb=1 << 16)
    need = L.mgpu_hip_sample_workspace_bytes(3, 16)
    assert L.mgpu_hip_sample_workspace_bytes(3, (1 << 24) + 1) == 0

    def call(**kw):
        a = dict(good, **kw)
        return L.mgpu_hip_sample(a["z"], a["zs"], a["rows"], a["vocab"], a["u"], a["t"], a["k"], a["tp"], a["mp"],
                                 1.0, 0, 1.0, 0.0, a["tok"], a["lp"], a["dt"], a["ws"], a["nb"], None)
    for bad in (dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(zs=-1), dict(dt=F64), dict(z=None),
                dict(u=None), dict(tok=None), dict(lp=None), dict(tok=p[0]), dict(lp=p[1]), dict(tok=p[7]),
                dict(tok=p[3]), dict(z=p[0] + 1), dict(t=p[2] + 1)):
        assert call(**bad) == INVALID, bad
    if need:
        assert call(nb=need - 1) == INVALID
        assert call(ws=None) == INVALID
    assert call(rows=0) == 0


def test_python_layer_refuses():
    t, ids = torch.zeros(4, 4), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        m.embedding_lookup(t, ids)
    with pytest.raises(TypeError):
        m.embedding_grad(t, ids, num_rows=4)
    with pytest.raises(TypeError):
        m.distill_loss(t, ids, t)
    with pytest.raises(TypeError):
        m.sample(t, torch.zeros(4))


def test_grad_refuses_a_small_workspace(mem):
    _, p = mem
    L = m.lib()
    need = L.mgpu_hip_embedding_grad_workspace_bytes(5000, 8, 4)
    assert need > 5000 * 4
    for ws, nb in ((p[3], need - 1), (None, need), (p[3] + 2, need)):
        assert L.mgpu_hip_embedding_grad(p[0], 4, p[5], 5000, 8, 4, 1.0, 0, p[2], 4, F16, F16, ws, nb, None) == INVALID


def test_numbers_past_what_kernels_index_are_refused(mem):
    """Rows at one address (stride 0) take no memory, so these sizes can be
    asked for; loops over a row would pass the largest int."""
    _, p = mem
    L = m.lib()
    big = (1 << 30) + 1
    assert L.mgpu_hip_embedding_lookup(p[0], 1, big, 0, p[1], 1, 1.0, p[2] + (1 << 40), big, F32, None) == INVALID
    for n, rows, dim in ((big, 1, 1), (1, big, 1), (1, 1, big)):
        assert L.mgpu_hip_embedding_grad_workspace_bytes(n, rows, dim) == 0
        assert L.mgpu_hip_embedding_grad(p[0], 0, p[1], n, rows, dim, 1.0, 0, p[2] + (1 << 40), dim, F32, F32,
                                         p[3], 1 << 62, None) == INVALID
    assert L.mgpu_hip_distill_loss(p[0], 0, 1, big, p[1] + (1 << 40), p[2] + (1 << 40), 1, 1.0, None,
                                   p[3] + (1 << 41), None, F32, F32, None) == INVALID
    assert L.mgpu_hip_distill_grad(p[0], 0, 1, big, p[3], p[1], p[2], 1, 1.0, None, p[2] + (1 << 41), big, F32, F32,
                                   None) == INVALID


def test_numbers_of_rows_past_2_30_are_refused(mem):
    """One row of logits for all (stride 0) is small; a counter of rows that
    go launch by launch would pass the largest int."""
    _, p = mem
    L = m.lib()
    far = lambda i: p[0] + (i << 40)  # noqa: E731
    for rows in ((1 << 30) + 1, (1 << 31) - 1):
        teacher = (far(1), far(2), 1, 1.0, None)
        assert L.mgpu_hip_distill_loss(p[0], 0, rows, 1, *teacher, far(3), far(4), F32, F32, None) == INVALID
        assert L.mgpu_hip_distill_grad(p[0], 0, rows, 1, far(4), *teacher, far(5), 1, F32, F32, None) == INVALID
        assert L.mgpu_hip_distill_loss_and_grad(p[0], 0, rows, 1, *teacher, far(3), far(5), 1, F32, F32, None) == INVALID
        assert L.mgpu_hip_sample_workspace_bytes(rows, 1) == 0
        assert L.mgpu_hip_sample(p[0], 0, rows, 1, far(1), None, None, None, None, 1.0, 0, 1.0, 0.0, far(2), far(3),
                                 F32, p[1], 1 << 40, None) == INVALID
