"""Operators between tokens and rows on torch device tensors: embedding lookup
and its gradient, distillation from a teacher's top logits, and sampling.

The same manner as ops.py: every call goes through the C ABI (see
include/mgpu_hip.h for the formulas), is enqueued on torch's current stream of
the tensors' device, and computes nothing on the CPU.  Nothing is recorded for
autograd: a training program calls the gradient where it needs it.  Workspaces
come from torch's allocator call by call, so calls on several streams and
captured graphs have their own.

Matrices are float32, float16 or bfloat16 with consecutive values in a row;
rows may lie any distance apart (a slice of a wider tensor, an expanded row).
"""
import math

import torch

from ._native import lib
from .ops import _check, _dev_i32, _ptr, _stream

_ROW_DTYPES = {torch.float32: 4, torch.float16: 6, torch.bfloat16: 7}


def _fits_int(n, name):
    if not -2 ** 31 <= n < 2 ** 31:
        raise ValueError("%s must fit a 32-bit int" % name)
    return n


def _rows_of(t, name, output=False):
    """(row stride, rows, row length) of a matrix; leading dimensions of a
    contiguous tensor count as one."""
    if t.dim():
        _fits_int(t.shape[-1], "the row length of " + name)
        _fits_int(math.prod(t.shape[:-1]), "the number of rows of " + name)
    if t.dtype not in _ROW_DTYPES or not t.is_cuda:
        raise TypeError("%s must be a float32, float16 or bfloat16 CUDA tensor" % name)
    if t.dim() != 2:
        if t.dim() == 0 or not t.is_contiguous():
            raise TypeError("%s must be two-dimensional or contiguous" % name)
        return t.shape[-1], math.prod(t.shape[:-1]), t.shape[-1]
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise TypeError("the values of a row of %s must be consecutive" % name)
    if output and rows > 1 and t.stride(0) < cols:
        raise TypeError("the rows of %s overlap" % name)
    return (t.stride(0) if rows > 1 else cols), rows, cols


def _column(t, dtype, n, name):
    """A contiguous vector of one value a row."""
    if t.dtype != dtype or not t.is_cuda or not t.is_contiguous():
        raise TypeError("%s must be a contiguous %s CUDA tensor" % (name, dtype))
    if t.numel() != n:
        raise ValueError("%s must have one value a row" % name)
    return t


def _same_device(first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError("all tensors must be on one device")


def _scratch(nbytes, device):
    return torch.empty(int(nbytes), dtype=torch.uint8, device=device) if nbytes else None


def _out(out, shape, dtype, device, name="out"):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if out.dtype != dtype:
        raise TypeError("%s must be a %s tensor" % (name, dtype))
    if tuple(out.shape) != tuple(shape):
        raise ValueError("%s must have the shape %s" % (name, tuple(shape)))
    return out


def embedding_lookup(table, ids, scale=1.0, out=None):
    """out[..., :] = scale * table[ids[...]] for an int32 tensor of ids.  Ids
    outside the table are padding and give zeros."""
    _dev_i32(ids, "ids")
    if table.dim() != 2:
        raise TypeError("table must be two-dimensional")
    stride, num_rows, dim = _rows_of(table, "table")
    _fits_int(ids.numel(), "the number of ids")
    out = _out(out, tuple(ids.shape) + (dim,), table.dtype, table.device)
    out_stride, _, _ = _rows_of(out, "out", output=True)
    _same_device(table, ids, out)
    with torch.cuda.device(table.device):
        _check(lib().mgpu_hip_embedding_lookup(
            _ptr(table), num_rows, dim, stride, _ptr(ids), ids.numel(), scale, _ptr(out),
            out_stride, _ROW_DTYPES[table.dtype], _stream()))
    return out


def embedding_grad(grad, ids, num_rows=None, scale=1.0, out=None, accumulate=False):
    """The table's gradient from grad, one row per id: out[v] = scale * (sum
    of the grad rows whose id is v) for all num_rows rows, or, with
    accumulate, that added to the rows of out that occur.

    Give num_rows for a new tensor of grad's type, or out: (num_rows, dim) of
    grad's type or float32.  Ids outside the table add to nothing.  Sums are
    32-bit, in an order that the sizes and ids alone decide, and rounded once
    together with what out held."""
    _dev_i32(ids, "ids")
    stride, count, dim = _rows_of(grad, "grad")
    if count != ids.numel():
        raise ValueError("grad must have one row per id")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        if num_rows is None:
            raise ValueError("num_rows or out must be given")
        out = torch.empty((num_rows, dim), dtype=grad.dtype, device=grad.device)
    if out.dtype not in (grad.dtype, torch.float32):
        raise TypeError("out must have grad's type or be float32")
    if out.dim() != 2 or out.shape[1] != dim or (num_rows is not None and out.shape[0] != num_rows):
        raise ValueError("out must be num_rows rows as long as grad's")
    out_stride, num_rows, _ = _rows_of(out, "out", output=True)
    _same_device(grad, ids, out)
    with torch.cuda.device(grad.device):
        ws = _scratch(lib().mgpu_hip_embedding_grad_workspace_bytes(count, num_rows, dim), grad.device)
        _check(lib().mgpu_hip_embedding_grad(
            _ptr(grad), stride, _ptr(ids), count, num_rows, dim, scale, int(bool(accumulate)),
            _ptr(out), out_stride, _ROW_DTYPES[grad.dtype], _ROW_DTYPES[out.dtype],
            _ptr(ws), ws.numel() if ws is not None else 0, _stream()))
    return out


def _distill_args(logits, teacher_ids, teacher_logits, weights):
    stride, rows, vocab = _rows_of(logits, "logits")
    _dev_i32(teacher_ids, "teacher_ids")
    if teacher_logits.dtype not in _ROW_DTYPES or not teacher_logits.is_cuda or not teacher_logits.is_contiguous():
        raise TypeError("teacher_logits must be a contiguous float32, float16 or bfloat16 CUDA tensor")
    if teacher_ids.shape != teacher_logits.shape or teacher_ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError("teacher_ids and teacher_logits must have a row for each row of logits")
    if weights is not None:
        _column(weights, torch.float32, rows, "weights")
    _same_device(logits, teacher_ids, teacher_logits, weights)
    return stride, rows, vocab, teacher_ids.shape[-1]


def distill_loss(logits, teacher_ids, teacher_logits, temperature=1.0, weights=None):
    """Loss of each row against the teacher's top logits: weight *
    temperature^2 * KL(softmax(teacher_logits / temperature) || softmax(logits
    / temperature)), the first over the entries whose id lies in the
    vocabulary (use -1 for padding).

    Returns ``(loss, norms)``, float32 with a value and with two values a row;
    ``distill_grad`` takes the norms.  Rows of weight 0 are not read; their
    loss and norms are 0."""
    stride, rows, vocab, top = _distill_args(logits, teacher_ids, teacher_logits, weights)
    lead = logits.shape[:-1]
    loss = torch.empty(lead, dtype=torch.float32, device=logits.device)
    norms = torch.empty(tuple(lead) + (2,), dtype=torch.float32, device=logits.device)
    with torch.cuda.device(logits.device):
        _check(lib().mgpu_hip_distill_loss(
            _ptr(logits), stride, rows, vocab, _ptr(teacher_ids), _ptr(teacher_logits), top,
            temperature, _ptr(weights), _ptr(loss), _ptr(norms), _ROW_DTYPES[logits.dtype],
            _ROW_DTYPES[teacher_logits.dtype], _stream()))
    return loss, norms


def distill_grad(logits, norms, teacher_ids, teacher_logits, weights=None, temperature=1.0, out=None):
    """The gradient of distill_loss's losses in the logits, times ``weights``:
    the loss's row weights times the gradient that arrives at each row's loss.
    ``out`` may be the logits themselves."""
    stride, rows, vocab, top = _distill_args(logits, teacher_ids, teacher_logits, weights)
    _column(norms, torch.float32, 2 * rows, "norms")
    out = _out(out, logits.shape, logits.dtype, logits.device)
    out_stride, _, _ = _rows_of(out, "out", output=True)
    _same_device(logits, norms, out)
    with torch.cuda.device(logits.device):
        _check(lib().mgpu_hip_distill_grad(
            _ptr(logits), stride, rows, vocab, _ptr(norms), _ptr(teacher_ids),
            _ptr(teacher_logits), top, temperature, _ptr(weights), _ptr(out), out_stride,
            _ROW_DTYPES[logits.dtype], _ROW_DTYPES[teacher_logits.dtype], _stream()))
    return out


def distill_loss_and_grad(logits, teacher_ids, teacher_logits, temperature=1.0, weights=None, out=None):
    """distill_loss and its gradient in one pass over the logits, for a
    training step whose row weights are known beforehand: ``(loss, grad)``,
    both with the weights in them.  ``out`` receives the gradient and may be
    the logits themselves."""
    stride, rows, vocab, top = _distill_args(logits, teacher_ids, teacher_logits, weights)
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=logits.device)
    out = _out(out, logits.shape, logits.dtype, logits.device)
    out_stride, _, _ = _rows_of(out, "out", output=True)
    _same_device(logits, out)
    with torch.cuda.device(logits.device):
        _check(lib().mgpu_hip_distill_loss_and_grad(
            _ptr(logits), stride, rows, vocab, _ptr(teacher_ids), _ptr(teacher_logits), top,
            temperature, _ptr(weights), _ptr(loss), _ptr(out), out_stride,
            _ROW_DTYPES[logits.dtype], _ROW_DTYPES[teacher_logits.dtype], _stream()))
    return loss, out


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token a row: ``(token, logprob)``, int32 and float32.

    ``uniform`` holds one float32 in [0, 1) a row.  Each setting is a number,
    or a tensor with one value a row (float32; int32 for top_k).  top_k <= 0,
    top_p >= 1 and min_p <= 0 keep everything; temperature <= 0 takes the
    largest logit, the first of several.  A row of nothing but -inf and NaN
    gives token -1 and logprob -inf."""
    stride, rows, vocab = _rows_of(logits, "logits")
    if logits.dim() != 2:
        raise TypeError("logits must be two-dimensional")
    _column(uniform, torch.float32, rows, "uniform")
    settings = []
    for value, dtype, name in ((temperature, torch.float32, "temperature"), (top_k, torch.int32, "top_k"),
                               (top_p, torch.float32, "top_p"), (min_p, torch.float32, "min_p")):
        if isinstance(value, torch.Tensor):
            settings.append((_column(value, dtype, rows, name), 0))
        else:
            settings.append((None, _fits_int(value, name) if dtype is torch.int32 else value))
    tensors = [t for t, _ in settings]
    _same_device(logits, uniform, *tensors)
    token = torch.empty(rows, dtype=torch.int32, device=logits.device)
    logprob = torch.empty(rows, dtype=torch.float32, device=logits.device)
    with torch.cuda.device(logits.device):
        ws = _scratch(lib().mgpu_hip_sample_workspace_bytes(rows, vocab), logits.device)
        _check(lib().mgpu_hip_sample(
            _ptr(logits), stride, rows, vocab, _ptr(uniform), *[_ptr(t) for t in tensors],
            *[v for _, v in settings], _ptr(token), _ptr(logprob), _ROW_DTYPES[logits.dtype],
            _ptr(ws), ws.numel() if ws is not None else 0, _stream()))
    return token, logprob
