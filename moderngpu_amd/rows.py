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
from .ops import _check

_ROW_DTYPES = {torch.float32: 4, torch.float16: 6, torch.bfloat16: 7}


def _fits_int(n, name):
    if not -2 ** 31 <= n < 2 ** 31:
        raise ValueError("%s must fit a 32-bit int" % name)
    return n


def _rows_of(t, name, output=False):
    """(row stride, rows, row length) of a matrix; leading dimensions of a
    contiguous tensor count as one."""
    if t.dtype not in _ROW_DTYPES or not t.is_cuda:
        raise TypeError("%s must be a float32, float16 or bfloat16 CUDA tensor" % name)
    shape = t.shape
    if len(shape) == 2:
        rows, cols = shape
        stride, step = t.stride()
        if cols > 1 and step != 1:
            raise TypeError("the values of a row of %s must be consecutive" % name)
        if rows <= 1:
            stride = cols
        elif output and stride < cols:
            raise TypeError("the rows of %s overlap" % name)
    else:
        if not shape or not t.is_contiguous():
            raise TypeError("%s must be two-dimensional or contiguous" % name)
        rows, stride, cols = math.prod(shape[:-1]), shape[-1], shape[-1]
    if rows >= 2 ** 31 or cols >= 2 ** 31:
        raise ValueError("the rows of %s, and their length, must fit a 32-bit int" % name)
    return stride, rows, cols


def _int32(t, name):
    if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise TypeError("%s must be a contiguous int32 CUDA tensor" % name)


# The current stream's handle; by way of a Stream object it takes 2 us.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name, device, *args):
    """The entry point on the current stream of the tensors' device."""
    fn = getattr(lib(), name)
    index = device.index
    if index == torch.cuda.current_device():
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            code = fn(*args, _raw_stream(index))
    if code:
        _check(code)


def _column(t, dtype, n, name):
    """A contiguous vector of one value a row."""
    if t.dtype != dtype or not t.is_cuda or not t.is_contiguous():
        raise TypeError("%s must be a contiguous %s CUDA tensor" % (name, dtype))
    if t.numel() != n:
        raise ValueError("%s must have one value a row" % name)
    return t


def _same_device(device, *tensors):
    for t in tensors:
        if t.device != device:
            raise ValueError("all tensors must be on one device")


def _out(out, shape, dtype):
    if out.dtype != dtype:
        raise TypeError("out must be a %s tensor" % dtype)
    if tuple(out.shape) != tuple(shape):
        raise ValueError("out must have the shape %s" % (tuple(shape),))
    return out


def embedding_lookup(table, ids, scale=1.0, out=None):
    """out[..., :] = scale * table[ids[...]] for an int32 tensor of ids.  Ids
    outside the table are padding and give zeros.  Nothing is recorded for
    autograd: embedding_grad is the gradient in the table."""
    _int32(ids, "ids")
    if table.dim() != 2:
        raise TypeError("table must be two-dimensional")
    stride, num_rows, dim = _rows_of(table, "table")
    count = _fits_int(ids.numel(), "the number of ids")
    if out is None:
        out = table.new_empty(tuple(ids.shape) + (dim,))
        out_stride = dim
    else:
        out = _out(out, tuple(ids.shape) + (dim,), table.dtype)
        out_stride, _, _ = _rows_of(out, "out", output=True)
    device = table.device
    _same_device(device, ids, out)
    _call("mgpu_hip_embedding_lookup", device, table.data_ptr(), num_rows, dim, stride,
          ids.data_ptr(), count, scale, out.data_ptr(), out_stride, _ROW_DTYPES[table.dtype])
    return out


def embedding_grad(grad, ids, num_rows=None, scale=1.0, out=None, accumulate=False):
    """The table's gradient from grad, one row per id: out[v] = scale * (sum
    of the grad rows whose id is v) for all num_rows rows, or, with
    accumulate, that added to the rows of out that occur.

    Give num_rows for a new tensor of grad's type, or out: (num_rows, dim) of
    grad's type or float32.  Ids outside the table add to nothing.  Sums are
    32-bit, in an order that the sizes and ids alone decide, and rounded once
    together with what out held."""
    _int32(ids, "ids")
    stride, count, dim = _rows_of(grad, "grad")
    if count != ids.numel():
        raise ValueError("grad must have one row per id")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        if num_rows is None:
            raise ValueError("num_rows or out must be given")
        out = grad.new_empty((num_rows, dim))
    if out.dtype != grad.dtype and out.dtype != torch.float32:
        raise TypeError("out must have grad's type or be float32")
    if out.dim() != 2 or out.shape[1] != dim or (num_rows is not None and out.shape[0] != num_rows):
        raise ValueError("out must be num_rows rows as long as grad's")
    out_stride, num_rows, _ = _rows_of(out, "out", output=True)
    device = grad.device
    _same_device(device, ids, out)
    nbytes = lib().mgpu_hip_embedding_grad_workspace_bytes(count, num_rows, dim)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _call("mgpu_hip_embedding_grad", device, grad.data_ptr(), stride, ids.data_ptr(), count,
          num_rows, dim, scale, 1 if accumulate else 0, out.data_ptr(), out_stride,
          _ROW_DTYPES[grad.dtype], _ROW_DTYPES[out.dtype], ws.data_ptr(), nbytes)
    return out


def _distill_args(logits, teacher_ids, teacher_logits, weights):
    stride, rows, vocab = _rows_of(logits, "logits")
    _int32(teacher_ids, "teacher_ids")
    if teacher_logits.dtype not in _ROW_DTYPES or not teacher_logits.is_cuda or not teacher_logits.is_contiguous():
        raise TypeError("teacher_logits must be a contiguous float32, float16 or bfloat16 CUDA tensor")
    if not teacher_ids.dim() or teacher_ids.shape != teacher_logits.shape or teacher_ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError("teacher_ids and teacher_logits must have a row for each row of logits")
    _same_device(logits.device, teacher_ids, teacher_logits)
    if weights is not None:
        _column(weights, torch.float32, rows, "weights")
        _same_device(logits.device, weights)
    return (logits.data_ptr(), stride, rows, vocab), (
        teacher_ids.data_ptr(), teacher_logits.data_ptr(), _fits_int(teacher_ids.shape[-1], "the number of entries")), (
        weights.data_ptr() if weights is not None else None), (
        _ROW_DTYPES[logits.dtype], _ROW_DTYPES[teacher_logits.dtype])


def _distill_out(out, logits):
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), logits.shape[-1]
    _out(out, logits.shape, logits.dtype)
    _same_device(logits.device, out)
    return out, _rows_of(out, "out", output=True)[0]


def distill_loss(logits, teacher_ids, teacher_logits, temperature=1.0, weights=None):
    """Loss of each row against the teacher's top logits: weight *
    temperature^2 * KL(softmax(teacher_logits / temperature) || softmax(logits
    / temperature)), the first over the entries whose id lies in the
    vocabulary (use -1 for padding).

    Returns ``(loss, norms)``, float32 with a value and with two values a row;
    ``distill_grad`` takes the norms.  Rows of weight 0, or without an entry
    that counts, have loss and norms 0, whatever their logits are.  Nothing is
    recorded for autograd: distill_grad is the gradient in the logits."""
    matrix, teacher, w, types = _distill_args(logits, teacher_ids, teacher_logits, weights)
    lead = logits.shape[:-1]
    loss = torch.empty(lead, dtype=torch.float32, device=logits.device)
    norms = torch.empty(tuple(lead) + (2,), dtype=torch.float32, device=logits.device)
    _call("mgpu_hip_distill_loss", logits.device, *matrix, *teacher, temperature, w,
          loss.data_ptr(), norms.data_ptr(), *types)
    return loss, norms


def distill_grad(logits, norms, teacher_ids, teacher_logits, weights=None, temperature=1.0, out=None):
    """The gradient of distill_loss's losses in the logits, times ``weights``:
    the loss's row weights times the gradient that arrives at each row's loss.
    ``out`` may be the logits themselves."""
    matrix, teacher, w, types = _distill_args(logits, teacher_ids, teacher_logits, weights)
    _column(norms, torch.float32, 2 * matrix[2], "norms")
    _same_device(logits.device, norms)
    out, out_stride = _distill_out(out, logits)
    _call("mgpu_hip_distill_grad", logits.device, *matrix, norms.data_ptr(), *teacher, temperature,
          w, out.data_ptr(), out_stride, *types)
    return out


def distill_loss_and_grad(logits, teacher_ids, teacher_logits, temperature=1.0, weights=None, out=None):
    """distill_loss and its gradient in one pass over the logits, for a
    training step whose row weights are known beforehand: ``(loss, grad)``,
    both with the weights in them.  ``out`` receives the gradient and may be
    the logits themselves."""
    matrix, teacher, w, types = _distill_args(logits, teacher_ids, teacher_logits, weights)
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=logits.device)
    out, out_stride = _distill_out(out, logits)
    _call("mgpu_hip_distill_loss_and_grad", logits.device, *matrix, *teacher, temperature, w,
          loss.data_ptr(), out.data_ptr(), out_stride, *types)
    return loss, out


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token a row: ``(token, logprob)``, int32 and float32.

    ``uniform`` holds one float32 in [0, 1) a row.  Each setting is a number,
    or a tensor with one value a row (float32; int32 for top_k).  top_k <= 0,
    top_p >= 1 and min_p <= 0 keep everything; temperature <= 0 takes the
    largest logit, the first of several; NaN settings count as 0 for the
    temperature, and as not given otherwise.  A row of nothing but -inf and NaN
    gives token -1 and logprob -inf."""
    if logits.dim() != 2:
        raise TypeError("logits must be two-dimensional")
    stride, rows, vocab = _rows_of(logits, "logits")
    device = logits.device
    _column(uniform, torch.float32, rows, "uniform")
    _same_device(device, uniform)
    pointers, values = [], []
    for value, dtype, name in ((temperature, torch.float32, "temperature"), (top_k, torch.int32, "top_k"),
                               (top_p, torch.float32, "top_p"), (min_p, torch.float32, "min_p")):
        if isinstance(value, torch.Tensor):
            _column(value, dtype, rows, name)
            _same_device(device, value)
            pointers.append(value.data_ptr())
            values.append(0)
        else:
            pointers.append(None)
            values.append(_fits_int(value, name) if dtype is torch.int32 else value)
    token = torch.empty(rows, dtype=torch.int32, device=device)
    logprob = torch.empty(rows, dtype=torch.float32, device=device)
    nbytes = lib().mgpu_hip_sample_workspace_bytes(rows, vocab)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _call("mgpu_hip_sample", device, logits.data_ptr(), stride, rows, vocab, uniform.data_ptr(),
          *pointers, *values, token.data_ptr(), logprob.data_ptr(), _ROW_DTYPES[logits.dtype],
          ws.data_ptr(), nbytes)
    return token, logprob
