"""Distillation from a teacher's top logits (gr_distill_topk): the loss between a model's logits and an answer that consists
of a few scored classes -- a victim's top answers, or the full-precision model's for a quantised one -- with its gradient.

    top = teacher_top(teacher_logits, k=5, tau=2.0)              # TeacherTop(index, value, lse)
    loss, grad = topk_distill(logits, top.index, top.value, tau=2.0, teacher_lse=top.lse)

engine.eot_gradient(..., teacher=top) takes the whitebox step on it.
"""
from collections import namedtuple

import torch

from . import _hip

TeacherTop = namedtuple("TeacherTop", "index value lse tau")


def teacher_top(logits, k, tau=1.0, rest=True):
    """The k best classes of the teacher's logits [N, V] (CUDA): index [N, k], value [N, k] = their logits and, with `rest`,
    lse [N] = logsumexp(logits / tau), which tells how much the other classes hold (None: they hold nothing)."""
    value, index = torch.topk(logits.float(), min(int(k), logits.shape[-1]), dim=-1)
    return TeacherTop(index, value, torch.logsumexp(logits.double() / tau, dim=-1).float() if rest else None, float(tau))


def topk_distill(logits, index, value, tau=1.0, teacher_lse=None, grad_loss=None, want_grad=True, grad_out=None):
    """logits [N, V] (float32 / bfloat16 / float16, CUDA) against a teacher that names up to k classes per row:
    index int64 [N, k] (-1 = empty slot), value [N, k] = the teacher's logits; one row [1, k] (or [k]) serves the whole batch.
    teacher_lse [N] (float32; one element for one teacher row): logsumexp of all the teacher's logits / tau -- the mass it
    leaves over is compared with the student's outside the named classes; None: the named classes are all there is.
    Returns (loss float32 [N], grad [N, V] of logits' type = grad_loss[n] * d loss[n] / d logits[n], None without
    want_grad); grad_loss float32 [N] defaults to 1.  grad_out: optional result tensor, which may be `logits` itself."""
    z, ldz = _hip.float_rows(logits, "logits")
    dev = z.device
    n, v = z.shape
    if index.dim() == 1:
        index = index[None]
    if value.dim() == 1:
        value = value[None]
    if index.dtype != torch.int64:
        raise _hip.GraphiteHipError(f"index has type {index.dtype}, expected int64")
    if index.device != dev or index.dim() != 2 or index.shape != value.shape or index.shape[1] < 1:
        raise _hip.GraphiteHipError(f"index {tuple(index.shape)} and value {tuple(value.shape)} must be [N, k] tensors on {dev}")
    rows, k = index.shape
    shared = rows == 1
    if rows != n and not shared:
        raise _hip.GraphiteHipError(f"index has {rows} rows, expected {n} or 1")
    if value.device != dev or value.dtype not in _hip.DTYPES:
        raise _hip.GraphiteHipError(f"value must be a float32, bfloat16 or float16 tensor on {dev}")
    index, value = index.contiguous(), value.contiguous()
    for name, t, size in (("teacher_lse", teacher_lse, rows), ("grad_loss", grad_loss, n)):
        if t is not None and (t.device != dev or t.dtype != torch.float32 or t.numel() != size):
            raise _hip.GraphiteHipError(f"{name} must be a float32 tensor of {size} elements on {dev}")
    teacher_lse = None if teacher_lse is None else teacher_lse.contiguous()
    grad_loss = None if grad_loss is None else grad_loss.contiguous()
    loss = torch.empty((n,), device=dev, dtype=torch.float32)
    grad, ldg = None, v
    if grad_out is not None:
        grad, ldg = _hip.float_rows(grad_out, "grad_out", dev, v)
        if grad is not grad_out or grad.dtype != z.dtype or grad.shape[0] != n:
            raise _hip.GraphiteHipError(f"grad_out must be a {z.dtype} tensor [{n}, {v}] with the elements of a row next to each other")
    elif want_grad:
        grad = z.new_empty((n, v))
    _hip.op_call("gr_distill_topk", dev, z.data_ptr(), _hip.DTYPES[z.dtype], n, v, ldz, index.data_ptr(), value.data_ptr(),
                 _hip.DTYPES[value.dtype], k, 0 if shared else k, None if teacher_lse is None else teacher_lse.data_ptr(), float(tau),
                 None if grad_loss is None else grad_loss.data_ptr(), loss.data_ptr(), None if grad is None else grad.data_ptr(), ldg)
    return loss, grad
