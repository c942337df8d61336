"""Distillation from a teacher's top logits (gr_distill_topk): the loss between a model's logits and an answer that consists
of a few scored classes -- a victim's top answers, or the full-precision model's for a quantised one -- with its gradient.

    top = teacher_top(teacher_logits, k=5, tau=2.0)              # TeacherTop(index, value, lse)
    loss, grad = topk_distill(logits, top.index, top.value, tau=2.0, teacher_lse=top.lse)

engine.eot_gradient(..., teacher=top) takes the whitebox step on it.
"""
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

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
    dev, dt = z.device, z.dtype
    n, v = z.shape
    if index.dim() == 1:
        index = index[None]
    if value.dim() == 1:
        value = value[None]
    if index.dtype != torch.int64:
        raise _hip.GraphiteHipError(f"index has type {index.dtype}, expected int64")
    rows, k = index.shape if index.dim() == 2 else (0, 0)
    if index.device != dev or index.shape != value.shape or k < 1:
        raise _hip.GraphiteHipError(f"index {tuple(index.shape)} and value {tuple(value.shape)} must be [N, k] tensors on {dev}")
    if rows != n and rows != 1:
        raise _hip.GraphiteHipError(f"index has {rows} rows, expected {n} or 1")
    vt = _hip.DTYPES.get(value.dtype)
    if value.device != dev or vt is None:
        raise _hip.GraphiteHipError(f"value must be a float32, bfloat16 or float16 tensor on {dev}")
    index, value = index.contiguous(), value.contiguous()
    graph = z.requires_grad and torch.is_grad_enabled()
    if graph and grad_out is not None and grad_out.untyped_storage().data_ptr() == z.untyped_storage().data_ptr():
        raise _hip.GraphiteHipError("grad_out in the place of logits that require a gradient: pass logits.detach()")
    lse_p = gl_p = grad_p = None
    if teacher_lse is not None:
        teacher_lse = _vector(teacher_lse, "teacher_lse", rows, dev)
        lse_p = teacher_lse.data_ptr()
    if grad_loss is not None:
        grad_loss = _vector(grad_loss, "grad_loss", n, dev)
        gl_p = grad_loss.data_ptr()
    loss = torch.empty((n,), device=dev, dtype=torch.float32)
    grad, ldg = None, v
    if grad_out is not None:
        grad, ldg = _hip.float_rows(grad_out, "grad_out", dev, v)
        if grad is not grad_out or grad.dtype != dt or grad.shape[0] != n:
            raise _hip.GraphiteHipError(f"grad_out must be a {dt} tensor [{n}, {v}] with the elements of a row next to each other")
        grad_p = grad.data_ptr()
    elif want_grad:
        grad = z.new_empty((n, v))
        grad_p = grad.data_ptr()
    _hip.op_call("gr_distill_topk", dev, z.data_ptr(), _hip.DTYPES[dt], n, v, ldz, index.data_ptr(), value.data_ptr(), vt, k,
                 0 if rows == 1 else k, lse_p, float(tau), gl_p, loss.data_ptr(), grad_p, ldg)
    if graph:
        loss = _Loss.apply(z, loss, index, value, float(tau), teacher_lse)
    return loss, grad


class _Loss(torch.autograd.Function):
    """The loss of `z`, already computed, as a function of it."""

    @staticmethod
    def forward(ctx, z, loss, index, value, tau, lse):
        ctx.save_for_backward(z, index, value, lse)
        ctx.tau = tau
        return loss.view_as(loss)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        z, index, value, lse = ctx.saved_tensors
        return topk_distill(z, index, value, ctx.tau, lse, grad_loss)[1], None, None, None, None, None


def _vector(t, name, size, dev):
    if t.device != dev or t.dtype != torch.float32 or t.numel() != size:
        raise _hip.GraphiteHipError(f"{name} must be a float32 tensor of {size} elements on {dev}")
    return t.contiguous()
