"""Linear layers with 4-bit weights and group scales (gr_linear_w4): what a victim deployed on a small device runs.

    q, scales, zeros = quantize(w, group=64)                  # or from a 4-bit checkpoint
    layer = LinearW4(q, scales, zeros, bias=b, group=64)
    y  = layer.forward(x, relu=True)                          # [N, out]
    gx = layer.input_grad(gy)                                 # d loss / d x, for the whitebox loops

float32, bfloat16 and float16 activations; every product is exact, every sum float32, the result is rounded once.
Where x requires a gradient, y takes part in torch.autograd (once differentiable; the weights and the bias are frozen).
models.GTSRBNet.set_linear_w4 runs a victim's fully connected layers this way.
"""
import ctypes as C

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from . import _hip


def quantize(w, group=64, symmetric=False):
    """Round-to-nearest 4-bit weights of w [out, in] (array or tensor, any float type): (q, scales, zeros) CPU tensors --
    q uint8 [out, ceil(in/2)] (input 2j in the low, 2j+1 in the high nibble), scales float32 [out, G], zeros uint8 [out, G],
    None when symmetric (zero point 8).  Groups of `group` consecutive inputs; a weight's error is at most half its group's
    scale.  Asymmetric groups span [min(w, 0), max(w, 0)] in 15 steps, symmetric ones [-max|w|, max|w|] in 14."""
    if group <= 0 or group % 32:
        raise ValueError(f"group {group} is not a positive multiple of 32")
    w = np.asarray(w.detach().cpu().float().numpy() if isinstance(w, torch.Tensor) else w, dtype=np.float64)
    if w.ndim != 2 or not w.size:
        raise ValueError(f"weights have shape {w.shape}, expected [out, in]")
    if not np.isfinite(w).all():
        raise ValueError("weights must be finite")
    m, k = w.shape
    groups = -(-k // group)
    g = np.zeros((m, groups * group))
    g[:, :k] = w
    g = g.reshape(m, groups, group)
    if symmetric:
        span, steps = np.abs(g).max(2), 7.0
        zeros = None
    else:
        lo, hi = np.minimum(g.min(2), 0.0), np.maximum(g.max(2), 0.0)
        span, steps = hi - lo, 15.0
    scales = (span / steps).astype(np.float32)
    scales[scales == 0] = 1.0                                  # a group of zeros
    s64 = scales.astype(np.float64)
    z = np.full_like(s64, 8.0) if symmetric else np.clip(np.rint(-lo / s64), 0, 15)
    q = np.clip(np.rint(g / s64[:, :, None]) + z[:, :, None], 0, 15).astype(np.uint8).reshape(m, -1)[:, :k]
    if k % 2:
        q = np.concatenate([q, np.zeros((m, 1), np.uint8)], 1)
    packed = q[:, 0::2] | (q[:, 1::2] << 4)
    return (torch.from_numpy(np.ascontiguousarray(packed)), torch.from_numpy(scales),
            None if symmetric else torch.from_numpy(z.astype(np.uint8)))


def dequantize(q, scales, zeros=None, group=64, in_features=None):
    """float32 [out, in] weights (q - z) * s of quantize()'s (or a checkpoint's) tensors, on their device."""
    k = 2 * q.shape[1] if in_features is None else int(in_features)
    codes = torch.stack((q & 15, q >> 4), dim=2).reshape(q.shape[0], -1)[:, :k].float()
    grp = torch.arange(k, device=q.device) // group
    z = 8.0 if zeros is None else zeros.float()[:, grp]
    return (codes - z) * scales.float()[:, grp]


class _Forward(torch.autograd.Function):
    """layer.forward(x, relu) of [rows, in], differentiable w.r.t. x (gr_linear_w4_input_grad)."""

    @staticmethod
    def forward(ctx, x, layer, relu):
        y = layer.forward(x, relu=relu)
        ctx.layer, ctx.relu = layer, relu
        if relu:
            ctx.save_for_backward(y)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        if ctx.relu:
            grad_y = grad_y.masked_fill(ctx.saved_tensors[0] <= 0, 0)
        return ctx.layer.input_grad(grad_y), None, None


class LinearW4:
    """gr_w4 handle: the weights laid out for the matrix units on one device.  q uint8 [out, ceil(in/2)], scales [out, G]
    (float32 / bfloat16 / float16, finite), zeros uint8 [out, G] or None, bias [out] or None; CPU tensors are moved to
    `device` (default: q's, or the current one).  in_features: the true number of inputs when it is odd.
    input_grad=False drops the transposed copy that `input_grad` reads (half the memory).  The object's memory must outlive
    what was captured with it: keep it as long as a HIP graph replays its calls."""

    def __init__(self, q, scales, zeros=None, bias=None, group=64, in_features=None, input_grad=True, device=None):
        self._h = C.c_void_p()
        if q.dtype != torch.uint8 or q.dim() != 2:
            raise _hip.GraphiteHipError("q must be a uint8 tensor [out, ceil(in/2)]")
        if zeros is not None and zeros.dtype != torch.uint8:
            raise _hip.GraphiteHipError(f"zeros has type {zeros.dtype}, expected uint8 (or None)")
        if scales.dtype not in _hip.DTYPES:
            raise _hip.GraphiteHipError(f"scales has type {scales.dtype}; float32, bfloat16 and float16 are supported")
        k = 2 * q.shape[1] if in_features is None else int(in_features)
        if group <= 0 or group % 32:
            raise _hip.GraphiteHipError(f"group {group} is not a positive multiple of 32")
        if k <= 0 or q.shape[0] <= 0 or q.shape[1] != (k + 1) // 2:
            raise _hip.GraphiteHipError(f"q has shape {tuple(q.shape)}, expected [out, {(k + 1) // 2}] for {k} inputs")
        want = (q.shape[0], -(-k // group))
        for name, t in (("scales", scales), ("zeros", zeros)):
            if t is not None and tuple(t.shape) != want:
                raise _hip.GraphiteHipError(f"{name} has shape {tuple(t.shape)}, expected {want}")
        if bias is not None and tuple(bias.shape) != (q.shape[0],):
            raise _hip.GraphiteHipError(f"bias has shape {tuple(bias.shape)}, expected ({q.shape[0]},)")
        if device is None:
            device = q.device if q.is_cuda else torch.device("cuda", _hip.device_index())
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise _hip.GraphiteHipError("LinearW4 lives on a ROCm device; graphite_amd has no CPU path")
        if self.device.index is None:
            self.device = torch.device("cuda", _hip.device_index())
        self.out_features, self.in_features, self.group = int(q.shape[0]), k, int(group)
        q, scales = q.to(self.device).contiguous(), scales.to(self.device).contiguous()
        zeros = None if zeros is None else zeros.to(self.device).contiguous()
        bias = None if bias is None else bias.to(self.device, torch.float32).contiguous()
        _hip.op_call("gr_w4_create", self.device, q.data_ptr(), q.shape[1], scales.data_ptr(), _hip.DTYPES[scales.dtype], want[1],
                     zeros.data_ptr() if zeros is not None else None, want[1], bias.data_ptr() if bias is not None else None,
                     self.out_features, k, self.group, int(bool(input_grad)), out=self._h)

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and _hip._lib is not None:
            _hip._lib.gr_w4_destroy(h)

    def _rows_of(self, out, n, cols, like):
        """Row stride of a caller's result tensor, after its checks."""
        if out.device != self.device or out.dtype != like.dtype or tuple(out.shape) != (n, cols):
            raise _hip.GraphiteHipError(f"out must be a {like.dtype} tensor [{n}, {cols}] on {self.device}")
        if (cols > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < cols):
            raise _hip.GraphiteHipError("out: the elements of a row must be next to each other")
        return out.stride(0) if n > 1 else cols

    def forward(self, x, relu=False, out=None):
        """x [..., in] -> [..., out] of x's type on the current stream; relu clamps negative results to 0.  Rows of x may be
        any distance apart.  out: optional result tensor [rows, out], which must not overlap x and takes no part in
        torch.autograd."""
        lead = None
        if x.dim() != 2:
            lead = x.shape[:-1]
            x = x.reshape(-1, x.shape[-1])
        x, ldx = _hip.float_rows(x, "x", self.device, self.in_features)
        n, m = x.shape[0], self.out_features
        if x.requires_grad and torch.is_grad_enabled():
            if out is not None:
                raise _hip.GraphiteHipError("out= takes no part in torch.autograd, and x requires a gradient: pass x.detach(), or no out")
            y = _Forward.apply(x, self, relu)
            return y if lead is None else y.view(*lead, m)
        if out is None:
            y, ldy = x.new_empty((n, m)), m
        else:
            y, ldy = out, self._rows_of(out, n, m, x)
        _hip.op_call("gr_linear_w4", self.device, self._h, x.data_ptr(), _hip.DTYPES[x.dtype], n, ldx, 1 if relu else 0, y.data_ptr(), ldy)
        return y if out is not None or lead is None else y.view(*lead, m)

    __call__ = forward

    def input_grad(self, grad_y, gate=None, out=None):
        """grad_y [..., out] -> d loss / d x [..., in] of its type; 0 where gate <= 0 (gate: the rectified activation the
        layer read, shape of the result).  A ReLU of this layer is the caller's to apply to grad_y.  out: as forward's.
        The result is a plain tensor: it carries no graph, whatever grad_y requires."""
        lead = None
        if grad_y.dim() != 2:
            lead = grad_y.shape[:-1]
            grad_y = grad_y.reshape(-1, grad_y.shape[-1])
        g, ldg = _hip.float_rows(grad_y, "grad_y", self.device, self.out_features)
        n, k = g.shape[0], self.in_features
        gp, ldgate = None, k
        if gate is not None:
            if gate.dtype != g.dtype:
                raise _hip.GraphiteHipError(f"gate has type {gate.dtype}, expected {g.dtype}")
            gate, ldgate = _hip.float_rows(gate.reshape(-1, gate.shape[-1]), "gate", self.device, k)
            if gate.shape[0] != n:
                raise _hip.GraphiteHipError(f"gate has {gate.shape[0]} rows, expected {n}")
            gp = gate.data_ptr()
        if out is None:
            gx, ldgx = g.new_empty((n, k)), k
        else:
            gx, ldgx = out, self._rows_of(out, n, k, g)
        _hip.op_call("gr_linear_w4_input_grad", self.device, self._h, g.data_ptr(), _hip.DTYPES[g.dtype], n, ldg, gp, ldgate,
                     gx.data_ptr(), ldgx)
        return gx if out is not None or lead is None else gx.view(*lead, k)
