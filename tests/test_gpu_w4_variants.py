"""Every kernel that gr_linear_w4 and gr_linear_w4_input_grad choose from, at the sizes of w4_cases.py (test_w4_host.py shows which
kernel each size takes), against float64 on the CPU: strided rows with NaN between them, strided results whose surroundings stay.

Tolerance, per output, as in test_gpu_w4.py: float32 sums of n terms n * 2^-23 * sum |x w| (the matrix unit may cut instead of
round), two-piece products 2^-15 * sum |gy w|, float32 ones 2^-23, and half a step of the stored type."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import lowbit_reference as R                                                # noqa: E402
import w4_cases                                                             # noqa: E402
from graphite_amd.linear_w4 import LinearW4                                 # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("case", w4_cases.FLAT, ids=w4_cases.label)
def test_kernel_matches_float64(case):
    kernel, grad, n, k, m, group, t = case
    dtype, half = DT[t.rstrip("*")], t.endswith("*")
    i = w4_cases.FLAT.index(case)
    g = torch.Generator().manual_seed(i)
    groups = -(-k // group)
    q = torch.randint(0, 256, (m, (k + 1) // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand((m, groups), generator=g) * 0.02 + 0.001).to((torch.float32, torch.bfloat16, torch.float16)[i % 3])
    z = torch.randint(0, 16, (m, groups), generator=g, dtype=torch.uint8) if i % 4 else None
    b = torch.randn(m, generator=g) if i % 2 else None
    w = R.weights(q.numpy(), s.double().numpy(), None if z is None else z.numpy(), group, k)
    layer = LinearW4(q.cuda(), s.cuda(), None if z is None else z.cuda(), None if b is None else b.cuda(), group=group, in_features=k)
    c, r = (m, k) if grad else (k, m)
    ld = c if dtype == torch.float32 else c + (c + half) % 2
    buf = torch.full((n * ld + 16,), float("nan"), device="cuda", dtype=dtype)
    x = buf.as_strided((n, c), (ld, 1), 1 if half else 0)
    x.copy_(torch.randn((n, c), generator=g))
    obuf = torch.full((n + 2, r + 5), 7.0, device="cuda", dtype=dtype)
    out = obuf[1:n + 1, 3:3 + r]
    xd = x.double().cpu().numpy()
    relu = i % 5 == 1
    if grad:
        gate = torch.randn((n, k), generator=g).to("cuda", dtype) if i % 2 else None
        layer.input_grad(x, gate=gate, out=out)
        ref, mag = R.input_grad(xd, w, None if gate is None else gate.double().cpu().numpy()), np.abs(xd) @ np.abs(w)
        extra = 2.0 ** -23 if dtype == torch.float32 else 2.0 ** -15
    else:
        layer.forward(x, relu=relu, out=out)
        bd = None if b is None else b.double().numpy()
        ref, mag = R.linear(xd, w, bd, relu), np.abs(xd) @ np.abs(w).T + (0 if b is None else np.abs(bd))
        extra = 0.0
    tol = mag * ((c + 1) * 2.0 ** -23 + extra) * 1.01 + np.abs(ref) * torch.finfo(dtype).eps / 2 * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.isfinite(err).all() and (err <= tol).all(), f"{np.nanmax(err / tol):.3g} of the tolerance"
    out.fill_(7.0)
    assert bool((obuf == 7.0).all())
