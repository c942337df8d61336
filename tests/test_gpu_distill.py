"""Distillation from a teacher's top logits (gr_distill_topk) against float64 on the CPU.

Tolerances.  u_i = (z_i - max) / tau is formed in float32 (three roundings, |u| <= U), so each exp is off by a relative
3 U 2^-24 + 2^-22 (exp2's last bits) and a sum of n of them by as much plus n_depth * 2^-24 (per-thread sums of at most 2^9
terms plus trees: 2^10): r = (3 U + 1030) 2^-24.  Probabilities: relative 2 r + 2^-23 each, so the gradient is off by
|tau gl| (2 r q + (2 r + 2^-23) target) plus half a step of the stored type.  The loss sums p (log p - log q): log q is off by
r + 2^-22 |log q|."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import lowbit_reference as R                                                # noqa: E402
from graphite_amd import _hip                                               # noqa: E402
from graphite_amd.distill import teacher_top, topk_distill                  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _inputs(n, v, k, dtype, seed=0, shared=False, scale=2.5, tau=1.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn((n, v), generator=g) * scale).cuda().to(dtype)
    t = z[:1 if shared else n].float() * 0.6 + (torch.randn((1 if shared else n, v), generator=g) * 1.5).cuda()
    return z, teacher_top(t, k, tau), torch.rand(n, generator=g).cuda() + 0.1


def _compare(z, index, value, tau, lse, gl, loss, grad):
    zd = z.double().cpu().numpy()
    n, v = zd.shape
    rl, rg = R.distill(zd, index.cpu().numpy(), value.double().cpu().numpy(), tau, None if lse is None else lse.double().cpu().numpy(),
                       None if gl is None else gl.double().cpu().numpy())
    u = zd / tau
    U = np.array([np.ptp(r[np.isfinite(r)]) if np.isfinite(r).any() else 0.0 for r in u])
    r = (3 * U + 1030) * 2.0 ** -24
    g1 = np.ones(n) if gl is None else gl.double().cpu().numpy()
    with np.errstate(all="ignore"):
        q = np.exp(u - u.max(1, keepdims=True))
        q = q / q.sum(1, keepdims=True)
        lq = np.abs(np.log(np.maximum(q, 1e-300))).max(1)
    lerr = np.abs(loss.double().cpu().numpy() - rl)
    ltol = tau * tau * (2 * r + 2.0 ** -21 * (1 + U + np.log(v))) + np.abs(rl) * 2.0 ** -23
    assert (lerr <= ltol).all(), (lerr / ltol).max()
    if grad is not None:
        gd = grad.double().cpu().numpy()
        tg = tau * np.abs(g1)[:, None]
        eps = torch.finfo(z.dtype).eps
        target = np.abs(q - rg / (tau * g1[:, None]))
        gtol = tg * ((2 * r + 2.0 ** -22)[:, None] * (q + target)) + np.abs(rg) * eps / 2 * 1.01 + (2.0 ** -25 if z.dtype == F16 else 1e-37)
        gerr = np.abs(gd - rg)
        assert np.isfinite(gd).all()
        assert (gerr <= gtol).all(), (gerr / gtol).max()


SHAPES = [  # N, V, k
    (1, 1, 1), (1, 2, 2), (3, 43, 5), (100, 43, 43), (5, 63, 3), (4, 64, 7), (2, 65, 9), (17, 1000, 10), (1, 4097, 64),
    (3, 8191, 128), (2, 32768, 64), (2, 50001, 17), (1, 131072, 100), (9, 2049, 1024), (300, 129, 1),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rest", [False, True], ids=["closed", "open"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_matches_float64(shape, rest, dtype):
    n, v, k = shape
    i = SHAPES.index(shape)
    tau = (1.0, 2.0, 0.7)[i % 3]
    shared = i % 4 == 3
    z, top, gl = _inputs(n, v, k, dtype, i, shared, tau=tau)
    gl = gl if i % 2 else None
    lse = top.lse if rest else None
    loss, grad = topk_distill(z, top.index, top.value, tau, lse, gl)
    assert loss.dtype == F32 and grad.dtype == dtype and grad.shape == z.shape
    _compare(z, top.index, top.value, tau, lse, gl, loss, grad)
    only, none = topk_distill(z, top.index, top.value, tau, lse, want_grad=False)
    assert none is None and torch.equal(only, loss)


@pytest.mark.parametrize("rest", [False, True], ids=["closed", "open"])
@pytest.mark.parametrize("v", [43, 1000, 40001])
def test_empty_slots_repeated_classes_and_empty_rows(v, rest):
    z, top, gl = _inputs(6, v, 8, F32, 21)
    index, value = top.index.clone(), top.value.clone()
    index[0, 3:] = -1                                   # three of eight slots used
    index[1] = -1                                       # nothing
    index[2, 5] = index[2, 0]                           # a class named twice
    index[3, :] = index[3, 0]                           # one class, eight times
    value[3] -= 3.0                                     # (its probabilities add up to less than one)
    value[4, 2] = float("-inf")                         # a slot without mass
    if not rest:
        value[5] = float("-inf")
    value[0, 3:] = float("nan")                         # what an empty slot holds is not read into anything
    lse = top.lse if rest else None
    loss, grad = topk_distill(z, index, value, 1.0, lse, gl)
    _compare(z, index, value, 1.0, lse, gl, loss, grad)
    assert float(loss[1]) == 0.0 and not bool(grad[1].any())
    if not rest:
        assert float(loss[5]) == 0.0 and not bool(grad[5].any())


@pytest.mark.parametrize("rest", [False, True], ids=["closed", "open"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("v", [50, 5000])
def test_masked_student_logits(v, dtype, rest):
    """-inf and the type's lowest value among the student's unnamed classes: probability and gradient 0."""
    z, top, gl = _inputs(4, v, 4, dtype, 22)
    free = torch.ones((4, v), dtype=torch.bool, device="cuda").scatter_(1, top.index, False)
    z[0] = torch.where(free[0] & (torch.arange(v, device="cuda") % 2 == 0), torch.tensor(float("-inf"), device="cuda", dtype=dtype), z[0])
    z[1] = torch.where(free[1] & (torch.arange(v, device="cuda") % 3 == 0), torch.tensor(torch.finfo(dtype).min, device="cuda", dtype=dtype), z[1])
    z[2] = torch.where(free[2], torch.tensor(float("-inf"), device="cuda", dtype=dtype), z[2])      # nothing outside the named
    lse = top.lse if rest else None
    loss, grad = topk_distill(z, top.index, top.value, 1.0, lse, gl)
    zc = torch.where(z.float() < -1e30, torch.full_like(z, float("-inf")), z)
    _compare(zc, top.index, top.value, 1.0, lse, gl, loss, grad)
    assert not bool(grad[2][free[2]].any())


@pytest.mark.parametrize("v", [43, 3000])
def test_student_sure_of_the_named_classes(v):
    """The unnamed classes hold e^-60 of the student: q_rest keeps its digits (1 - sum q would be 0)."""
    z, top, _ = _inputs(3, v, 4, F32, 23)
    z = z.scatter_add(1, top.index, torch.full((3, 4), 60.0, device="cuda"))
    loss, grad = topk_distill(z, top.index, top.value, 1.0, top.lse)
    _compare(z, top.index, top.value, 1.0, top.lse, None, loss, grad)
    assert float(loss.min()) > 1.0


@pytest.mark.parametrize("v", [43, 3000])
def test_bad_values_stay_in_their_rows(v):
    z, top, gl = _inputs(6, v, 4, F32, 24)
    want_l, want_g = topk_distill(z, top.index, top.value, 1.0, top.lse, gl)
    index, z2 = top.index.clone(), z.clone()
    index[0, 1] = v
    index[1, 0] = -2
    index[2, 3] = 2 ** 40
    z2[3, v - 1] = float("nan")
    z2[4, 0] = float("inf")
    loss, grad = topk_distill(z2, index, top.value, 1.0, top.lse, gl)
    for i in range(5):
        assert bool(torch.isnan(loss[i])) and bool(torch.isnan(grad[i]).any())
    assert torch.equal(loss[5], want_l[5]) and torch.equal(grad[5], want_g[5])


@pytest.mark.parametrize("v", [43, 2500, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_strided_rows_in_place_and_untouched_surroundings(v, dtype):
    z, top, gl = _inputs(5, v, 6, dtype, 25)
    want_l, want_g = topk_distill(z, top.index, top.value, 1.0, top.lse, gl)
    for off, ld in ((0, v + (-v) % 8 + 8), (1, v + 3), (5, v + 6)):
        buf = torch.full((7, ld), 9.0, device="cuda", dtype=dtype)
        view = buf.as_strided((5, v), (ld, 1), ld + off)
        view.copy_(z)
        gbuf = torch.full((7, ld), 9.0, device="cuda", dtype=dtype)
        gview = gbuf.as_strided((5, v), (ld, 1), ld + off)
        loss, _ = topk_distill(view, top.index, top.value, 1.0, top.lse, gl, grad_out=gview)
        _compare(z, top.index, top.value, 1.0, top.lse, gl, loss, gview)
        loss2, _ = topk_distill(view, top.index, top.value, 1.0, top.lse, gl, grad_out=view)      # in place
        assert torch.equal(loss2, loss) and torch.equal(view, gview)
        view.fill_(9.0)
        gview.fill_(9.0)
        assert bool((buf == 9.0).all()) and bool((gbuf == 9.0).all())


@pytest.mark.parametrize("rest", [False, True], ids=["closed", "open"])
def test_gradient_is_the_difference_of_losses(rest):
    """Central differences of the 64-bit loss with a step of 2^-10: their own error is h^2/6 times the third derivative
    (at most 2 / tau for this loss) -- 4e-7 -- and the gradient's is the one of the file's header."""
    z, top, _ = _inputs(2, 43, 5, F32, 26, tau=2.0)
    lse = top.lse if rest else None
    _, grad = topk_distill(z, top.index, top.value, 2.0, lse)
    h = 2.0 ** -10
    zd = z.double().cpu().numpy()
    for i in range(43):
        d = np.zeros_like(zd)
        d[:, i] = h
        a = (top.index.cpu().numpy(), top.value.double().cpu().numpy(), 2.0, None if lse is None else lse.double().cpu().numpy())
        fd = (R.distill(zd + d, *a)[0] - R.distill(zd - d, *a)[0]) / (2 * h)
        assert np.abs(grad[:, i].double().cpu().numpy() - fd).max() <= 1e-6 + 4 * 1100 * 2.0 ** -24


def test_runs_agree_bit_for_bit_streams_and_graphs():
    cases = [_inputs(n, v, k, dt, 30) for n, v, k, dt in ((100, 43, 5, F32), (7, 9000, 20, BF16), (3, 70000, 64, F32))]
    want = [topk_distill(z, t.index, t.value, 1.0, t.lse, gl) for z, t, gl in cases]
    torch.cuda.synchronize()
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            got = [topk_distill(z, t.index, t.value, 1.0, t.lse, gl) for z, t, gl in cases]
        s.synchronize()
        for (l, g), (lw, gw) in zip(got, want):
            assert torch.equal(l, lw) and torch.equal(g, gw)
    for z, t, gl in cases:
        g = torch.empty_like(z)
        zs = z.clone()
        topk_distill(zs, t.index, t.value, 1.0, t.lse, gl, grad_out=g)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss, _ = topk_distill(zs, t.index, t.value, 1.0, t.lse, gl, grad_out=g)
        for i in range(3):
            zs.copy_(z.roll(i, 1))
            graph.replay()
            torch.cuda.synchronize()
            lw, gw = topk_distill(zs, t.index, t.value, 1.0, t.lse, gl)
            assert torch.equal(loss, lw) and torch.equal(g, gw)


def test_value_types_and_layouts():
    z, top, gl = _inputs(6, 300, 5, F32, 31)
    vb = top.value.to(BF16)
    loss, grad = topk_distill(z, top.index, vb, 1.0, None, gl)
    _compare(z, top.index, vb, 1.0, None, gl, loss, grad)
    l2, g2 = topk_distill(z, top.index.t().contiguous().t(), vb.t().contiguous().t(), 1.0, None, gl)
    assert torch.equal(l2, loss) and torch.equal(g2, grad)
    l3, _ = topk_distill(z[:1].expand(4, 300), top.index[0], vb[0], 1.0)
    assert l3.shape == (4,) and bool((l3 == l3[0]).all())
    e, ge = topk_distill(z[:0], top.index[:0], vb[:0], 1.0)
    assert e.shape == (0,) and ge.shape == (0, 300)


def test_refusals():
    z, top, gl = _inputs(4, 100, 5, F32, 32)
    E = _hip.GraphiteHipError
    a = (top.index, top.value)
    for bad in (lambda: topk_distill(z.cpu(), *a), lambda: topk_distill(z.double(), *a), lambda: topk_distill(z, *a, tau=0.0),
                lambda: topk_distill(z, *a, tau=-1.0), lambda: topk_distill(z, *a, tau=float("nan")), lambda: topk_distill(z, *a, tau=float("inf")),
                lambda: topk_distill(z, top.index.int(), top.value), lambda: topk_distill(z, top.index[:, :4], top.value),
                lambda: topk_distill(z, top.index[:3], top.value[:3]), lambda: topk_distill(z, *a, teacher_lse=top.lse[:2]),
                lambda: topk_distill(z, *a, teacher_lse=top.lse.double()), lambda: topk_distill(z, *a, grad_loss=gl[:1]),
                lambda: topk_distill(z, *a, grad_out=torch.empty(4, 99, device="cuda")),
                lambda: topk_distill(z, *a, grad_out=torch.empty(100, 4, device="cuda").t()),
                lambda: topk_distill(z, top.index.repeat(1, 300), top.value.repeat(1, 300)),
                lambda: topk_distill(z[:, :0], *a), lambda: topk_distill(z, top.index.cpu(), top.value)):
        with pytest.raises(E):
            bad()
    wide = torch.zeros((1, 2 ** 20 + 1), device="cuda")
    with pytest.raises(E):
        topk_distill(wide, torch.zeros((1, 1), dtype=torch.int64, device="cuda"), torch.zeros((1, 1), device="cuda"),
                     teacher_lse=torch.ones(1, device="cuda"))
    i, v = torch.tensor([[7]], device="cuda"), torch.zeros((1, 1), device="cuda")
    loss, grad = topk_distill(wide, i, v)
    assert abs(float(loss) - np.log(2 ** 20 + 1)) <= 1e-4 and abs(float(grad[0, 7]) + 1) <= 1e-5
    loss, grad = topk_distill(wide[:, 1:], i, v, teacher_lse=torch.full((1,), np.log(2.0), device="cuda"))
    assert abs(float(loss) - (0.5 * np.log(0.5 * 2 ** 20) + 0.5 * np.log(0.5))) <= 1e-4


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [43, 3000, 40001])
@pytest.mark.parametrize("case", ["nothing_unnamed_is_left", "named_mass_above_one"])
def test_gradient_where_the_target_does_not_add_up_to_one(case, v, dtype):
    """No p_rest enters the loss: every unnamed student logit is -inf, or the named p_j (of logits rounded to bfloat16, beside
    the float32 logsumexp of the unrounded ones) add up to more than 1.  Against the 64-bit gradient, and against central
    differences of the 64-bit loss: step 2^-10, their own error h^2 / 6 times the third derivative, at most 2 P, P < 2."""
    g = torch.Generator().manual_seed(27)
    n, k, tau = 3, 4, 1.0
    z = (torch.randn((n, v), generator=g) * 2.5).cuda()
    t = (torch.randn((n, v), generator=g) * 1.5).cuda()
    if case == "named_mass_above_one":
        hot = torch.tensor([[25.07, 25.19, 24.06, 23.07]], device="cuda")     # each goes up when rounded to bfloat16
        t[:, 5:9] = hot
    top = teacher_top(t, k, tau)
    value = top.value.to(BF16) if case == "named_mass_above_one" else top.value
    if case == "nothing_unnamed_is_left":
        named = torch.zeros((n, v), dtype=torch.bool, device="cuda").scatter_(1, top.index, True)
        z = torch.where(named, z, torch.full_like(z, float("-inf")))
    z = z.to(dtype)
    mass = torch.exp(value.double() / tau - top.lse.double()[:, None]).sum(1)
    assert bool((mass > 1.02).all()) if case == "named_mass_above_one" else bool((mass < 0.98).all())
    gl = torch.rand(n, generator=g).cuda() + 0.1
    loss, grad = topk_distill(z, top.index, value, tau, top.lse, gl)
    _compare(z, top.index, value, tau, top.lse, gl, loss, grad)
    zd, h = z.double().cpu().numpy(), 2.0 ** -10
    a = (top.index.cpu().numpy(), value.double().cpu().numpy(), tau, top.lse.double().cpu().numpy(), gl.double().cpu().numpy())
    gd = grad.double().cpu().numpy()
    scale = gl.double().cpu().numpy()
    for i in [int(top.index[0, 0]), int(top.index[0, 3])] + ([0, 9] if case == "named_mass_above_one" else []):
        d = np.zeros_like(zd)
        d[:, i] = h
        up, down = R.distill(zd + d, *a)[0], R.distill(zd - d, *a)[0]
        fd = np.where(np.isfinite(zd[:, i]), scale * (up - down) / (2 * h), 0.0)
        tol = scale * 2 * (1e-6 + 4 * 1100 * 2.0 ** -24) + np.abs(gd[:, i]) * torch.finfo(dtype).eps / 2
        assert (np.abs(gd[:, i] - fd) <= tol).all()


def test_rows_past_one_launch():
    """2^26 rows of two classes are more threads than one launch counts: every row as in a small batch."""
    n, t = 2 ** 26 + 1024, 1024
    z, top, _ = _inputs(t, 2, 1, F16, 33)
    want_l, want_g = topk_distill(z, top.index, top.value, 1.0, top.lse)
    loss, grad = topk_distill(z.repeat(n // t, 1), top.index.repeat(n // t, 1), top.value.repeat(n // t, 1), 1.0, top.lse.repeat(n // t))
    assert torch.equal(loss.view(-1, t), want_l.expand(n // t, t)) and torch.equal(grad.view(-1, t, 2), want_g.expand(n // t, t, 2))
    del loss, grad
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rest", [False, True], ids=["closed", "open"])
def test_loss_takes_part_in_autograd(rest, dtype):
    """backward() of the loss gives the gradient of the explicit form for the same grad_loss, bit for bit."""
    z, top, gl = _inputs(6, 300, 5, dtype, 41)
    lse = top.lse if rest else None
    want_l, want_g = topk_distill(z, top.index, top.value, 1.0, lse, gl)
    leaf = z.clone().requires_grad_(True)
    loss, grad = topk_distill(leaf, top.index, top.value, 1.0, lse, gl)
    assert loss.requires_grad and not grad.requires_grad and torch.equal(loss, want_l) and torch.equal(grad, want_g)
    (loss * gl).sum().backward()
    assert leaf.grad.dtype == dtype and torch.equal(leaf.grad, want_g)
    leaf.grad = None
    (2.0 * leaf).backward(topk_distill(2.0 * leaf.detach(), top.index, top.value, 1.0, lse)[1])     # the explicit form stays
    assert leaf.grad.shape == z.shape
    leaf.grad = None
    topk_distill(leaf, top.index, top.value, 1.0, lse, want_grad=False)[0].sum().backward()           # expanded gradient
    assert torch.equal(leaf.grad, topk_distill(z, top.index, top.value, 1.0, lse)[1])
    with torch.no_grad():
        assert not topk_distill(leaf, top.index, top.value, 1.0, lse)[0].requires_grad
    with pytest.raises(_hip.GraphiteHipError):
        topk_distill(leaf, top.index, top.value, 1.0, lse, grad_out=leaf)
    out = torch.empty_like(z)
    loss, grad = topk_distill(leaf, top.index, top.value, 1.0, lse, gl, grad_out=out)
    assert grad is out and loss.requires_grad and torch.equal(out, want_g)
    (g,) = torch.autograd.grad(loss.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_layer_and_loss_train_an_input_together():
    """The whitebox step written with torch.autograd: the 4-bit layer's logits, the loss, the gradient at the input; against the
    explicit chain."""
    from graphite_amd.linear_w4 import LinearW4, quantize
    g = torch.Generator().manual_seed(43)
    layer = LinearW4(*quantize(torch.randn((43, 256), generator=g) / 16, 64), group=64)
    x = torch.randn((20, 256), generator=g).cuda().requires_grad_(True)
    top = teacher_top(torch.randn((1, 43), generator=g).cuda() * 2, 5, 2.0)
    topk_distill(layer.forward(x), top.index, top.value, 2.0, top.lse)[0].mean().backward()
    _, gz = topk_distill(layer.forward(x.detach()), top.index, top.value, 2.0, top.lse, torch.full((20,), 1 / 20, device="cuda"))
    assert torch.equal(x.grad, layer.input_grad(gz))


@pytest.mark.parametrize("tau", [1.0, 20.0, 100.0, 1000.0, 1e4])
@pytest.mark.parametrize("k", [5, 43], ids=["open", "all-named"])
def test_loss_at_high_temperatures(k, tau):
    """Student and teacher nearly alike: the loss is tau^2 times a sum that all but cancels.  Open form: with one or no unnamed
    logit a lane, Sr is off by e = (3 U + 4 + 8) 2^-24 (three roundings of u, exp2's last bits, adding), the loss by
    tau^2 |q_rest - p_rest| e and, second order, tau^2 e^2; closed with every class named it holds no float sum.  Both: 64-bit
    arithmetic, tau^2 2^-46, and the rounding of the result."""
    z, top, _ = _inputs(8, 43, k, F32, 51, tau=tau)
    lse = top.lse if k < 43 else None
    loss, _ = topk_distill(z, top.index, top.value, tau, lse)
    zd, idx, val = z.double().cpu().numpy(), top.index.cpu().numpy(), top.value.double().cpu().numpy()
    ref, _ = R.distill(zd, idx, val, tau, None if lse is None else lse.double().cpu().numpy())
    tol = tau * tau * 2.0 ** -46 + np.abs(ref) * 2.0 ** -23
    if lse is not None:
        q = np.exp(zd / tau)
        q /= q.sum(1, keepdims=True)
        q_rest = 1 - np.take_along_axis(q, idx, 1).sum(1)
        p_rest = 1 - np.exp(val / tau - lse.double().cpu().numpy()[:, None]).sum(1)
        e = (3 * np.ptp(zd, axis=1) / tau + 12) * 2.0 ** -24
        tol = tol + tau * tau * (np.abs(q_rest - p_rest) * e + e * e)
    err = np.abs(loss.double().cpu().numpy() - ref)
    assert (err <= tol).all(), (err / tol).max()
