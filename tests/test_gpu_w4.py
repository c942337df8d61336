"""4-bit linear layers (gr_linear_w4, gr_linear_w4_input_grad) against float64 on the CPU.

Tolerance, per output: products are exact and sums float32, so a sum of n terms is off by at most n * 2^-23 * sum |x w|
(2^-23: the matrix unit may cut instead of round); two-piece products of the 16-bit gradients add 2^-15 * sum |gy w|, the
float32 product gy * s 2^-24; the stored result adds half a step of its type, |y| * eps / 2 (below float16's normal range
2^-25)."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import lowbit_reference as R                                                # noqa: E402
from graphite_amd import _hip                                               # noqa: E402
from graphite_amd.linear_w4 import LinearW4, dequantize, quantize           # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _layer(m, k, group, sdt=F32, zeros=True, bias=False, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (m, (k + 1) // 2), generator=g, dtype=torch.uint8)      # an odd row's last nibble is garbage
    groups = -(-k // group)
    s = (torch.rand((m, groups), generator=g) * 0.02 + 0.001).to(sdt)
    z = torch.randint(0, 16, (m, groups), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(m, generator=g) if bias else None
    w = R.weights(q.numpy(), s.double().numpy(), None if z is None else z.numpy(), group, k)
    return LinearW4(q.to(device), s.to(device), None if z is None else z.to(device), None if b is None else b.to(device),
                    group=group, in_features=k), w, None if b is None else b.double().numpy()


def _tol(ref, mag, terms, dtype, extra=0.0):
    eps = torch.finfo(dtype).eps
    return mag * (terms * 2.0 ** -23 + extra) * 1.01 + np.abs(ref) * eps / 2 * 1.01 + (2.0 ** -25 if dtype == F16 else 1e-37)


def _check(got, ref, tol):
    err = np.abs(got.double().cpu().numpy() - ref)
    assert np.isfinite(err).all()
    assert (err <= tol).all(), f"{(err / tol).max():.3g} of the tolerance at {np.unravel_index((err / tol).argmax(), err.shape)}"


def _check_forward(layer, w, b, x, relu):
    y = layer.forward(x, relu=relu)
    assert y.dtype == x.dtype and tuple(y.shape) == (x.shape[0], w.shape[0])
    xd = x.double().cpu().numpy()
    ref = R.linear(xd, w, b, relu)
    mag = np.abs(xd) @ np.abs(w).T + (0 if b is None else np.abs(b))
    _check(y, ref, _tol(ref, mag, w.shape[1] + 64, x.dtype))


def _check_grad(layer, w, gy, gate=None):
    gx = layer.input_grad(gy, gate=gate)
    assert gx.dtype == gy.dtype and tuple(gx.shape) == (gy.shape[0], w.shape[1])
    gd = gy.double().cpu().numpy()
    ref = R.input_grad(gd, w, None if gate is None else gate.double().cpu().numpy())
    _check(gx, ref, _tol(ref, np.abs(gd) @ np.abs(w), w.shape[0] + 64, gy.dtype, 2.0 ** -23 if gy.dtype == F32 else 2.0 ** -15))


SHAPES = [  # N, K, M, group
    (1, 1, 1, 32), (1, 32, 16, 32), (2, 31, 17, 32), (1, 2048, 1024, 64), (7, 129, 43, 64), (15, 257, 15, 128),
    (16, 128, 128, 128), (17, 96, 130, 96), (33, 1000, 129, 160), (100, 2048, 1024, 64), (129, 321, 300, 32),
    (130, 640, 257, 128), (300, 1024, 43, 64), (1, 5001, 33, 32), (3, 100, 1000, 1024), (257, 511, 385, 256), (600, 64, 10, 32),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_forward_and_gradient_match_float64(shape, dtype):
    n, k, m, group = shape
    i = SHAPES.index(shape)
    sdt = (F32, dtype, F16)[i % 3]
    layer, w, b = _layer(m, k, group, sdt, zeros=i % 2 == 0, bias=i % 3 != 1, seed=i)
    g = torch.Generator().manual_seed(100 + i)
    _check_forward(layer, w, b, torch.randn((n, k), generator=g).to("cuda", dtype), relu=i % 4 == 3)
    gate = torch.randn((n, k), generator=g).to("cuda", dtype) if i % 2 else None
    _check_grad(layer, w, torch.randn((n, m), generator=g).to("cuda", dtype), gate)


# More outputs than the few-row kernels take (12288 tiles of 16 x 16): the LDS-tiled kernel, with contractions of less than a
# stage, of whole stages, with a ragged end, and groups that end inside, at and across its 64-step stages.
MANY = [(1, 32), (31, 64), (64, 32), (64, 128), (129, 96), (200, 64), (320, 32), (321, 128), (512, 256), (385, 160), (450, 1024)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("depth,group", MANY, ids=["x".join(map(str, s)) for s in MANY])
def test_many_rows_match_float64(depth, group, dtype):
    i = MANY.index((depth, group))
    g = torch.Generator().manual_seed(200 + i)
    n, wide = 2100, 1610
    layer, w, b = _layer(wide, depth, group, (F32, dtype, F16)[i % 3], zeros=i % 2 == 0, bias=i % 3 != 1, seed=50 + i)
    _check_forward(layer, w, b, torch.randn((n, depth), generator=g).to("cuda", dtype), relu=i % 4 == 3)
    layer, w, _ = _layer(depth, wide, group, (F32, dtype, F16)[i % 3], zeros=i % 2 == 0, seed=70 + i)
    gate = torch.randn((n, wide), generator=g).to("cuda", dtype) if i % 2 else None
    _check_grad(layer, w, torch.randn((n, depth), generator=g).to("cuda", dtype), gate)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_many_strided_rows(dtype):
    n, k, m = 2060, 1700, 1605                             # 129 x 107 and 129 x 101 tiles
    layer, w, b = _layer(m, k, 64, bias=True, seed=3)
    x = torch.full((n + 1, k + 3), float("nan"), device="cuda", dtype=dtype).as_strided((n, k), (k + 3, 1), 1)
    x.copy_(torch.randn((n, k), generator=torch.Generator().manual_seed(5)))
    obuf = torch.full((n + 2, m + 6), 7.0, device="cuda", dtype=dtype)
    layer.forward(x, out=obuf[1:n + 1, 3:3 + m])
    xd = x.double().cpu().numpy()
    ref = R.linear(xd, w, b)
    _check(obuf[1:n + 1, 3:3 + m], ref, _tol(ref, np.abs(xd) @ np.abs(w).T + np.abs(b), k + 64, dtype))
    obuf[1:n + 1, 3:3 + m] = 7.0
    assert bool((obuf == 7.0).all())
    gy = torch.full((n + 1, m + 9), float("inf"), device="cuda", dtype=dtype).as_strided((n, m), (m + 9, 1), 3)
    gy.copy_(torch.randn((n, m), generator=torch.Generator().manual_seed(6)))
    xbuf = torch.full((n + 2, k + 5), 7.0, device="cuda", dtype=dtype)
    layer.input_grad(gy, out=xbuf[1:n + 1, 2:2 + k])
    gd = gy.double().cpu().numpy()
    ref = R.input_grad(gd, w)
    _check(xbuf[1:n + 1, 2:2 + k], ref, _tol(ref, np.abs(gd) @ np.abs(w), m + 64, dtype, 2.0 ** -15))
    xbuf[1:n + 1, 2:2 + k] = 7.0
    assert bool((xbuf == 7.0).all())


def test_many_rows_runs_agree_and_replay():
    layer, w, b = _layer(1610, 330, 64, bias=True, seed=13)
    wide, _, _ = _layer(330, 1610, 64, seed=14)
    x = torch.zeros((2100, 330), device="cuda", dtype=BF16)
    y, gx = torch.empty((2100, 1610), device="cuda", dtype=BF16), torch.empty((2100, 1610), device="cuda", dtype=BF16)
    layer.forward(x, out=y)
    wide.input_grad(x, out=gx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(x, relu=True, out=y)
        wide.input_grad(x, gate=y, out=gx)
    for i in range(3):
        x.copy_(torch.randn((2100, 330), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        yw = layer.forward(x, relu=True)
        assert torch.equal(y, yw) and torch.equal(gx, wide.input_grad(x, gate=yw))
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_strided_rows_and_untouched_surroundings(n, dtype):
    k, m = 200, 75
    layer, w, b = _layer(m, k, 64, bias=True, seed=3)
    for off, ld in ((0, 256), (1, 203), (3, 201)):          # aligned rows, odd rows, rows that start off a 16-byte border
        buf = torch.full((n + 1, ld), float("nan"), device="cuda", dtype=dtype)
        x = buf.as_strided((n, k), (ld, 1), off)
        x.copy_(torch.randn((n, k), generator=torch.Generator().manual_seed(n)))
        obuf = torch.full((n + 2, m + 6), 7.0, device="cuda", dtype=dtype)
        out = obuf[1:n + 1, 2:2 + m]
        assert layer.forward(x, out=out) is out
        xd = x.double().cpu().numpy()
        ref = R.linear(xd, w, b)
        _check(out, ref, _tol(ref, np.abs(xd) @ np.abs(w).T + np.abs(b), k + 64, dtype))
        keep = obuf.clone()
        keep[1:n + 1, 2:2 + m] = 7.0
        assert bool((keep == 7.0).all())
        gbuf = torch.full((n + 1, m + 9), float("inf"), device="cuda", dtype=dtype)
        gy = gbuf.as_strided((n, m), (m + 9, 1), off)
        gy.copy_(torch.randn((n, m), generator=torch.Generator().manual_seed(n + 1)))
        xbuf = torch.full((n + 2, k + 5), 7.0, device="cuda", dtype=dtype)
        gx = xbuf[1:n + 1, 3:3 + k]
        layer.input_grad(gy, out=gx)
        gd = gy.double().cpu().numpy()
        ref = R.input_grad(gd, w)
        _check(gx, ref, _tol(ref, np.abs(gd) @ np.abs(w), m + 64, dtype, 2.0 ** -15))
        xbuf[1:n + 1, 3:3 + k] = 7.0
        assert bool((xbuf == 7.0).all())


def test_views_that_are_not_rows_are_copied():
    layer, w, b = _layer(40, 96, 32, seed=5)
    x = torch.randn(96, 20, device="cuda")
    _check_forward(layer, w, b, x.t(), False)
    _check_forward(layer, w, b, torch.randn(1, 96, device="cuda").expand(9, 96), False)
    y = layer.forward(torch.randn(2, 3, 96, device="cuda"))
    assert tuple(y.shape) == (2, 3, 40)
    assert tuple(layer.forward(torch.empty(0, 96, device="cuda")).shape) == (0, 40)
    assert tuple(layer.input_grad(torch.empty(0, 40, device="cuda")).shape) == (0, 96)
    assert tuple(layer.forward(torch.randn(96, device="cuda")).shape) == (40,)


@pytest.mark.parametrize("n", [3, 40, 300, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_infinities_stay_in_their_rows(dtype, n):
    """x[i,k] = inf gives +-inf by the sign of the weight and NaN for a weight of 0, as the formula says; other rows keep
    their values bit for bit.  A gradient row with an infinity is nowhere finite."""
    layer, w, b = _layer(70, 130, 32, seed=8)
    x = torch.randn((n, 130), generator=torch.Generator().manual_seed(1)).to("cuda", dtype)
    base = layer.forward(x)
    x2 = x.clone()
    x2[1, 129] = float("inf")
    x2[2, 64] = float("nan")
    y = layer.forward(x2)
    want = torch.from_numpy(np.where(w[:, 129] > 0, np.inf, np.where(w[:, 129] < 0, -np.inf, np.nan)))
    assert torch.equal(torch.nan_to_num(y[1].double().cpu(), nan=1.0), torch.nan_to_num(want, nan=1.0))
    assert bool(torch.isnan(y[2]).all())
    keep = [i for i in range(n) if i not in (1, 2)]
    assert torch.equal(y[keep], base[keep])
    gy = torch.randn((n, 70), generator=torch.Generator().manual_seed(2)).to("cuda", dtype)
    gbase = layer.input_grad(gy)
    gy2 = gy.clone()
    gy2[1, 69] = float("-inf")
    gy2[2, 3] = float("nan")
    gx = layer.input_grad(gy2)
    assert not bool(torch.isfinite(gx[1]).any()) and bool(torch.isnan(gx[2]).all())
    assert torch.equal(gx[keep], gbase[keep])


@pytest.mark.parametrize("n", [2, 300, 40000])
def test_float32_extremes(n):
    """Activations near both ends of float32's range: the three-piece cut neither overflows nor loses its low pieces."""
    layer, w, b = _layer(33, 64, 32, zeros=False, seed=9)
    for scale in (2.0 ** 120, 2.0 ** -90):
        x = (torch.rand((n, 64), generator=torch.Generator().manual_seed(4)) + 0.5).cuda() * scale
        _check_forward(layer, w, b, x, False)


@pytest.mark.parametrize("n", [1, 20, 300])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_gradient_is_the_forward_difference(n, dtype):
    """The layer is linear: <gy, f(x + d) - f(x - d)> / 2 = <gx, d> up to the roundings of both sides (64-bit inner
    products; float32 forward)."""
    layer, w, b = _layer(150, 260, 64, bias=True, seed=11)
    g = torch.Generator().manual_seed(7)
    x, d = torch.randn((n, 260), generator=g).cuda(), torch.randn((n, 260), generator=g).cuda()
    gy = torch.randn((n, 150), generator=g).cuda().to(dtype)
    diff = (layer.forward(x + d).double() - layer.forward(x - d).double()) / 2
    left, right = float((gy.double() * diff).sum()), float((layer.input_grad(gy).double() * d.double()).sum())
    mag = (gy.double().abs().cpu().numpy() * ((np.abs((x + d).cpu().numpy()) + np.abs((x - d).cpu().numpy())) / 2 @ np.abs(w).T
                                             + np.abs(b))).sum()
    gmag = ((gy.double().abs().cpu().numpy() @ np.abs(w)) * np.abs(d.cpu().numpy())).sum()
    assert abs(left - right) <= mag * 330 * 2.0 ** -23 + gmag * (220 * 2.0 ** -23 + torch.finfo(dtype).eps / 2 + 2.0 ** -15)


def test_runs_agree_bit_for_bit_and_streams_do_not_mix():
    layer, w, b = _layer(300, 700, 64, bias=True, seed=12)
    xs = [torch.randn((n, 700), device="cuda") for n in (1, 64, 400)]
    want = [layer.forward(x) for x in xs]
    gw = [layer.input_grad(y) for y in want]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s in (s1, s2):
        with torch.cuda.stream(s):
            got.append([(layer.forward(x), layer.input_grad(y)) for x, y in zip(xs, want)])
    torch.cuda.synchronize()
    for ys in got:
        for (y, g), yw, gww in zip(ys, want, gw):
            assert torch.equal(y, yw) and torch.equal(g, gww)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_captured_graph_replays(n):
    layer, w, b = _layer(200, 330, 64, bias=True, seed=13)
    x = torch.zeros((n, 330), device="cuda", dtype=BF16)
    y, gx = torch.empty((n, 200), device="cuda", dtype=BF16), torch.empty((n, 330), device="cuda", dtype=BF16)
    layer.forward(x, out=y)
    layer.input_grad(y, out=gx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(x, relu=True, out=y)
        layer.input_grad(y, gate=x, out=gx)
    for i in range(4):
        x.copy_(torch.randn((n, 330), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        yw = layer.forward(x, relu=True)
        assert torch.equal(y, yw) and torch.equal(gx, layer.input_grad(yw, gate=x))
        torch.cuda.synchronize()


def test_quantize_bounds_and_dequantize():
    g = torch.Generator().manual_seed(0)
    w = torch.randn((50, 131), generator=g) * torch.rand((50, 1), generator=g)
    w[3] = 0
    w[4, :64] = w[4, :64].abs() + 1                                          # a group away from zero
    for sym in (False, True):
        q, s, z = quantize(w, 64, sym)
        back = R.weights(q.numpy(), s.numpy(), None if z is None else z.numpy(), 64, 131)
        step = s.double().numpy()[:, np.arange(131) // 64]
        # rounding: half a step; asymmetric: the zero point is rounded too
        assert (np.abs(back - w.double().numpy()) <= step * (0.5 if sym else 1.0) * 1.0001).all()
        dq = dequantize(q.cuda(), s.cuda(), None if z is None else z.cuda(), 64, 131)
        assert np.abs(dq.cpu().double().numpy() - back).max() <= 2.0 ** -24 * np.abs(back).max()
        layer = LinearW4(q, s, z, group=64, in_features=131)
        _check_forward(layer, back, None, torch.randn((5, 131), device="cuda"), False)


def test_refusals():
    layer, _, _ = _layer(16, 64, 32)
    E = _hip.GraphiteHipError
    q, s = torch.zeros((16, 32), dtype=torch.uint8, device="cuda"), torch.ones((16, 2), device="cuda")
    for bad in (lambda: LinearW4(q, s, group=48), lambda: LinearW4(q, s, group=0), lambda: LinearW4(q, s, group=64),
                lambda: LinearW4(q.int(), s, group=32), lambda: LinearW4(q, s.double(), group=32),
                lambda: LinearW4(q, s, s, group=32), lambda: LinearW4(q, s, group=32, in_features=61),
                lambda: LinearW4(q, s, group=32, bias=torch.zeros(15)), lambda: LinearW4(q, s, group=32, device="cpu"),
                lambda: layer.forward(torch.zeros(2, 63, device="cuda")), lambda: layer.forward(torch.zeros(2, 64)),
                lambda: layer.forward(torch.zeros(2, 64, device="cuda", dtype=torch.float64)),
                lambda: layer.input_grad(torch.zeros(2, 64, device="cuda")),
                lambda: layer.input_grad(torch.zeros(2, 16, device="cuda"), gate=torch.zeros(3, 64, device="cuda")),
                lambda: layer.input_grad(torch.zeros(2, 16, device="cuda"), gate=torch.zeros(2, 64, device="cuda", dtype=F16)),
                lambda: layer.forward(torch.zeros(2, 64, device="cuda"), out=torch.zeros(2, 15, device="cuda")),
                lambda: layer.forward(torch.zeros(2, 64, device="cuda"), out=torch.zeros(16, 2, device="cuda").t()),
                lambda: LinearW4(q, s, group=32, input_grad=False).input_grad(torch.zeros(2, 16, device="cuda"))):
        with pytest.raises(E):
            bad()


def test_c_entry_refusals():
    layer, _, _ = _layer(16, 64, 32)
    lib, ctx = _hip.load_library(), _hip.ctx()
    x, y = torch.zeros((2, 64), device="cuda"), torch.zeros((2, 16), device="cuda")
    p, st = _hip._p, _hip._stream()
    f = lambda **k: lib.gr_linear_w4(ctx, k.get("w", layer._h), k.get("x", p(x)), k.get("dt", 0), k.get("n", 2), k.get("ldx", 64), 0,
                                     k.get("y", p(y)), k.get("ldy", 16), st)
    assert f() == 0
    assert f(n=0, x=None, y=None) == 0
    for bad in (dict(w=None), dict(x=None), dict(y=None), dict(dt=3), dict(n=-1), dict(ldx=63), dict(ldy=15), dict(n=2 ** 40)):
        assert f(**bad) == -1 and lib.gr_last_error(ctx)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,length", [(1, 5), (1, 75), (3, 7), (17, 131), (40, 8), (64, 255), (150, 401), (700, 333), (2600, 521)])
def test_rows_that_begin_inside_a_dword(dtype, n, length):
    """Where a row begins in memory must not change a bit of its result, nor must what lies beside it: the sums and their order
    are those of aligned rows, so equality is exact."""
    g = torch.Generator().manual_seed(n + length)
    other = 300
    for grad in (False, True):
        m, k = (length, other) if grad else (other, length)
        w = (torch.randn(m, k, generator=g) / length ** 0.5).cuda()
        group = 128 if k >= 128 else 32
        q, s, z = (v.cuda() for v in quantize(w, group))
        layer = LinearW4(q, s, z, group=group, in_features=k, input_grad=grad)
        x = torch.randn(n, length, generator=g).cuda().to(dtype)
        run = layer.input_grad if grad else layer.forward
        even = torch.zeros(n, length + length % 2, device="cuda", dtype=dtype)[:, :length]
        even.copy_(x)
        expect = run(even)
        for first, gap in ((0, 1 - length % 2), (1, 0), (1, 1), (3, 8), (2, 5)):
            flat = torch.full((first + n * (length + gap) + 1,), float("nan"), device="cuda", dtype=dtype)
            rows = torch.as_strided(flat, (n, length), (length + gap, 1), first)
            rows.copy_(x)
            assert torch.equal(run(rows), expect), (grad, first, gap)


def test_rows_past_32_bits():
    """More than 2^32 elements, and more small tiles than a launch holds: every offset and the choice of the kernel."""
    n, k, m = 140_000_003, 33, 10
    layer, w, _ = _layer(m, k, 32, sdt=F16)
    with_grad = LinearW4(*_packed(m, k), group=32, in_features=k, input_grad=True)
    rows = torch.tensor([0, 1, 65_075_262, 65_075_263, 130_150_524, 130_150_525, n - 2, n - 1], device="cuda")
    for run, a, b, ref in ((layer.forward, k, m, w.T), (with_grad.input_grad, m, k, w)):
        x = torch.zeros(n, a, device="cuda", dtype=F16)
        vals = torch.randn(len(rows), a, generator=torch.Generator().manual_seed(3)).to(F16)
        x[rows] = vals.cuda()
        y = run(x)
        del x
        v = vals.double().numpy()
        expect, mag = v @ ref, np.abs(v) @ np.abs(ref)
        assert (np.abs(y[rows].cpu().double().numpy() - expect) <= _tol(expect, mag, a, F16, 2.0 ** -15)).all()
        y[rows] = 0
        assert not y.any()
        del y
    torch.cuda.empty_cache()


def _packed(m, k):
    g = torch.Generator().manual_seed(0)                                            # the tensors of _layer(m, k, 32, F16)
    q = torch.randint(0, 256, (m, (k + 1) // 2), generator=g, dtype=torch.uint8)
    groups = -(-k // 32)
    s = (torch.rand((m, groups), generator=g) * 0.02 + 0.001).to(F16)
    return q.cuda(), s.cuda(), torch.randint(0, 16, (m, groups), generator=g, dtype=torch.uint8).cuda()


@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
def test_rows_past_one_launch(dtype):
    """2^30 rows of one input and one output: more workgroups of the tiled kernels than one launch counts threads for."""
    n = 2 ** 30 + 300
    layer, w, _ = _layer(1, 1, 32, sdt=F16, seed=2)
    rows = torch.tensor([0, 1, 2 ** 29, 2 ** 30 - 129, 2 ** 30 - 128, 2 ** 30 - 1, 2 ** 30, n - 2, n - 1], device="cuda")
    x = torch.zeros(n, 1, device="cuda", dtype=dtype)
    vals = torch.randn(len(rows), 1, generator=torch.Generator().manual_seed(3)).to(dtype)
    x[rows] = vals.cuda()
    for run in (layer.forward, layer.input_grad):
        y = run(x)
        expect = vals.double().numpy() * w[0, 0]
        assert (np.abs(y[rows].cpu().double().numpy() - expect) <= _tol(expect, np.abs(expect), 1, dtype, 2.0 ** -15)).all()
        y[rows] = 0
        assert not y.any()
        del y
    torch.cuda.empty_cache()


def _weights_of(rows, m, k, group):
    """(LinearW4 [m, k], its float64 weights) that are zero but for `rows`: {row: (code - zero point, scales [groups])}."""
    groups = -(-k // group)
    q, z, s = np.full((m, k + k % 2), 8, np.uint8), np.full((m, groups), 8, np.uint8), np.ones((m, groups), np.float32)
    for r, (c, scales) in rows.items():
        z[r] = 8 if abs(c) <= 7 else 2
        q[r], s[r] = int(z[r, 0]) + c, scales
    w = (q[:, :k].astype(np.float64) - z.astype(np.float64)[:, np.arange(k) // group]) * s.astype(np.float64)[:, np.arange(k) // group]
    packed = q[:, 0::2] | (q[:, 1::2] << 4)
    return LinearW4(torch.from_numpy(packed).cuda(), torch.from_numpy(s).cuda(), torch.from_numpy(z).cuda(), group=group, in_features=k), w


# The sizes take the LDS-tiled gradient (w4_cases.py) or the few-row one.
PRODUCTS = [(723, 1827, 639), (2, 40, 70)]


@pytest.mark.parametrize("n,k,m", PRODUCTS, ids=["tiled", "rows"])
def test_single_products_of_the_float32_gradient(n, k, m):
    """Two weight rows count and nearly cancel: gy5 w5 - w6 with w6 the float32 next to gy5 w5 and gy6 = -1, a product that three
    pieces hold exactly.  What is left shows the error of the first, promised to be within 1.5 * 2^-23 of it; the large pieces of
    both meet in one instruction, so the twelve additions, each off by 2^-23, stay below 2^-5.  w5 = 1 + a 2^-15 and
    gy5 = 1 + 2^-8 + b 2^-23, a and b < 256: a cut into pieces that leaves out a 2^-15 times b 2^-23 is off by up to 2^-22."""
    g = np.random.default_rng(0)
    groups = -(-k // 32)
    a = np.concatenate([[255, 254, 253, 129], g.integers(1, 256, max(0, groups - 4))])[:groups]
    b = np.concatenate([[255, 128], g.integers(1, 256, max(0, n - 2))])[:n]
    worst = 0.0
    for bb in sorted(set(b.tolist()))[-8:]:
        s5 = (1 + a * 2.0 ** -15).astype(np.float32)
        gy = np.zeros((n, m))
        gy[:, 5], gy[:, 6] = 1 + 2.0 ** -8 + bb * 2.0 ** -23, -1.0
        layer, w = _weights_of({5: (1, s5), 6: (1, (gy[0, 5] * s5.astype(np.float64)).astype(np.float32))}, m, k, 32)
        gx = layer.input_grad(torch.from_numpy(gy).float().cuda()).double().cpu().numpy()
        err, mag = np.abs(gx - gy @ w), gy[0, 5] * np.abs(w[5])
        worst = max(worst, float((err / mag).max()))
    assert worst <= 1.5 * 2.0 ** -23 + 12 * 2.0 ** -28, worst * 2.0 ** 23


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n,k,m", PRODUCTS + [(419, 3884, 619)], ids=["tiled", "rows", "tiled-bf16"])
def test_single_products_of_the_16_bit_gradients(n, k, m, dtype):
    """Two weight rows count and nearly cancel: gy5 w5 - gy6 w6 with w6 the 16-bit value next to gy5 w5 / gy6 and gy6 a power of
    two, a product that two pieces hold exactly.  What is left shows the error of the first, promised to be within 2^-15 of it."""
    g = np.random.default_rng(1)
    groups = -(-k // 32)
    s = np.concatenate([[0.011451721], g.uniform(0.01, 0.02, max(0, groups - 1))])[:groups].astype(np.float32)
    a = float(torch.tensor(1.0537109375).to(dtype))
    prod = a * 11.0 * s.astype(np.float64)
    e = np.floor(np.log2(prod)) - 15
    s6 = (np.round(prod / 2.0 ** e) * 2.0 ** e).astype(np.float32)
    layer, w = _weights_of({5: (11, s), 6: (-1, s6)}, m, k, 32)
    gy = np.zeros((n, m))
    up = 2.0 ** (np.arange(n) % 4 + 8)
    gy[:, 5], gy[:, 6] = a * up, up
    gx = layer.input_grad(torch.from_numpy(gy).to(dtype).cuda()).double().cpu().numpy()
    ref, mag = gy @ w, np.abs(gy) @ np.abs(w)
    tol = mag / 2 * 1.001 * 2.0 ** -15 + mag * 8 * 2.0 ** -23 + np.abs(ref) * torch.finfo(dtype).eps / 2 * 1.01 + 2.0 ** -25
    assert (np.abs(gx - ref) <= tol).all(), (np.abs(gx - ref) / tol).max()


@pytest.mark.parametrize("dtype,patterns", [(F32, (0x7f800001, 0x7fffffff, -1, -0x400000)), (BF16, (0x7f81, 0x7fff, -1, -0x40)),
                                            (F16, (0x7c01, 0x7fff, -1, -0x200))], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,k,m", PRODUCTS + [(419, 3884, 619), (2060, 678, 1604)], ids=["tiled", "rows", "tiled-bf16", "tiled-forward"])
def test_every_nan_stays_one(n, k, m, dtype, patterns):
    """NaNs of any payload: the pieces and halves that the kernels make of them must not turn into numbers."""
    layer, _, _ = _layer(m, k, 32, seed=15)
    ints = torch.int32 if dtype == F32 else torch.int16
    for run, c in ((layer.forward, k), (layer.input_grad, m)):
        x = torch.randn((n, c), generator=torch.Generator().manual_seed(1)).to(dtype)
        rows = min(n, len(patterns))
        for i in range(rows):
            x.view(ints)[i, (7 * i + 5) % c] = patterns[i]
        y = run(x.cuda())
        assert bool(torch.isnan(y[:rows]).all()) and bool(torch.isfinite(y[rows:]).all())


@pytest.mark.parametrize("n,k,m", PRODUCTS, ids=["tiled", "rows"])
def test_float32_gradient_extremes(n, k, m):
    """grad_y at float32's largest values and at 2^-100: rounding a piece must not overflow, nor may the low pieces be lost."""
    layer, w = _weights_of({5: (3, np.full(-(-k // 32), 2.0 ** -6, np.float32))}, m, k, 32)
    gy = np.zeros((n, m))
    top = float(torch.finfo(F32).max)
    gy[:, 5] = np.resize([top, -top, top * (1 - 2.0 ** -9), (1 + 2.0 ** -9) * 2.0 ** -100], n)
    gx = layer.input_grad(torch.from_numpy(gy).float().cuda()).double().cpu().numpy()
    ref = torch.from_numpy(gy).float().double().numpy() @ w
    assert (np.abs(gx - ref) <= 2.0 ** -21 * np.abs(ref)).all()


@pytest.mark.parametrize("relu", [False, True], ids=["linear", "relu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_forward_takes_part_in_autograd(dtype, relu):
    """backward() gives what input_grad gives for the same grad_y, bit for bit, and the formula's gradient."""
    layer, w, b = _layer(75, 200, 64, bias=True, seed=21)
    g = torch.Generator().manual_seed(22)
    x = torch.randn((2, 9, 200), generator=g).to("cuda", dtype).requires_grad_(True)
    gy = torch.randn((2, 9, 75), generator=g).to("cuda", dtype)
    y = layer.forward(x, relu=relu)
    assert y.requires_grad and torch.equal(y, layer.forward(x.detach(), relu=relu))
    y.backward(gy)
    want = gy.masked_fill(y.detach() <= 0, 0) if relu else gy
    assert x.grad.dtype == dtype and torch.equal(x.grad, layer.input_grad(want))
    gd = want.double().cpu().numpy().reshape(18, 75)
    ref = R.input_grad(gd, w)
    _check(x.grad.reshape(18, 200), ref, _tol(ref, np.abs(gd) @ np.abs(w), 75 + 64, dtype, 2.0 ** -15))
    # broadcast gradients (sum), transposed and shared inputs, twice through the same layer
    a = torch.randn((200, 5), generator=g).cuda().requires_grad_(True)
    (layer.forward(a.t()).sum() + layer.forward(a.t()).mul(2.0).sum()).backward()
    ref = 3.0 * np.repeat(w.sum(0)[:, None], 5, 1)
    _check(a.grad, ref, 3.0 * np.abs(w).sum(0)[:, None] * (140 * 2.0 ** -23 + 2.0 ** -22) + 1e-30)
    with torch.no_grad():
        assert not layer.forward(x).requires_grad
    with pytest.raises(_hip.GraphiteHipError):
        layer.forward(a.t(), out=torch.empty(5, 75, device="cuda"))
    one = _layer(75, 200, 64, seed=21)[0]
    (gx,) = torch.autograd.grad(one.forward(a.t()).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    no = LinearW4(torch.zeros((4, 16), dtype=torch.uint8), torch.ones((4, 1)), group=32, input_grad=False)
    with pytest.raises(_hip.GraphiteHipError):
        no.forward(torch.ones((2, 32), device="cuda", requires_grad=True)).sum().backward()


def test_autograd_in_a_captured_graph():
    layer, _, _ = _layer(200, 330, 64, bias=True, seed=23)
    x, gy = torch.zeros((40, 330), device="cuda"), torch.randn((40, 200), device="cuda")

    def step():
        leaf = x.detach().requires_grad_(True)
        y = layer.forward(leaf, relu=True)
        return y.detach(), torch.autograd.grad(y, leaf, gy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = step()
    for i in range(3):
        x.copy_(torch.randn((40, 330), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        yw, gw = step()
        assert torch.equal(y, yw) and torch.equal(gx, gw)
        torch.cuda.synchronize()
