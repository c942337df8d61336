"""Host side of the 4-bit linear layers and the distillation loss: quantisation, shapes, refusals without a GPU, and the
64-bit restatements the GPU tests compare with."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import lowbit_reference as R                                                # noqa: E402
from graphite_amd import _hip                                               # noqa: E402
from graphite_amd.linear_w4 import LinearW4, dequantize, quantize           # noqa: E402


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("shape,group", [((1, 1), 32), ((5, 31), 32), ((3, 64), 32), ((7, 129), 64), ((2, 100), 4096)])
def test_quantize_stays_within_its_steps(shape, group, symmetric):
    w = np.random.default_rng(0).standard_normal(shape)
    w[0, :] = np.abs(w[0, :]) + 0.5                                          # a group on one side of zero
    q, s, z = quantize(w, group, symmetric)
    m, k = shape
    assert q.dtype == torch.uint8 and tuple(q.shape) == (m, (k + 1) // 2) and tuple(s.shape) == (m, -(-k // group))
    assert (z is None) == symmetric and (symmetric or int(z.max()) <= 15)
    back = R.weights(q.numpy(), s.numpy(), None if symmetric else z.numpy(), group, k)
    step = s.double().numpy()[:, np.arange(k) // group]
    assert (np.abs(back - w) <= step * (0.5 if symmetric else 1.0) * 1.0001).all()
    if k % 2:
        assert int((q[:, -1] >> 4).max()) == 0
    assert np.abs(dequantize(q, s, z, group, k).double().numpy() - back).max() <= 2.0 ** -23 * np.abs(back).max()


def test_quantize_refuses():
    w = np.ones((4, 64))
    for bad in (lambda: quantize(w, 0), lambda: quantize(w, 33), lambda: quantize(w[0]), lambda: quantize(w[:0]),
                lambda: quantize(np.full((2, 32), np.nan), 32), lambda: quantize(np.full((2, 32), np.inf), 32)):
        with pytest.raises(ValueError):
            bad()


def test_zero_groups_and_checkpoint_layout():
    w = np.zeros((2, 64))
    w[1, 32:] = np.arange(32) / 31.0
    q, s, z = quantize(w, 32)
    assert not R.weights(q.numpy(), s.numpy(), z.numpy(), 32, 64)[0].any()
    codes = R.unpack(q.numpy(), 64)
    assert codes[1, 32] == 0 and codes[1, 63] == 15 and int(q[1, 31]) >> 4 == 15 and int(q[1, 16]) & 15 == 0


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    q, s, z = quantize(np.ones((4, 64)), 32)
    with pytest.raises(_hip.GraphiteHipError):
        LinearW4(q, s, z, group=32)
    from graphite_amd.distill import topk_distill
    with pytest.raises(_hip.GraphiteHipError):
        topk_distill(torch.zeros(2, 5), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))
    with pytest.raises(_hip.GraphiteHipError):
        LinearW4(q, s, z, group=48)
    with pytest.raises(_hip.GraphiteHipError):
        LinearW4(q.int(), s, z, group=32)


def test_c_entries_refuse_without_a_context():
    lib = _hip.load_library()
    assert lib.gr_w4_create(None, None, 0, None, 0, 0, None, 0, None, 1, 1, 32, 0, None, None) == -1
    assert lib.gr_linear_w4(None, None, None, 0, 1, 1, 0, None, 1, None) == -1
    assert lib.gr_linear_w4_input_grad(None, None, None, 0, 1, 1, None, 0, None, 1, None) == -1
    assert lib.gr_distill_topk(None, None, 0, 1, 1, 1, None, None, 0, 1, 1, None, 1.0, None, None, None, 1, None) == -1
    assert lib.gr_model_set_linear_w4(None, 0, None) == -1
    assert lib.gr_model_input_grad_topk(None, None, None, 1, None, None, 1, 1, None, 1.0, None, None, None, None) == -1
    lib.gr_w4_destroy(None)


@pytest.mark.parametrize("rest", [False, True])
def test_reference_gradient_is_the_difference_of_its_losses(rest):
    g = np.random.default_rng(1)
    z, t = g.standard_normal((2, 20)) * 2, g.standard_normal((2, 20)) * 2
    idx = np.argsort(-t, 1)[:, :4]
    idx[1, 3] = -1
    val = np.take_along_axis(t, np.maximum(idx, 0), 1)
    lse = np.log(np.exp(t / 1.5).sum(1)) if rest else None
    loss, grad = R.distill(z, idx, val, 1.5, lse)
    for i in range(20):
        d = np.zeros_like(z)
        d[:, i] = 1e-5
        fd = (R.distill(z + d, idx, val, 1.5, lse)[0] - R.distill(z - d, idx, val, 1.5, lse)[0]) / 2e-5
        assert np.abs(fd - grad[:, i]).max() <= 1e-8
    assert (loss > 0).all() and np.abs(grad.sum(1)).max() <= 1e-12


@pytest.mark.parametrize("case", ["nothing_unnamed_is_left", "named_mass_above_one", "all_classes_named"])
def test_reference_gradient_where_the_target_does_not_add_up_to_one(case):
    """Open form without a p_rest term: the named p_j alone weigh the loss, and the softmax's normaliser takes their sum."""
    g = np.random.default_rng(2)
    v = 10
    z, t = g.standard_normal((2, v)) * 2, g.standard_normal((2, v)) * 2
    k = v if case == "all_classes_named" else 4
    idx = np.argsort(-t, 1)[:, :k]
    val = np.take_along_axis(t, idx, 1)
    lse = np.log(np.exp(t / 1.5).sum(1))
    if case == "nothing_unnamed_is_left":
        keep = np.take_along_axis(z, idx, 1)
        z[:] = -np.inf
        np.put_along_axis(z, idx, keep, 1)
    else:
        lse = lse - (0.8 if case == "named_mass_above_one" else -0.3)
    mass = np.exp(val / 1.5 - lse[:, None]).sum(1)
    assert (mass > 1.05).all() if case == "named_mass_above_one" else (mass < 0.95).all()
    _, grad = R.distill(z, idx, val, 1.5, lse)
    assert not grad[~np.isfinite(z)].any() and np.abs(grad.sum(1)).max() <= 1e-12
    for i in range(v):
        d = np.zeros_like(z)
        d[:, i] = 1e-5
        fd = (R.distill(z + d, idx, val, 1.5, lse)[0] - R.distill(z - d, idx, val, 1.5, lse)[0]) / 2e-5
        assert np.abs(np.where(np.isfinite(z[:, i]), fd - grad[:, i], 0.0)).max() <= 1e-8
