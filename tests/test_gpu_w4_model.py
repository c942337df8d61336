"""The 4-bit linear layers and the soft-target gradient inside the classifiers and the attacks that call them
(gr_model_set_linear_w4, gr_model_input_grad_topk, engine.eot_gradient(teacher=), whitebox_attack, main --linear_w4)."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
from cases import INP, PT14, gtsrb_candidates, gtsrb_case                   # noqa: E402
from graphite_amd import _hip, engine, models, synth, transforms as T       # noqa: E402
from graphite_amd.distill import TeacherTop, teacher_top, topk_distill      # noqa: E402
from graphite_amd.linear_w4 import LinearW4, dequantize, quantize           # noqa: E402

pytestmark = pytest.mark.gpu

FC = ("fc5_1", "fc6_1", "fc7_1")


def _rounded(sd, names, group):
    """The state dict with the named layers' weights replaced by the values their 4-bit forms stand for."""
    out = dict(sd)
    for n in names:
        q, s, z = quantize(sd[n + ".weight"], group)
        out[n + ".weight"] = dequantize(q, s, z, group, sd[n + ".weight"].shape[1]).numpy()
    return out


def _pair(group=64, names=FC):
    """(4-bit GTSRBNet, the float GTSRBNet of the same weights, that one's state dict)."""
    sd = synth.gtsrb_state_dict(readout="toy3")
    ref = _rounded(sd, names, group)
    a, b = models.GTSRBNet(), models.GTSRBNet()
    a.load_state_dict(sd)
    b.load_state_dict(ref)
    return a.quantize_linear(sd, group, layers=names), b, ref


# Two float32 evaluations of the same three linear layers on the same features: the bar the float model is held to against
# torch (1e-4 of the largest logit; a wrong order, group or zero point is off by the logits themselves).
LOGIT_BAR = 1e-4


@pytest.mark.parametrize("names", [FC, ("fc5_1",), ("fc6_1", "fc7_1")], ids=["all", "fc5", "fc6-fc7"])
def test_gtsrbnet_logits_and_labels(names):
    a, b, _ = _pair(64, names)
    x = torch.from_numpy(synth.synth_images("w4-model", 37))
    for n in (1, 17, 37):
        la, lb = a.forward(x[:n]), b.forward(x[:n])
        assert float((la - lb).abs().max()) <= LOGIT_BAR * float(lb.abs().max())
    la = a.forward(x)
    assert torch.equal(a.hip_model.predict_dev(x), la.argmax(1))
    # a float layer again: bit for bit what the model gave before
    plain = models.GTSRBNet()
    plain.load_state_dict(synth.gtsrb_state_dict(readout="toy3"))
    a.set_linear_w4({n: None for n in names})
    assert torch.equal(a.forward(x), plain.forward(x))


def test_large_batches_cross_the_kernels():
    """700 images: other kernels than 37 images take, the same logits within the bar."""
    a, b, _ = _pair(128)
    x = torch.from_numpy(synth.synth_images("w4-model-large", 700))
    la, lb = a.forward(x), b.forward(x)
    assert float((la - lb).abs().max()) <= LOGIT_BAR * float(lb.abs().max())
    assert torch.equal(a.hip_model.predict_dev(x), la.argmax(1))
    assert float((a.forward(x[:37]) - la[:37]).abs().max()) <= LOGIT_BAR * float(lb.abs().max())


def test_tr_hits_counts_the_four_bit_victims_labels():
    a, _, _ = _pair(64)
    c = gtsrb_case(num_xforms=40)
    masks, thetas = gtsrb_candidates(c, 3)
    px = _hip.warp_batch_dev(c["vic"], masks, thetas, c["tab"], 1.0, True)
    labels = a.hip_model.predict_dev(px.reshape(-1, 3, 32, 32)).view(3, -1)
    target = int(labels.flatten().mode().values)
    hits, preds = engine.tr_hits(a, c["vic"], masks, thetas, c["tab"], target, return_preds=True)
    assert torch.equal(preds, labels) and torch.equal(hits.long(), (labels == target).sum(1))


def test_input_gradient_matches_the_float_model_of_the_same_weights():
    """Both sides take the same ReLU decisions but where a pre-activation lies within rounding of zero; without such a flip
    the gradients differ by float32 rounding (bar 1e-5 of the largest element, as for the float model against torch), a flip
    changes one of 1024 hidden units."""
    a, b, _ = _pair(64)
    x = torch.from_numpy(synth.synth_images("w4-grad", 37))
    la, ga = a.hip_model.input_grad(x, 27)
    lb, gb = b.hip_model.input_grad(x, 27)
    assert torch.equal(la, a.forward(x))
    scale = gb.abs().amax(dim=(1, 2, 3))
    err = (ga - gb).abs().amax(dim=(1, 2, 3))
    assert float((err <= 1e-5 * scale).float().mean()) >= 0.85, (err / scale).tolist()
    rel = (ga - gb).flatten(1).norm(dim=1) / gb.flatten(1).norm(dim=1)
    assert float(rel.max()) <= 0.25


@pytest.mark.parametrize("kind", ["gtsrb", "gtsrb-w4", "wrn", "wrn-w4"])
def test_soft_target_gradient_is_the_combination_of_the_label_gradients(kind):
    """g = d loss / d logits sums to 0 over the classes, so J^T g = -sum_c g_c J^T (q - e_c): the soft-target gradient is a
    combination of gr_model_input_grad's, at the same forward pass and the same decisions.  Each of the C + 1 backward passes
    is off by float32 rounding, taken as 2e-5 of its largest element (measured for the float model: 5e-7 against torch)."""
    if kind.startswith("gtsrb"):
        sd = synth.gtsrb_state_dict(readout="toy3")
        m, ncls = models.GTSRBNet(), 43
        m.load_state_dict(sd)
    else:
        sd = synth.wrn_state_dict("wrn-soft", depth=10, widen=2, num_classes=10)
        m, ncls = models.WideResNet(depth=10, num_classes=10, widen_factor=2), 10
        m.load_state_dict(sd)
    if kind.endswith("w4"):
        m.quantize_linear(sd, 32)
    h = m.hip_model
    x = torch.from_numpy(synth.synth_images("soft-target", 6, *((0.0, 1.0) if kind.startswith("wrn") else ())))
    logits = m.forward(x)
    other = torch.from_numpy(synth.synth_images("soft-target-teacher", 6, *((0.0, 1.0) if kind.startswith("wrn") else ())))
    for tau, rest, rows in ((1.0, False, 6), (2.0, True, 1)):
        top = teacher_top(m.forward(other)[:rows], 5, tau, rest)
        lg, gx, loss = h.input_grad_topk(x, top)
        want_loss, g = topk_distill(logits, top.index, top.value, tau, top.lse)
        assert torch.equal(lg, logits) and torch.equal(loss, want_loss)
        ref, tol = torch.zeros_like(gx, dtype=torch.float64), torch.zeros(6, dtype=torch.float64, device="cuda")
        for c in range(ncls):
            ig = h.input_grad(x, c)[1].double()
            ref -= g[:, c].double().view(-1, 1, 1, 1) * ig
            tol += 2e-5 * g[:, c].double().abs() * ig.abs().amax(dim=(1, 2, 3))
        tol += 2e-5 * ref.abs().amax(dim=(1, 2, 3))
        assert bool(((gx.double() - ref).abs().amax(dim=(1, 2, 3)) <= tol).all())
    # one class: the cross entropy to it
    one = TeacherTop(torch.full((1, 1), 3, device="cuda"), torch.zeros((1, 1), device="cuda"), None, 1.0)
    _, gx, loss = h.input_grad_topk(x, one)
    _, ce = h.input_grad(x, 3)
    assert float((gx - ce).abs().amax()) <= 1e-4 * float(ce.abs().amax())
    want = torch.nn.functional.cross_entropy(logits.double(), torch.full((6,), 3, device="cuda"), reduction="none")
    assert float((loss.double() - want).abs().amax()) <= 1e-5 * (1 + float(want.abs().amax()))


def test_soft_target_rows_follow_the_chunks():
    """1030 images pass the gradient in two chunks (1024 + 6): every row meets its own teacher row."""
    sd = synth.gtsrb_state_dict(readout="toy3")
    m = models.GTSRBNet()
    m.load_state_dict(sd)
    x = torch.from_numpy(synth.synth_images("soft-chunks", 1030))
    top = teacher_top(m.forward(x).flip(0).contiguous(), 4, 1.5)
    lg, _, loss = m.hip_model.input_grad_topk(x, top)
    assert torch.equal(loss, topk_distill(lg, top.index, top.value, 1.5, top.lse, want_grad=False)[0])


def test_eot_gradient_of_a_four_bit_victim_toward_its_full_precision_answers():
    """The operators together, as the whitebox loop uses them: 4-bit victim, EOT over the transforms, the loss its distance
    to what the float model answers for the target image -- and some steps along the gradient's sign reduce that loss."""
    a, _, _ = _pair(64)
    full = models.GTSRBNet()
    full.load_state_dict(synth.gtsrb_state_dict(readout="toy3"))
    c = gtsrb_case(num_xforms=24)
    orig = torch.from_numpy(0.04 + 0.92 * c["vic"]).cuda()
    mask = torch.zeros(3, 244, 244, device="cuda")
    mask[:, 40:200, 30:215] = 1.0
    tab = T.build_wb_table(c["xf"], 244, 244, PT14)
    target = torch.from_numpy(synth.synth_images("eot-teacher", 1))
    top = teacher_top(full.forward(target), 5, 2.0)
    grad, logits = engine.eot_gradient(a, orig, orig, mask, tab, None, teacher=top)
    assert grad.shape == orig.shape and bool(torch.isfinite(grad).all()) and not bool(grad[mask == 0].any())
    x = _hip.wb_forward(orig, orig, mask, tab) - 0.5
    lg, gx, loss = a.hip_model.input_grad_topk(x, top)
    assert torch.equal(lg, logits) and torch.equal(loss, topk_distill(lg, top.index, top.value, 2.0, top.lse)[0])
    want = _hip.wb_backward(orig, orig, mask, tab, gx) / len(tab)
    assert float((grad - want).abs().max()) <= 1e-5 * float(want.abs().max())          # float atomics reorder the sums


def test_whitebox_attack_takes_a_teacher():
    import random
    from graphite_amd.imageio import load_image_chw, load_image_u8_hwc, resize_u8_linear
    from graphite_amd.whitebox_attack import whitebox_attack
    from graphite_amd.whitebox_patch import whitebox_patch_attack
    a, _, _ = _pair(64)
    img = torch.from_numpy(load_image_chw(os.path.join(INP, "GTSRB/images/14.png")))
    hull = resize_u8_linear(load_image_u8_hwc(os.path.join(INP, "GTSRB/Hulls/14.png")), 244, 244)
    mask = torch.from_numpy((np.where(hull > 128, 255, 0).transpose(2, 0, 1) / 255.0).astype(np.float32))
    np.random.seed(42); torch.manual_seed(42); random.seed(42)
    xforms = T.get_transform_params(8, 'GTSRB')
    top = TeacherTop(torch.tensor([[27, 14]], device="cuda"), torch.tensor([[4.0, -4.0]], device="cuda"), None, 1.0)
    r = whitebox_attack(a, img, mask, 27, PT14, step_size=4 / 255, iters=3, min_tr=0.0, first_round_iters=4, max_rounds=1,
                        xforms=xforms, teacher=top)
    assert r["rounds"] == 1 and r["adversarial"].shape == img.shape and 0.0 <= r["transform_robustness"] <= 1.0
    r = whitebox_patch_attack(a, img, 27, PT14, 60, iters=1, xforms=xforms, teacher=top)
    assert len(r["per_position"]) == 5 and r["adversarial"].shape == img.shape


def test_the_attack_command_runs_on_a_four_bit_victim(tmp_path, monkeypatch, capsys):
    from graphite_amd import main
    monkeypatch.chdir(INP + "/..")
    argv = ["-v", "14", "-t", "27", "-m", "8", "-b", "8", "--no_outputs", "--linear_w4", "64", "--out_path", str(tmp_path) + "/"]
    monkeypatch.setattr(sys, "argv", ["main.py"] + argv)
    r = main.main(argv)
    assert r["queries"] > 0 and 0.0 <= r["transform_robustness"] <= 1.0


def test_wideresnet_and_bagnet_heads():
    from graphite_amd.patchguard.patchguard_predict import PatchGuard
    sd = synth.wrn_state_dict("wrn-w4", depth=10, widen=2, num_classes=10)
    x = torch.from_numpy(synth.synth_images("wrn-w4", 9, 0.0, 1.0))
    q = models.WideResNet(depth=10, num_classes=10, widen_factor=2).load_state_dict(sd).quantize_linear(sd, 32)
    f = models.WideResNet(depth=10, num_classes=10, widen_factor=2).load_state_dict(_rounded(sd, ("fc",), 32))
    lq, lf = q.forward(x), f.forward(x)
    # one linear layer of 128 inputs on identical activations: 2 * 192 * 2^-23 of the sum of |x w|, bounded by 8 times the logits
    assert float((lq - lf).abs().max()) <= 2 * 192 * 2.0 ** -23 * 8 * float(lf.abs().max())
    gq, gf = q.hip_model.input_grad(x, 4)[1], f.hip_model.input_grad(x, 4)[1]
    rel = (gq - gf).flatten(1).norm(dim=1) / gf.flatten(1).norm(dim=1)
    assert float((rel <= 1e-4).float().mean()) >= 0.6 and float(rel.max()) <= 0.25
    sd = synth.bagnet_state_dict()
    w = sd["fc.weight"] if "fc.weight" in sd else sd["module.fc.weight"]
    bias = sd["fc.bias"] if "fc.bias" in sd else sd["module.fc.bias"]
    qq, s, z = quantize(w, 64)
    ref = dict(sd)
    ref["fc.weight" if "fc.weight" in sd else "module.fc.weight"] = dequantize(qq, s, z, 64).numpy()
    pq, pf = PatchGuard(sd), PatchGuard(ref)
    pq.hip_model.set_linear_w4(0, LinearW4(qq, s, z, bias=torch.as_tensor(bias), group=64))
    x = torch.from_numpy(synth.synth_images("bag-w4", 3))
    a, b = pq.local_logits(x), pf.local_logits(x)
    assert float((a - b).abs().max()) <= 2 * 2112 * 2.0 ** -23 * 8 * float(b.abs().max())


def test_refusals():
    sd = synth.gtsrb_state_dict(readout="toy3")
    m = models.GTSRBNet()
    m.load_state_dict(sd)
    q, s, z = quantize(sd["fc6_1.weight"], 64)
    fc6 = LinearW4(q, s, z, group=64)
    E = _hip.GraphiteHipError
    with pytest.raises(E):
        m.set_linear_w4({"fc5_1": fc6})                                     # 1024 -> 1024 is not 2048 -> 1024
    with pytest.raises(ValueError):
        m.set_linear_w4({"fc8": fc6})
    with pytest.raises(E):
        m.hip_model.set_linear_w4(3, fc6)
    m.set_linear_w4({"fc6_1": fc6})
    with pytest.raises(E):
        m.set_precision("bf16")
    m.set_linear_w4({"fc6_1": None})
    m.set_precision("bf16")
    with pytest.raises(E):
        m.set_linear_w4({"fc6_1": fc6})
    m.set_precision("f32")
    x = torch.from_numpy(synth.synth_images("w4-refuse", 2))
    m.set_linear_w4({"fc6_1": LinearW4(q, s, z, group=64, input_grad=False)})
    m.forward(x)
    with pytest.raises(E):
        m.hip_model.input_grad(x, 1)
    top = teacher_top(m.forward(x), 3)
    m.set_linear_w4({"fc6_1": None})
    for bad in (top._replace(index=top.index[:, :2]), top._replace(tau=0.0), top._replace(lse=top.lse[:1]),
                TeacherTop(top.index.repeat(2, 1), top.value.repeat(2, 1), None, 1.0)):
        with pytest.raises(E):
            m.hip_model.input_grad_topk(x, bad)


@pytest.mark.parametrize("group", [32, 64, 96, 256])
def test_an_image_gets_the_same_bits_in_every_batch(group):
    """Chunk size, workspace limit and rank count decide which images pass a layer together; results do not follow them."""
    sd = synth.gtsrb_state_dict(readout="toy3")
    m = models.GTSRBNet().load_state_dict(sd).quantize_linear(sd, group)
    x = torch.from_numpy(synth.synth_images("w4-batches", 1030)).cuda()
    top = teacher_top(m.forward(x[:1]), 5, 2.0)
    logits, labels = m.forward(x), m.hip_model.predict_dev(x)
    grads, soft = m.hip_model.input_grad(x, 3)[1], m.hip_model.input_grad_topk(x, top)[1]
    for a, b in ((0, 1), (3, 20), (100, 137), (0, 640), (300, 1024), (1024, 1030)):
        assert torch.equal(m.forward(x[a:b]), logits[a:b]) and torch.equal(m.hip_model.predict_dev(x[a:b]), labels[a:b])
        assert torch.equal(m.hip_model.input_grad(x[a:b], 3)[1], grads[a:b])
        if a % 4 == 0:                                  # the loss sums a row of 43 logits from its first 16-byte border on
            assert torch.equal(m.hip_model.input_grad_topk(x[a:b], top)[1], soft[a:b])
    try:
        for limit in (64 << 20, 150 << 20):             # 80 images a chunk and more
            _hip.set_workspace_limit(limit)
            assert torch.equal(m.forward(x), logits) and torch.equal(m.hip_model.input_grad(x, 3)[1], grads)
            assert torch.equal(m.hip_model.input_grad_topk(x, top)[1], soft)
    finally:
        _hip.set_workspace_limit(8 << 30)


def test_heads_of_the_other_models_in_every_batch():
    from graphite_amd.patchguard.patchguard_predict import PatchGuard
    sd = synth.wrn_state_dict("wrn-w4", depth=10, widen=2, num_classes=10)
    x = torch.from_numpy(synth.synth_images("wrn-batches", 700, 0.0, 1.0)).cuda()
    m = models.WideResNet(depth=10, num_classes=10, widen_factor=2).load_state_dict(sd).quantize_linear(sd, 32)
    logits = m.forward(x)
    for a, b in ((0, 1), (3, 20), (100, 641)):
        assert torch.equal(m.forward(x[a:b]), logits[a:b])
    sd = synth.bagnet_state_dict()
    key = "fc" if "fc.weight" in sd else "module.fc"
    q, s, z = quantize(sd[key + ".weight"], 64)
    p = PatchGuard(sd)
    p.hip_model.set_linear_w4(0, LinearW4(q, s, z, bias=torch.as_tensor(sd[key + ".bias"]), group=64))
    x = torch.from_numpy(synth.synth_images("bag-batches", 24)).cuda()
    local = p.local_logits(x)
    for a, b in ((0, 1), (3, 20)):
        assert torch.equal(p.local_logits(x[a:b]), local[a:b])


def test_hits_do_not_follow_the_chunk():
    a, _, _ = _pair(64)
    c = gtsrb_case(num_xforms=60)
    masks, thetas = gtsrb_candidates(c, 12)
    lib, ctx = _hip.load_library(), _hip.ctx()
    want = None
    try:
        for chunk in (8192, 64, 200, 641):
            assert lib.gr_ctx_set_chunk(ctx, chunk) == 0
            hits, preds = engine.tr_hits(a, c["vic"], masks, thetas, c["tab"], 27, return_preds=True)
            want = (hits, preds) if want is None else want
            assert torch.equal(hits, want[0]) and torch.equal(preds, want[1])
    finally:
        lib.gr_ctx_set_chunk(ctx, 8192)


def test_gradient_chunks_of_a_few_images():
    """WideResNet-34-10 keeps 17 MB an image: 64 MiB hold three, whose rows of logits lie elsewhere within 16 bytes than the whole
    batch's; also where the caller asks for no logits."""
    sd = synth.wrn_state_dict()
    m = models.WideResNet(num_classes=10).load_state_dict(sd).quantize_linear(sd, 64)
    x = torch.from_numpy(synth.synth_images("wrn-chunks", 11, 0.0, 1.0)).cuda()
    top = teacher_top(m.forward(x[:1]), 3, 1.0)
    h, p = m.hip_model, _hip._p

    def no_logits():
        loss, gx = torch.empty(11, device="cuda"), torch.empty_like(x)
        assert _hip.load_library().gr_model_input_grad_topk(_hip.ctx(), h._h, p(x), 11, p(top.index), p(top.value), 3, 0, p(top.lse), 1.0,
                                                            p(loss), None, p(gx), _hip._stream()) == 0
        return loss, gx

    want = h.input_grad(x, 3)[1], *h.input_grad_topk(x, top)[1:], *no_logits()
    assert torch.equal(want[1], want[4]) and torch.equal(want[2], want[3]) and bool(want[0].any()) and bool(want[1].any())
    try:
        _hip.set_workspace_limit(64 << 20)
        got = h.input_grad(x, 3)[1], *h.input_grad_topk(x, top)[1:], *no_logits()
    finally:
        _hip.set_workspace_limit(8 << 30)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
