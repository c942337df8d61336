"""Host side of the 4-bit layers' and the distillation loss' C entries, on the CPU (hip_recorder.c stands in for the runtime)."""
import hip_recorder
import w4_cases


def test_destroying_a_layer_leaves_the_current_device(tmp_path):
    """A layer of device 1 is collected while the caller works on device 0."""
    got = hip_recorder.run(tmp_path, """
ctx = rec.context(1)
w = rec.layer(ctx, 43, 1024, 64)
result = [rec.hip.rec_device()]
rec.hip.hipSetDevice(0)
rec.lib.gr_w4_destroy(w)
result.append(rec.hip.rec_device())
""")
    assert got == [1, 0]


LAUNCHES = """
ctx = rec.context()
p, out = 1 << 40, []
for dtype, nt, n, v in ((0, 64, 2 ** 26 + 77, 43), (1, 256, 2 ** 24 + 5, 3000), (2, 1024, 2 ** 22 + 1, 70001), (0, 64, 2 ** 31 - 1, 1), (0, 64, 3, 43)):
    rc = rec.lib.gr_distill_topk(ctx, p, dtype, n, v, v, p, p, 0, 1, 1, p, 1.0, None, p, p, v, None)
    out.append([rc, n, [l[1][0] for l in rec.launches()]])
result = out
"""


def test_rows_of_the_loss_past_one_launch(tmp_path):
    """A launch's threads are counted in 32 bits; every row belongs to exactly one launch."""
    for rc, n, rows in hip_recorder.run(tmp_path, LAUNCHES):
        assert rc == 0 and sum(rows) == n


def test_rows_of_the_layers_past_one_launch(tmp_path):
    got = hip_recorder.run(tmp_path, """
ctx = rec.context()
p, result = 1 << 40, []
for m, k in ((1, 1), (10, 33), (100, 40)):
    w = rec.layer(ctx, m, k, 32)
    for dtype in (0, 1, 2):
        for n in (2 ** 30 + 300, 2 ** 31 + 5, 2 ** 32 + 1):
            rc = rec.lib.gr_linear_w4(ctx, w, p, dtype, n, k, 0, p, m, None)
            result.append([rc, n, m, [l[:2] for l in rec.launches()]])
            rc = rec.lib.gr_linear_w4_input_grad(ctx, w, p, dtype, n, m, None, 0, p, k, None)
            result.append([rc, n, k, [l[:2] for l in rec.launches()]])
""")
    for rc, n, cols, launches in got:
        assert rc == 0 and len(launches) >= (1 if n < 2 ** 31 else 2), (rc, n, cols, launches)
        assert all("k_w4_gemm" in name for name, _ in launches)
        assert any(sum(g[0] for _, g in launches) == -(-cols // 128) * -(-n // rows) for rows in (128, 256))


def test_layers_of_more_weights_than_a_launch_packs_are_refused(tmp_path):
    got = hip_recorder.run(tmp_path, """
ctx = rec.context()
result, w = [], C.c_void_p()
for m, k in ((1 << 17, 1 << 18), (1, (1 << 28) + 1), ((1 << 31) - 400, 64), (1 << 17, (1 << 18) - 128), (1 << 27, 128)):
    rc = rec.lib.gr_w4_create(ctx, 1 << 40, (k + 1) // 2, 1 << 40, 0, 1, None, 0, None, m, k, 1 << 30, 1, None, C.byref(w))
    result.append([rc, bool(rec.launches()), bool(w.value)])
""")
    assert got == [[-1, False, False]] * 3 + [[0, True, True]] * 2


CHOICES = """
import re
def parse(name):
    a = [int(v) for v in re.findall("L[ib]([0-9]+)E", name)]
    if "k_w4_rows" in name:
        dt, st, half, nt, mt, gs, d, grad = a
        return [["rows", nt, mt, gs], grad, dt, half]
    dt, st, half, grad, tm, tn, wm, wn, ks = a
    return [["tiled", tn, ks], grad, dt, half]
ctx, p, chosen = rec.context(), 1 << 40, []
for kernel, grad, n, k, m, group, t in cases:
    w = rec.layer(ctx, m, k, group)
    dt, half = ("f32", "bf16", "f16").index(t.rstrip("*")), t.endswith("*")
    c = m if grad else k
    x, ld = p + (2 if half else 0), c if dt == 0 else c + (c + half) % 2
    if grad: rc = rec.lib.gr_linear_w4_input_grad(ctx, w, x, dt, n, ld, None, 0, p, k, None)
    else: rc = rec.lib.gr_linear_w4(ctx, w, x, dt, n, ld, 0, p, m, None)
    names = [l[0] for l in rec.launches()]
    chosen.append([rc, len(names), parse(names[0])])
result = [chosen, [parse(n) for n in rec.kernels() if "k_w4_rows" in n or "k_w4_gemm" in n]]
"""


def test_every_kernel_of_the_layers_has_its_case(tmp_path):
    """The sizes of w4_cases.py take the kernels they name, and there is no kernel that none of them takes."""
    chosen, built = hip_recorder.run(tmp_path, f"cases = {w4_cases.FLAT!r}\n" + CHOICES)
    as_set = lambda rows: {(tuple(k), *rest) for k, *rest in rows}
    for case, (rc, count, got) in zip(w4_cases.FLAT, chosen):
        kernel, grad, *_, t = case
        dt = ("f32", "bf16", "f16").index(t.rstrip("*"))
        assert rc == 0 and count == 1 and got == [list(kernel), int(grad), dt, int(t.endswith("*"))], (w4_cases.label(case), got)
    assert as_set(g for _, _, g in chosen) == as_set(built)
