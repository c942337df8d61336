"""Host side of the 4-bit layers' and the distillation loss' C entries, on the CPU (hip_recorder.c stands in for the runtime)."""
import hip_recorder


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
