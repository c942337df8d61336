"""Runs code against libgraphite_hip.so on the CPU, with hip_recorder.c in the place of the HIP runtime, in a process of its own:
    run(tmp_path, '''
    ctx = rec.context(0)
    ...
    result = rec.launches()
    ''')
returns `result` (plain values).  No kernel runs; the library's host code does."""
import ctypes as C
import json
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def run(tmp_path, code, timeout=120):
    so = os.path.join(str(tmp_path), "hip_recorder.so")
    if not os.path.exists(so):
        subprocess.check_call(["gcc", "-O1", "-shared", "-fPIC", "-w", "-I" + os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"),
                               os.path.join(HERE, "hip_recorder.c"), "-o", so])
    r = subprocess.run([sys.executable, os.path.abspath(__file__), so], input=code, capture_output=True, text=True, timeout=timeout)
    assert r.returncode == 0, r.stdout + r.stderr
    return json.loads(r.stdout.splitlines()[-1])


class Recorder:
    """The stand-in and the library behind it; pointers given to entry points may be any aligned numbers."""

    def __init__(self, so):
        self.hip = C.CDLL(so, mode=C.RTLD_GLOBAL)        # before the library: its symbols are found first
        self.hip.rec_name.restype = self.hip.rec_kernel.restype = C.c_char_p
        self.hip.rec_grid.restype = self.hip.rec_block.restype = C.POINTER(C.c_uint)
        self.hip.rec_lds.restype = C.c_size_t
        self.hip.rec_arg.restype = C.c_uint64
        sys.path.insert(0, ROOT)
        from graphite_amd import _hip
        self.lib = _hip.load_library()

    def context(self, device=0):
        ctx = C.c_void_p()
        assert self.lib.gr_ctx_create(device, C.byref(ctx)) == 0, self.lib.gr_last_error(None)
        return ctx

    def layer(self, ctx, out_features, in_features, group, scale_type=0, input_grad=1, p=1 << 40):
        w = C.c_void_p()
        g = -(-in_features // group)
        rc = self.lib.gr_w4_create(ctx, p, (in_features + 1) // 2, p, scale_type, g, p, g, None, out_features, in_features, group,
                                   input_grad, None, C.byref(w))
        assert rc == 0, (rc, self.lib.gr_last_error(ctx))
        self.hip.rec_clear()
        return w

    def kernels(self):
        """Names of every kernel that was registered."""
        return [self.hip.rec_kernel(i).decode() for i in range(self.hip.rec_kernels())]

    def launches(self):
        """[(kernel, grid, block, LDS bytes, first argument's first eight bytes)] since the last call."""
        out = []
        for i in range(self.hip.rec_launches()):
            out.append([self.hip.rec_name(i).decode(), list(self.hip.rec_grid(i)[:3]), list(self.hip.rec_block(i)[:3]), self.hip.rec_lds(i),
                        self.hip.rec_arg(i)])
        self.hip.rec_clear()
        return out


if __name__ == "__main__":
    scope = {"rec": Recorder(sys.argv[1]), "C": C}
    exec(sys.stdin.read(), scope)
    print(json.dumps(scope["result"]))
