"""One size for every kernel that the 4-bit layers choose from, each with ragged ends and with more steps than the kernel's
unrolled loops hold.  test_w4_host.py shows that these sizes take these kernels and that no other one is built;
test_gpu_w4_variants.py runs them.

(kernel, gradient, rows, in, out, group, types) -- kernel ("rows", batch tiles, row tiles, groups a chunk) or ("tiled", batch
tiles a wave, steps a stage); types: bf16* and f16* are rows that begin in the middle of a dword."""

ALL = ("f32", "bf16", "f16", "bf16*", "f16*")
HALF, WHOLE, BITS16 = ("bf16*", "f16*"), ("bf16", "f16"), ("bf16", "f16", "bf16*", "f16*")
ONE_DEEP = ("f32",) + HALF                     # one chunk at a time; the aligned 16-bit kernels for one batch tile take two

CASES = [
    # forward, few rows
    (("rows", 1, 1, 1), False, 1, 2073, 2, 128, ONE_DEEP), (("rows", 1, 1, 1), False, 1, 4708, 2, 128, WHOLE),
    (("rows", 1, 1, 2), False, 1, 2084, 2, 192, ONE_DEEP), (("rows", 1, 1, 2), False, 1, 5164, 2, 64, WHOLE),
    (("rows", 1, 1, 4), False, 1, 2201, 2, 96, ONE_DEEP), (("rows", 1, 1, 4), False, 1, 4243, 2, 32, WHOLE),
    (("rows", 1, 2, 1), False, 1, 2235, 4350, 256, ONE_DEEP), (("rows", 1, 2, 1), False, 1, 4152, 4478, 384, WHOLE),
    (("rows", 1, 2, 2), False, 1, 2269, 4486, 192, ONE_DEEP), (("rows", 1, 2, 2), False, 1, 4665, 4965, 64, WHOLE),
    (("rows", 1, 2, 4), False, 1, 2583, 3895, 32, ("f32",)), (("rows", 1, 2, 4), False, 1, 2572, 4147, 96, HALF),
    (("rows", 1, 2, 4), False, 2, 4284, 4558, 160, WHOLE),
    (("rows", 2, 2, 1), False, 51, 1043, 2773, 256, BITS16), (("rows", 2, 2, 2), False, 2727, 1104, 37, 192, BITS16),
    (("rows", 2, 2, 4), False, 2660, 1161, 36, 96, BITS16),
    (("rows", 2, 4, 1), False, 4029, 1196, 34, 384, ("f32",)), (("rows", 2, 4, 1), False, 171, 1026, 1549, 128, BITS16),
    (("rows", 2, 4, 2), False, 17, 1261, 8292, 64, ("f32",)), (("rows", 2, 4, 2), False, 106, 1160, 2485, 192, BITS16),
    (("rows", 2, 4, 4), False, 329, 1081, 737, 160, ("f32",)), (("rows", 2, 4, 4), False, 4691, 1092, 35, 160, BITS16),
    (("rows", 4, 4, 1), False, 167, 1091, 3653, 128, WHOLE), (("rows", 4, 4, 1), False, 1587, 1153, 623, 128, HALF),
    (("rows", 4, 4, 2), False, 289, 1027, 2557, 192, WHOLE), (("rows", 4, 4, 2), False, 163, 2132, 5374, 64, HALF),
    (("rows", 4, 4, 4), False, 297, 1070, 3094, 32, WHOLE),
    # forward, many rows
    (("tiled", 2, 1), False, 8173, 668, 133, 64, ("f32",)), (("tiled", 2, 1), False, 8173, 668, 133, 192, ("f32",)),
    (("tiled", 2, 1), False, 2060, 678, 1604, 96, ("f32",)), (("tiled", 2, 1), False, 8173, 668, 133, 1024, ("f32",)),
    (("tiled", 2, 2), False, 162, 678, 8004, 256, BITS16), (("tiled", 2, 2), False, 162, 678, 8004, 64, BITS16),
    (("tiled", 2, 2), False, 2060, 678, 1604, 32, BITS16), (("tiled", 2, 2), False, 2060, 678, 1604, 96, BITS16),
    (("tiled", 4, 2), False, 403, 646, 8395, 64, BITS16), (("tiled", 4, 2), False, 403, 646, 8395, 192, BITS16),
    (("tiled", 4, 2), False, 403, 646, 8395, 1024, BITS16),
    # gradient, few rows
    (("rows", 1, 2, 1), True, 1, 2, 2073, 128, ALL), (("rows", 1, 4, 1), True, 3, 7406, 2053, 128, ("f32",)),
    (("rows", 1, 4, 1), True, 1, 8957, 2591, 64, BITS16), (("rows", 2, 8, 1), True, 5477, 67, 1096, 256, ("f32",)),
    (("rows", 2, 8, 1), True, 4465, 71, 1198, 256, BITS16),
    # gradient, many rows
    (("tiled", 2, 1), True, 723, 1827, 639, 96, ("f32", "f16", "f16*")), (("tiled", 2, 1), True, 723, 1827, 639, 32, ("f32", "f16", "f16*")),
    (("tiled", 4, 1), True, 419, 3884, 619, 32, ("bf16", "bf16*")), (("tiled", 4, 1), True, 419, 3884, 619, 96, ("bf16", "bf16*")),
]
FLAT = [(kernel, grad, n, k, m, group, t) for kernel, grad, n, k, m, group, types in CASES for t in types]


def label(case):
    kernel, grad, n, k, m, group, t = case
    return f"{'gradient' if grad else 'forward'}-{t}-{'x'.join(map(str, kernel))}-{n}x{k}x{m}-{group}"
