"""Which kernels the shapes of dense_stack_shapes take, on the CPU: the library
runs on a model of the HIP runtime that counts launches."""
from dense_stack_shapes import MX4_LAYERS, NORMS, UPDATES
from host_hip_child import host_hip  # noqa: F401

SETUP = """
from chimera_amd import operators as op
L = capi.lib()
ctx = context()
A = 1 << 40  # arrays apart from each other; nothing reads them
NAME = {"f32": "f", "f16": "DF16_", "bf16": "DF16b"}

def launches(part):
    return hip.host_hip_launches(part.encode())

def need(call, *args):
    n = C.c_size_t()
    capi.check(call(*args, C.byref(n)))
    hip.host_hip_reset_launches()
    return n.value

def numbers(values):
    return "".join(f"Li{v}E" for v in values)
"""


def test_norms(host_hip):  # noqa: F811
    host_hip(SETUP + f"""
for rows, n, type, out, forward, backward in {NORMS}:
    s = op.NormShape(rows, n, op.TYPES[type], op.TYPES[out], 1e-5)
    bytes = need(L.chimera_norm_workspace, C.byref(s))
    f = op.NormForward(A, 2 * A, 3 * A, 4 * A, 5 * A, 6 * A, n, n)
    b = op.NormBackward(A, 2 * A, 3 * A, 5 * A, 6 * A, 7 * A, 8 * A, 9 * A, n, n, n, 10 * A, bytes)
    capi.check(L.chimera_norm_forward_device(ctx.handle, C.byref(s), C.byref(f)))
    capi.check(L.chimera_norm_backward_device(ctx.handle, C.byref(s), C.byref(b)))
    tail = lambda v: numbers(v[:2]) + f"LNS0_3FitE{{v[2]}}E"
    assert launches("norm_forward_kernel") == 1 and launches(tail(forward)) >= 1, (rows, n)
    if backward == "wide":
        assert launches("norm_wide_kernel") == 1 and launches("norm_wide_sums_kernel") == 1, (rows, n)
        assert launches("norm_backward_kernel") == 0 and launches(tail(forward)) == 1, (rows, n)
    else:
        assert backward == forward and launches("norm_backward_kernel") == 1 and launches(tail(forward)) == 2, (rows, n)
    assert launches("norm_join_kernel") == 1
""")


def test_4_bit_layers(host_hip):  # noqa: F811
    host_hip(SETUP + f"""
for rows, k, n, type, normalize, kernel in {MX4_LAYERS}:
    s = op.LinearShape(rows, k, n, op.TYPES[type], op.TYPES[type], 0, int(normalize))
    bytes = need(L.chimera_mx4_linear_workspace, C.byref(s))
    a = op.Mx4LinearArgs(A, 2 * A, 3 * A, None, None, 6 * A, k, n, n, 8 * A if bytes else None, bytes)
    capi.check(L.chimera_mx4_linear_device(ctx.handle, C.byref(s), C.byref(a)))
    found = kernel[1:3] if kernel[0] == "few" else kernel[1:]
    name = f"mx4_{{kernel[0]}}_kernelI" + NAME[type] + numbers(found)
    assert launches(name) == 1, (rows, k, n, type)
    if kernel[0] == "few":
        assert launches(name + f"Lb{{kernel[3]}}ELi{{kernel[4]}}E") == 1
    assert launches("mx4_quantise_kernel") == int(kernel[0] != "few")
""")


def test_updates(host_hip):  # noqa: F811
    host_hip(SETUP + f"""
for rows, cols, symmetric, x in {UPDATES}:
    s = op.OrthogonalShape(rows, cols, 0, 0, 2, 3.4445, -4.775, 2.0315)
    bytes = need(L.chimera_orthogonal_workspace, C.byref(s))
    a = op.OrthogonalArgs(gradient=A, out=2 * A, gradient_stride=cols, out_stride=cols, workspace=3 * A, workspace_bytes=bytes)
    capi.check(L.chimera_orthogonal_update_device(ctx.handle, C.byref(s), C.byref(a)))
    both = x == "both"
    for kind in (2, 3):
        assert launches(f"orthogonal_both_kernelILNS0_4KindE{{kind}}E") == int(both), (rows, cols)
    for kind, kernel, count in ((0, symmetric, 2), (1, symmetric, 2), (2, x, 1), (3, x, 1))[:1 if both else 4]:
        if kind == 3 and kernel == ("tile", 128, 2, 2, 4):
            kernel = ("tile", 128, 2, 4, 4)
        name = f"orthogonal_{{kernel[0]}}_kernelILNS0_4KindE{{kind}}E" + numbers(kernel[1:])
        assert launches(name) == count, (rows, cols, name)
    assert launches("orthogonal_") == 2 + (4 if both else 6), (rows, cols)
""")


def test_every_kernel_has_a_shape(host_hip):  # noqa: F811
    """The kernels that the rules can choose, all of them in the lists."""
    forward = {f for *_, f, _ in NORMS}
    assert forward == {(16, 1, 2), (16, 1, 1)} | {(64, c, f) for c in (1, 2) for f in (0, 1)} | \
        {(256, c, f) for c in (1, 2, 4) for f in (0, 1)} | {(1024, c, f) for c in (2, 4, 8) for f in (0, 1)}
    layers = {k for *_, k in MX4_LAYERS}
    assert layers == {("few", *v, r) for v in ((1, 8, 0), (4, 4, 1), (2, 8, 1)) for r in (8, 32)} | {
        ("few", 4, 1, 1, 32), ("tile", 64, 64), ("tile", 128, 128), ("walk", 8, 8, 1)} | {("walk", s, 4, 1) for s in (1, 2, 3, 4, 8)} | {("walk", s, 8, 2) for s in (1, 2, 3, 4)}
    few, tiles = {("few", 64, 4, 2, 8), ("few48",)}, {("tile", 64, 2, 2, 4), ("tile", 128, 2, 2, 4)}
    assert {s for *_, s, _ in UPDATES} == few | tiles | {("few", 32, 8, 1, 8)}
    assert {x for *_, x in UPDATES} == few | tiles | {("few", 32, 4, 2, 4), "both"}
