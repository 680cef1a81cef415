"""Refusals of the dense stack's entry points (layer norm, 4-bit layers,
orthogonal updates), on the CPU: the library runs on a model of the HIP
runtime, whose kernels do nothing. A refused call launches nothing and names
what is wrong."""
from host_hip_child import host_hip  # noqa: F401
from test_operator_arguments import SETUP

def test_norm(host_hip):  # noqa: F811
    host_hip(SETUP + """
M = 1 << 20
s = op.NormShape(100, 64, 2, 0, 1e-5)
need = C.c_size_t()
assert L.chimera_norm_workspace(C.byref(s), C.byref(need)) == 0 and need.value > 0
f = op.NormForward(M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, 64, 64)
b = op.NormBackward(M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, 7 * M, 8 * M, 64, 64, 64, 9 * M, need.value)
fwd = lambda: L.chimera_norm_forward_device(ctx.handle, C.byref(s), C.byref(f))
bwd = lambda: L.chimera_norm_backward_device(ctx.handle, C.byref(s), C.byref(b))
for call in (fwd, bwd):
    for field, value, word in (("rows", -1, "negative row"), ("rows", (1 << 31) + 1, "2^31"), ("features", 0, "features"),
                               ("features", 65537, "features"), ("type", 3, "type"), ("out_type", 1, "output"),
                               ("eps", 0.0, "eps"), ("eps", -1.0, "eps"), ("eps", float("nan"), "eps"),
                               ("eps", float("inf"), "eps")):
        refuses(call, s, field, value, word)
for field in ("x", "y"):
    refuses(fwd, f, field, None, "null argument: " + field)
for field in ("x", "weight", "bias"):
    refuses(fwd, f, field, M + 1, field + " is not aligned")
for field in ("y", "mean", "rstd"):
    refuses(fwd, f, field, M + 2, field + " is not aligned")
for args, call, names in ((f, fwd, ("x", "y")), (b, bwd, ("x", "dy", "dx"))):
    for name in names:
        refuses(call, args, name + "_stride", 63, "row stride of " + name)
        for stride in (1 << 61, (1 << 63) - 1):
            refuses(call, args, name + "_stride", stride, "row stride of " + name)
refuses(fwd, f, "y", M, "y overlaps x")
refuses(fwd, f, "mean", 4 * M + 64, "y overlaps mean")
refuses(fwd, f, "rstd", 2 * M, "rstd overlaps weight")
for field in ("x", "dy", "mean", "rstd"):
    refuses(bwd, b, field, None, "null argument: " + field)
refuses(bwd, b, "workspace", None, "workspace", 4)
refuses(bwd, b, "workspace_bytes", need.value - 1, "workspace", 4)
refuses(bwd, b, "workspace", 9 * M + 128, "256")
refuses(bwd, b, "dx", 3 * M, "dx overlaps dy")
refuses(bwd, b, "dweight", 8 * M + 64, "dweight overlaps dbias")
refuses(bwd, b, "dbias", 5 * M, "dbias overlaps rstd")
refuses(bwd, b, "workspace", M, "the workspace overlaps x")
rc(1, "null context", L.chimera_norm_forward_device, None, C.byref(s), C.byref(f))
rc(1, "null", L.chimera_norm_forward_device, ctx.handle, None, C.byref(f))
rc(1, "null", L.chimera_norm_forward_device, ctx.handle, C.byref(s), None)
rc(1, "null", L.chimera_norm_backward_device, ctx.handle, C.byref(s), None)
rc(1, "null", L.chimera_norm_workspace, C.byref(s), None)
assert hip.host_hip_launches(b"norm") == 0
assert fwd() == 0 and bwd() == 0, L.chimera_last_error()
assert hip.host_hip_launches(b"norm_forward") == 1 and hip.host_hip_launches(b"norm_backward") == 1
# without sums over rows there is no workspace; without rows nothing is read
b.dweight = b.dbias = b.workspace = None
assert bwd() == 0, L.chimera_last_error()
hip.host_hip_reset_launches()
s.rows = 0
empty = op.NormForward()
assert L.chimera_norm_forward_device(ctx.handle, C.byref(s), C.byref(empty)) == 0
assert hip.host_hip_launches(b"norm") == 0
""")


def test_mx4(host_hip):  # noqa: F811
    host_hip(SETUP + """
M = 1 << 20
i64, i32 = C.c_int64, C.c_int32
row, scales = i32(), i32()
for k, want in ((1, (16, 8)), (32, (16, 8)), (33, (32, 8)), (256, (128, 8)), (257, (144, 16)), (65536, (32768, 2048))):
    assert L.chimera_mx4_row(k, C.byref(row), C.byref(scales)) == 0 and (row.value, scales.value) == want
for k in (0, -1, 65537):
    rc(1, "features", L.chimera_mx4_row, k, C.byref(row), C.byref(scales))
rc(1, "null", L.chimera_mx4_row, 8, None, C.byref(scales))
write = lambda rows=M, type=0, stride=96, n=5, k=96, codes=2 * M, scales=3 * M: L.chimera_mx4_quantise_device(
    ctx.handle, C.c_void_p(rows), type, i64(stride), i64(n), k, C.c_void_p(codes), C.c_void_p(scales))
read = lambda rows=M, type=0, stride=96, n=5, k=96, codes=2 * M, scales=3 * M: L.chimera_mx4_read_device(
    ctx.handle, C.c_void_p(codes), C.c_void_p(scales), i64(n), k, C.c_void_p(rows), type, i64(stride))
for call in (write, read):
    rc(1, "negative row", lambda: call(n=-1))
    rc(1, "2^28", lambda: call(n=1 << 28))
    rc(1, "features", lambda: call(k=0))
    rc(1, "features", lambda: call(k=65537, stride=65537))
    rc(1, "type", lambda: call(type=7))
    rc(1, "null", lambda: call(rows=None))
    rc(1, "aligned", lambda: call(rows=M + 2))
    rc(1, "stride", lambda: call(stride=95))
    rc(1, "stride", lambda: call(stride=1 << 61))
    rc(1, "codes", lambda: call(codes=None))
    rc(1, "codes is not aligned", lambda: call(codes=M + 8))
    rc(1, "scales", lambda: call(scales=None))
    rc(1, "scales is not aligned", lambda: call(scales=M + 4))
    rc(1, "overlaps", lambda: call(codes=M + 64))
    rc(1, "overlaps", lambda: call(scales=M + 64))
rc(1, "codes overlaps scales", lambda: write(scales=2 * M + 16))
short = op.LinearShape(100, 64, 129, 2, 0, 2, 1)
need = C.c_size_t()
rc(1, "128", L.chimera_mx4_linear_workspace, C.byref(short), C.byref(need))
short.out_features = 128
assert L.chimera_mx4_linear_workspace(C.byref(short), C.byref(need)) == 0 and need.value == 0  # quantised on its way
s = op.LinearShape(3000, 64, 544, 2, 0, 2, 0)
assert L.chimera_mx4_linear_workspace(C.byref(s), C.byref(need)) == 0 and need.value > 0
M = 1 << 24
f = op.Mx4LinearArgs(M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, 64, 544, 544, 7 * M, need.value)
layer = lambda: L.chimera_mx4_linear_device(ctx.handle, C.byref(s), C.byref(f))
for field, value, word in (("rows", -1, "negative row"), ("in_features", 0, "features"), ("in_features", 65537, "features"),
                           ("normalize", 1, "128"), ("type", 3, "type"), ("out_type", 1, "output"),
                           ("activation", 5, "activation"), ("normalize", 2, "normalize"), ("rows", 1 << 32, "too many rows")):
    refuses(layer, s, field, value, word)
for field in ("x", "codes", "scales", "y"):
    refuses(layer, f, field, None, "null argument: " + field)
for field, v in (("x", M + 1), ("codes", M + 8), ("scales", M + 4), ("bias", M + 1), ("residual", M + 1), ("y", M + 2)):
    refuses(layer, f, field, v, field + " is not aligned")
for field, v in (("x_stride", 63), ("y_stride", 543), ("residual_stride", 543), ("y_stride", 1 << 61)):
    refuses(layer, f, field, v, "row stride of " + field[:-7])
refuses(layer, f, "workspace", None, "workspace", 4)
refuses(layer, f, "workspace_bytes", 10, "workspace", 4)
refuses(layer, f, "workspace", M + 128, "256")
refuses(layer, f, "y", M, "y overlaps x")
refuses(layer, f, "y", 2 * M + 512, "y overlaps codes")
refuses(layer, f, "workspace", 3 * M, "the workspace overlaps scales")
rc(1, "null", L.chimera_mx4_linear_device, ctx.handle, None, C.byref(f))
rc(1, "null", L.chimera_mx4_linear_device, ctx.handle, C.byref(s), None)
rc(1, "null", L.chimera_mx4_linear_workspace, C.byref(s), None)
assert hip.host_hip_launches(b"mx4") == 0
assert write() == 0 and read() == 0 and layer() == 0, L.chimera_last_error()
assert hip.host_hip_launches(b"mx4") > 2
hip.host_hip_reset_launches()
s.rows = 0
assert write(n=0) == 0 and read(n=0) == 0 and layer() == 0
assert hip.host_hip_launches(b"mx4") == 0
""")


def test_orthogonal(host_hip):  # noqa: F811
    host_hip(SETUP + """
M = 1 << 20
s = op.OrthogonalShape(96, 64, 2, 0, 5, 3.4445, -4.775, 2.0315)
need = C.c_size_t()
assert L.chimera_orthogonal_workspace(C.byref(s), C.byref(need)) == 0 and need.value > 0
g = op.OrthogonalArgs(M, 2 * M, 3 * M, 0.9, 1, 4 * M, 5 * M, 6 * M, 7 * M, 0.1, 0.01, 64, 64, 64, 64, 64, 64, 64, 8 * M, need.value)
call = lambda: L.chimera_orthogonal_update_device(ctx.handle, C.byref(s), C.byref(g))
nan, inf = float("nan"), float("inf")
for field, value, word in (("rows", 0, "rows and columns"), ("cols", 0, "rows and columns"), ("rows", 65537, "rows and columns"),
                           ("type", 3, "type"), ("out_type", 1, "output"), ("steps", 0, "steps"), ("steps", 101, "steps"),
                           ("a", nan, "finite"), ("b", inf, "finite"), ("c", -inf, "finite")):
    refuses(call, s, field, value, word)
for rows, cols, word in ((8193, 8193, "shorter side"), (65536, 8192, "2^28")):
    wide = op.OrthogonalShape(rows, cols, 2, 0, 5, 1.0, 0.0, 0.0)
    rc(1, word, L.chimera_orthogonal_workspace, C.byref(wide), C.byref(need))
assert L.chimera_orthogonal_workspace(C.byref(s), C.byref(need)) == 0
for field, value, word in (("nesterov", 2, "nesterov"), ("mu", nan, "finite"), ("rate", inf, "finite"), ("decay", nan, "finite"),
                           ("gradient", None, "null argument: gradient"), ("new_momentum", None, "null argument: new_momentum"),
                           ("new_weight", None, "null argument: new_weight"), ("gradient", M + 1, "gradient is not aligned"),
                           ("momentum", M + 2, "momentum is not aligned"), ("weight", M + 2, "weight is not aligned"),
                           ("rounded", M + 1, "rounded is not aligned"), ("out", M + 2, "out is not aligned"),
                           ("workspace", 8 * M + 128, "256")):
    refuses(call, g, field, value, word)
for name in ("gradient", "momentum", "new_momentum", "out", "weight", "new_weight", "rounded"):
    for stride in (63, 1 << 61):
        refuses(call, g, name + "_stride", stride, "row stride of " + name)
refuses(call, g, "workspace", None, "workspace", 4)
refuses(call, g, "workspace_bytes", need.value - 1, "workspace", 4)
refuses(call, g, "out", M, "out overlaps gradient")
refuses(call, g, "new_momentum", 2 * M + 64, "new_momentum overlaps momentum")
refuses(call, g, "new_weight", 5 * M + 64, "new_weight overlaps weight")
refuses(call, g, "rounded", 6 * M, "new_weight overlaps rounded")
refuses(call, g, "new_weight", 2 * M, "new_weight overlaps momentum")
refuses(call, g, "workspace", 5 * M, "the workspace overlaps weight")
# in its place only with the same rows
g.new_momentum = g.momentum
refuses(call, g, "new_momentum_stride", 65, "new_momentum overlaps momentum")
g.new_weight = g.weight
refuses(call, g, "new_weight_stride", 65, "new_weight overlaps weight")
rc(1, "null context", L.chimera_orthogonal_update_device, None, C.byref(s), C.byref(g))
rc(1, "null", L.chimera_orthogonal_update_device, ctx.handle, None, C.byref(g))
rc(1, "null", L.chimera_orthogonal_update_device, ctx.handle, C.byref(s), None)
rc(1, "null", L.chimera_orthogonal_workspace, C.byref(s), None)
assert hip.host_hip_launches(b"orthogonal") == 0
assert call() == 0, L.chimera_last_error()
assert hip.host_hip_launches(b"orthogonal") > 10
g.out = None
assert call() == 0, L.chimera_last_error()
g.weight = None
rc(1, "out and weight", call)
""")


def test_python_checks(host_hip):  # noqa: F811
    host_hip(SETUP + """
def raises(kind, call, *args, **kw):
    try:
        call(*args, **kw)
    except kind as e:
        return str(e)
    raise AssertionError("not refused")

e = ctx.empty
x, y = e((100, 64), "bf16"), e((100, 64), np.float32)
# layer norm
raises(ValueError, op.LayerNorm, ctx)
raises(ValueError, op.LayerNorm, ctx, features=64, type="int8")
raises(ValueError, op.LayerNorm, ctx, e((2, 64), "bf16"))
raises(ValueError, op.LayerNorm, ctx, e((64,), "bf16"), e((64,), np.float32))
raises(ValueError, op.LayerNorm, ctx, e((64,), "bf16"), e((65,), "bf16"))
raises(ValueError, op.LayerNorm, ctx, e((64,), np.int32))
raises(capi.ChimeraError, op.LayerNorm, ctx, e((64,), "bf16"), eps=0.0)
raises(ValueError, op.LayerNorm, ctx, features=(1 << 32) + 64, type="f32")
norm = op.LayerNorm(ctx, e((64,), "bf16"), max_rows=100, training=True)
stat = e((100,), np.float32)
norm.forward(x, y, mean=stat, rstd=e((100,), np.float32))
raises(ValueError, norm.forward, e((100, 63), "bf16"), y)
raises(ValueError, norm.forward, y, y)
raises(ValueError, norm.forward, x, e((99, 64), np.float32))
raises(ValueError, norm.forward, x, y, mean=e((99,), np.float32))
raises(capi.ChimeraError, norm.forward, x, e((100, 64), np.float16))
raises(ValueError, norm.backward, x, e((99, 64), np.float32), stat, stat)
raises(ValueError, norm.backward, x, y, e((100,), np.float16), stat)
raises(ValueError, norm.backward, x, y, stat, stat, dx=y)
raises(ValueError, norm.backward, x, y, stat, stat, dweight=e((65,), "bf16"))
norm.backward(x, y, stat, stat, dx=e((100, 64), "bf16"), dweight=e((64,), "bf16"))
many = e((9000, 64), "bf16"), e((9000, 64), np.float32), e((9000,), np.float32), e((9000,), np.float32)
assert "workspace" in raises(capi.ChimeraError, norm.backward, *many, dweight=e((64,), "bf16"))
norm.forward(many[0], many[1])  # needs none
raises(ValueError, op.LayerNorm(ctx, e((64,), "bf16")).backward, x, y, stat, stat)
used = hip.host_hip_used()
norm.close()
assert hip.host_hip_used() < used
assert "workspace" in raises(capi.ChimeraError, norm.backward, x, y, stat, stat, dweight=e((64,), "bf16"))
norm.forward(x, y)
# 4-bit rows and layers
raises(ValueError, op.mx4_row, (1 << 32) + 64)
codes, scales = e((100, 32), np.uint8), e((100, 8), np.uint8)
op.mx4_quantise(ctx, x, codes, scales)
op.mx4_read(ctx, codes, scales, y)
raises(ValueError, op.mx4_quantise, ctx, x, e((100, 31), np.uint8), scales)
raises(ValueError, op.mx4_quantise, ctx, x, e((99, 32), np.uint8), scales)
raises(ValueError, op.mx4_quantise, ctx, x, codes, e((100, 2), np.uint8))
raises(ValueError, op.mx4_quantise, ctx, e((100, 64), np.int32), codes, scales)
raises(ValueError, op.mx4_read, ctx, codes, scales, e((100, 65), np.float32))
class Apart:
    ptr, shape, dtype, stride = codes.ptr, (50, 32), np.dtype(np.uint8), 64
raises(ValueError, op.mx4_read, ctx, Apart(), e((50, 8), np.uint8), e((50, 64), np.float32))
raises(ValueError, op.Mx4Linear, ctx, codes, scales, 65)
raises(ValueError, op.Mx4Linear, ctx, codes, scales, 64, activation="swish")
raises(ValueError, op.Mx4Linear, ctx, codes, scales, 64, type="int4")
raises(ValueError, op.Mx4Linear, ctx, codes, scales, 64, bias=e((100,), np.float32))
raises(capi.ChimeraError, op.Mx4Linear, ctx, e((129, 32), np.uint8), e((129, 8), np.uint8), 64, normalize=True)
layer = op.Mx4Linear(ctx, codes, scales, 64, max_rows=8000)
out = e((100, 100), np.float32)
layer.forward(x, out)
raises(ValueError, layer.forward, y, out)
raises(ValueError, layer.forward, x, y)
raises(ValueError, layer.forward, x, out, residual=out)
raises(capi.ChimeraError, layer.forward, x, e((100, 100), np.float16))
assert "workspace" in raises(capi.ChimeraError, layer.forward, many[0], e((9000, 100), np.float32))
eight = e((8000, 64), "bf16"), e((8000, 100), np.float32)
layer.forward(*eight)
layer.close()
assert "workspace" in raises(capi.ChimeraError, layer.forward, *eight)
layer.forward(x, out)  # needs none
# orthogonal update
raises(ValueError, op.OrthogonalUpdate, ctx, 32, 64, type="int8")
raises(ValueError, op.OrthogonalUpdate, ctx, (1 << 32) + 32, 64)
raises(capi.ChimeraError, op.OrthogonalUpdate, ctx, 32, 64, steps=0)
update = op.OrthogonalUpdate(ctx, 32, 64, type="bf16")
g, w, o = e((32, 64), "bf16"), e((32, 64), np.float32), e((32, 64), "bf16")
update.orthogonalize(g, o)
update.step(g, w)
update.step(g, w, momentum=e((32, 64), np.float32), rounded=o)
raises(ValueError, update.orthogonalize, w, o)
raises(ValueError, update.orthogonalize, g, e((32, 65), "bf16"))
raises(ValueError, update.orthogonalize, g, o, new_momentum=w)
raises(ValueError, update.step, g, g)
raises(ValueError, update.step, g, w, rounded=w)
raises(capi.ChimeraError, update.step, g, w, rate=float("nan"))
raises(capi.ChimeraError, update.orthogonalize, g, e((32, 64), np.float16))
update.orthogonalize(g, o)  # nothing of the refused calls is left
update.close()
assert "workspace" in raises(capi.ChimeraError, update.orthogonalize, g, o)
""")


def test_workspaces_grow_with_the_rows(host_hip):  # noqa: F811
    """A workspace made for some rows serves fewer."""
    host_hip(SETUP + """
rng = np.random.default_rng(3)
need = [C.c_size_t(), C.c_size_t()]
for i in range(20_000):
    k, n = (int(2 ** rng.uniform(0, 16)) for _ in range(2))
    n = min(n, (1 << 30) // k)
    rows = sorted(int(2 ** rng.uniform(0, 18)) for _ in range(2))
    if i % 2:
        rows[0] = max(1, rows[1] - int(rng.integers(0, 600)))
    for r, v in zip(rows, need):
        capi.check(L.chimera_norm_workspace(C.byref(op.NormShape(r, k, 2, 2, 1e-5)), C.byref(v)))
    assert need[0].value <= need[1].value, (rows, k)
    if (rows[1] + 127) // 128 * ((max(k, n) + 127) // 128) > 1 << 21:
        continue
    for r, v in zip(rows, need):
        capi.check(L.chimera_mx4_linear_workspace(C.byref(op.LinearShape(r, k, n, 2, 2, 0, 0)), C.byref(v)))
    assert need[0].value <= need[1].value, (rows, k, n)
""")
