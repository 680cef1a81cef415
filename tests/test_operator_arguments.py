"""Refusals of the operators' entry points, on the CPU: the library runs on a
model of the HIP runtime, whose kernels do nothing. A refused call launches
nothing and names what is wrong."""
import pytest

from host_hip_child import host_hip  # noqa: F401

SETUP = """
from chimera_amd import operators as op
L = capi.lib()
ctx = context()
hip.host_hip_reset_launches()

def rc(code, word, call, *args):
    got = call(*args)
    message = L.chimera_last_error().decode()
    assert got == code, (got, code, message)
    assert word in message, message

def refuses(call, good, field, value, word, code=1):
    old = getattr(good, field)
    setattr(good, field, value)
    rc(code, word, call)
    setattr(good, field, old)
"""


def test_linear(host_hip):  # noqa: F811
    host_hip(SETUP + """
s = op.LinearShape(100, 64, 32, 2, 0, 2, 1)
need = C.c_size_t()
assert L.chimera_linear_workspace(C.byref(s), 1, C.byref(need)) == 0 and need.value > 0
M = 1 << 20
f = op.LinearForward(M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, 7 * M, 64, 64, 32, 32, 32, 8 * M, need.value)
b = op.LinearBackward(M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, 7 * M, 8 * M, 9 * M, 10 * M, 64, 64, 32, 32, 32, 64, 64,
                      32, 11 * M, need.value)
fwd = lambda: L.chimera_linear_forward_device(ctx.handle, C.byref(s), C.byref(f))
bwd = lambda: L.chimera_linear_backward_device(ctx.handle, C.byref(s), C.byref(b))
for call in (fwd, bwd):
    for field, value, word in (("rows", -1, "negative row"), ("in_features", 0, "features"),
                               ("in_features", 65537, "features"), ("out_features", 0, "features"),
                               ("out_features", 129, "128"), ("type", 3, "type"), ("out_type", 1, "output"),
                               ("activation", 5, "activation"), ("normalize", 2, "normalize"),
                               ("rows", 1 << 32, "too many rows"), ("rows", 1 << 30, "too many rows")):
        refuses(call, s, field, value, word)
for field in ("x", "weight", "y"):
    refuses(fwd, f, field, None, "null argument: " + field)
for field in ("x", "weight", "bias", "residual", "saved"):
    refuses(fwd, f, field, M + 1, field + " is not aligned")
refuses(fwd, f, "y", M + 2, "y is not aligned")
for field, v in (("x_stride", 63), ("weight_stride", 63), ("y_stride", 31), ("residual_stride", 31), ("saved_stride", -32)):
    refuses(fwd, f, field, v, "row stride of " + field[:-7])
refuses(fwd, f, "workspace", None, "workspace", 4)
refuses(fwd, f, "workspace_bytes", 10, "workspace", 4)
refuses(fwd, f, "workspace", M + 128, "256")
s.normalize = 0
rc(1, "norms", fwd)
s.normalize = 1
for field in ("dy", "x", "weight", "saved", "y", "norms"):
    refuses(bwd, b, field, None, "null argument: " + field)
for field, v in (("dy_stride", 31), ("dx_stride", 63), ("dweight_stride", 63), ("dresidual_stride", 31)):
    refuses(bwd, b, field, v, "row stride of " + field[:-7])
refuses(bwd, b, "workspace_bytes", need.value // 1000, "workspace", 4)
# outputs lie apart from inputs and each other; columns of one matrix do
refuses(fwd, f, "y", M, "y overlaps x")
refuses(fwd, f, "saved", 2 * M + 512, "saved overlaps weight")
refuses(fwd, f, "norms", 5 * M + 64, "y overlaps norms")
refuses(fwd, f, "workspace", 4 * M, "the workspace overlaps residual")
refuses(bwd, b, "dx", 3 * M, "dx overlaps dy")
refuses(bwd, b, "dweight", 7 * M + 128, "dx overlaps dweight")
refuses(bwd, b, "dbias", 4 * M, "dbias overlaps saved")
for y, stride, code in ((M + 128, 64, 0), (M + 124, 64, 1), (M + 128, 63, 1), (M + 64, 64, 1)):
    wide = op.LinearForward.from_buffer_copy(f)
    wide.x_stride, wide.y, wide.y_stride = 128, y, stride  # rows of 256 bytes: x in 128, y in 128
    got = L.chimera_linear_forward_device(ctx.handle, C.byref(s), C.byref(wide))
    assert got == code, (stride, y, got, L.chimera_last_error())
hip.host_hip_reset_launches()
refuses(fwd, s, "in_features", 65536, "row stride")
s2 = op.LinearShape(1, 65536, 65536, 2, 2, 0, 0)
rc(1, "2^30", L.chimera_linear_workspace, C.byref(s2), 0, C.byref(need))
assert L.chimera_linear_workspace(C.byref(s), 1, C.byref(need)) == 0
rc(1, "null context", L.chimera_linear_forward_device, None, C.byref(s), C.byref(f))
rc(1, "null", L.chimera_linear_forward_device, ctx.handle, None, C.byref(f))
rc(1, "null", L.chimera_linear_forward_device, ctx.handle, C.byref(s), None)
rc(1, "null", L.chimera_linear_backward_device, ctx.handle, C.byref(s), None)
rc(1, "null", L.chimera_linear_workspace, C.byref(s), 0, None)
assert hip.host_hip_launches(b"linear") == 0
assert fwd() == 0 and bwd() == 0, L.chimera_last_error()
assert hip.host_hip_launches(b"linear") > 0
# nothing to read or write without rows
hip.host_hip_reset_launches()
s.rows = 0
empty = op.LinearForward()
assert L.chimera_linear_forward_device(ctx.handle, C.byref(s), C.byref(empty)) == 0
assert hip.host_hip_launches(b"linear") == 0
""")


def test_cache(host_hip):  # noqa: F811
    host_hip(SETUP + """
M = 1 << 20
c = op.CacheDesc(0, 96, 32, 16, 50, M, 2 * M)
row, scales = C.c_int32(), C.c_int32()
assert L.chimera_cache_row(C.byref(c), C.byref(row), C.byref(scales)) == 0 and (row.value, scales.value) == (96, 3)
i64 = C.c_int64
write = lambda rows=3 * M, type=0, stride=96, slots=4 * M, n=5: L.chimera_cache_write_device(
    ctx.handle, C.byref(c), C.c_void_p(rows), type, i64(stride), C.c_void_p(slots), i64(n))
read = lambda rows=3 * M, type=0, stride=96, slots=4 * M, n=5: L.chimera_cache_read_device(
    ctx.handle, C.byref(c), C.c_void_p(slots), i64(n), C.c_void_p(rows), type, i64(stride))
m = op.CacheMaxsim(queries=M, type=0, nq=2, query_len=32, page_start=M, doc_lens=M, pages=M, num_docs=9,
                   num_page_entries=20, max_doc_tokens=100, cand_ids=M, cand_cap=12, scores=M)
score = lambda: L.chimera_cache_maxsim_device(ctx.handle, C.byref(c), C.byref(m))
for call in (write, read, score):
    for field, value, word in (("format", 3, "format"), ("dim", 0, "dim"), ("dim", 129, "dim"), ("group", 16, "group"),
                               ("page_tokens", 12, "page"), ("page_tokens", 0, "page"), ("page_tokens", 8192, "page"),
                               ("num_pages", -1, "pages"), ("num_pages", 1 << 31, "pages"), ("codes", None, "null"),
                               ("scales", M + 4, "16 bytes")):
        refuses(call, c, field, value, word)
for call in (write, read):
    rc(1, "negative row", lambda: call(n=-1))
    rc(1, "2^28", lambda: call(n=1 << 28))
    rc(1, "type", lambda: call(type=7))
    rc(1, "null", lambda: call(rows=None))
    rc(1, "slots", lambda: call(slots=None))
    rc(1, "aligned", lambda: call(rows=M + 2))
    rc(1, "stride", lambda: call(stride=95))
for field, value, word in (("nq", -1, "queries"), ("nq", 65536, "queries"), ("query_len", 0, "query length"),
                           ("query_len", 1025, "query length"), ("cand_cap", 0, "capacity"),
                           ("cand_cap", (1 << 24) + 1, "capacity"), ("max_doc_tokens", -1, "longest"), ("type", 9, "type"),
                           ("num_docs", -1, "negative"), ("num_page_entries", -1, "negative"), ("k", -1, "negative"),
                           ("k", 3, "top-k"), ("queries", None, "queries"), ("cand_ids", None, "cand_ids"),
                           ("scores", None, "scores"), ("page_start", None, "page_start"), ("doc_lens", None, "doc_lens"),
                           ("pages", None, "pages")):
    refuses(score, m, field, value, word)
m.k, m.top_ids, m.top_counts = 3, M, M
refuses(score, m, "cand_cap", 8193, "8192")
m.k = 0
# few long documents are split, which takes a workspace
m.max_doc_tokens = 10_000
need = C.c_size_t()
assert L.chimera_cache_maxsim_workspace(C.byref(m), C.byref(need)) == 0 and need.value > 0
rc(4, "workspace", score)
m.workspace, m.workspace_bytes = M, need.value - 1
rc(4, "workspace", score)
assert hip.host_hip_launches(b"cache") == 0
m.workspace_bytes = need.value
assert score() == 0 and write() == 0 and read() == 0, L.chimera_last_error()
hip.host_hip_reset_launches()
m.nq = 0
assert write(n=0) == 0 and read(n=0) == 0 and score() == 0
assert hip.host_hip_launches(b"cache") == 0
""")


def test_python_checks(host_hip):  # noqa: F811
    host_hip(SETUP + """
from chimera_amd.store import TokenStore

def raises(kind, call, *args, **kw):
    try:
        call(*args, **kw)
    except kind:
        return
    raise AssertionError("not refused")

e = ctx.empty
w = e((32, 64), "bf16")
raises(ValueError, op.Linear, ctx, w, activation="swish")
raises(ValueError, op.Linear, ctx, e((64,), "bf16"))
raises(ValueError, op.Linear, ctx, e((32, 64), np.int32))
raises(ValueError, op.Linear, ctx, w, e((32,), np.float32))
raises(capi.ChimeraError, op.Linear, ctx, e((129, 64), "bf16"), normalize=True)
layer = op.Linear(ctx, w, e((32,), "bf16"), max_rows=100)
x, y = e((100, 64), "bf16"), e((100, 32), np.float32)
layer.forward(x, y)
raises(ValueError, layer.forward, e((100, 63), "bf16"), y)
raises(ValueError, layer.forward, e((100, 64), np.float16), y)
raises(ValueError, layer.forward, e((99, 64), "bf16"), y)
raises(ValueError, layer.forward, x, y, residual=y)
raises(ValueError, layer.forward, x, y, saved=e((100, 31), "bf16"))
raises(ValueError, layer.backward, x, y)
raises(capi.ChimeraError, layer.forward, x, e((100, 32), np.float16))
big = (e((70000, 64), "bf16"), e((70000, 32), np.float32))
raises(capi.ChimeraError, layer.forward, *big)  # more rows than the workspace was made for
codes, scales = e((64, 128), np.uint8), e((64, 1), np.float32)
cache = op.TokenCache(ctx, codes, scales)
raises(ValueError, op.TokenCache, ctx, codes, scales, format="int2")
raises(ValueError, op.TokenCache, ctx, codes, scales, format="int4")
raises(ValueError, op.TokenCache, ctx, codes, scales, page_tokens=48)
raises(ValueError, cache.write, e((3, 96), np.float32), e((3,), np.int64))
raises(ValueError, cache.write, e((3, 128), np.float32), e((4,), np.int64))
raises(ValueError, cache.read, e((3,), np.int32), e((3, 128), np.float32))
raises(ValueError, cache.read, e((3,), np.int64), e((3, 128), np.int32))
t = dict(q=e((2, 32, 128), np.float32), s=e((4,), np.int64), n=e((4,), np.int32), p=e((9,), np.int32),
         c=e((2, 5), np.int32), o=e((2, 5), np.float32))
cache.maxsim(t["q"], t["s"], t["n"], t["p"], 20, t["c"], t["o"])
raises(ValueError, cache.maxsim, e((2, 32, 64), np.float32), t["s"], t["n"], t["p"], 20, t["c"], t["o"])
raises(ValueError, cache.maxsim, t["q"], t["n"], t["n"], t["p"], 20, t["c"], t["o"])
raises(ValueError, cache.maxsim, t["q"], t["s"], t["n"], t["p"], 20, t["c"], e((2, 6), np.float32))
raises(ValueError, cache.maxsim, t["q"], t["s"], t["n"], t["p"], 20, t["c"], t["o"], query_lens=e((3,), np.int32))
raises(ValueError, TokenStore, ctx, 0)
for v in (layer, cache):
    v.close()
""")
