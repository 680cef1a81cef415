"""Numbers that do not fit the ABI's 32 bits, and page sizes that no call
takes: refused where they are given, on the CPU (the library runs on a model
of the HIP runtime)."""
from host_hip_child import host_hip  # noqa: F401

SETUP = """
from chimera_amd import operators as op
from chimera_amd.store import TokenStore

def refuses(word, call, *args, **kw):
    try:
        call(*args, **kw)
    except (ValueError, capi.ChimeraError) as e:
        assert word in str(e), e
        return
    raise AssertionError(word + " not refused")

ctx = context()
codes, scales = ctx.empty((96, 128), np.uint8), ctx.empty((96, 1), np.float32)
BIG = 1 << 32
"""


def test_numbers_past_32_bits(host_hip):  # noqa: F811
    host_hip(SETUP + """
refuses("dim", op.cache_row, "int8", BIG + 128, 128)
refuses("group", op.cache_row, "int8", 128, BIG + 128)
refuses("group", op.TokenCache, ctx, codes, scales, group=BIG + 128)
cache = op.TokenCache(ctx, codes, scales)
e = ctx.empty
a = [e((1, 32, 128), np.float32), e((4,), np.int64), e((4,), np.int32), e((9,), np.int32)]
ids, scores = e((1, 5), np.int32), e((1, 5), np.float32)
hip.host_hip_reset_launches()
refuses("max_doc_tokens", cache.maxsim, *a, BIG + 5, ids, scores)  # 5 tokens of each would be scored
refuses("k", cache.maxsim, *a, 5, ids, scores, k=BIG)               # no top-k would be taken
assert hip.host_hip_launches(b"cache") == 0
refuses("tokens", cache.maxsim, *a, -1, ids, scores)
cache.maxsim(*a, 5, ids, scores)
""")


def test_page_sizes(host_hip):  # noqa: F811
    host_hip(SETUP + """
used = hip.host_hip_used()
for tokens in (48, 0, 3):
    refuses("page", op.TokenCache, ctx, codes, scales, page_tokens=tokens)
    refuses("page", TokenStore, ctx, 10, page_tokens=tokens)
refuses("page", TokenStore, ctx, 10, page_tokens=8192)
assert hip.host_hip_used() == used
""")


def test_strides_past_the_address_space(host_hip):  # noqa: F811
    """A matrix whose last row's offset does not fit 62 bits."""
    host_hip(SETUP + """
L = capi.lib()
M = 1 << 20
s = op.LinearShape(100, 64, 32, 0, 0, 2, 0)
need = C.c_size_t()
capi.check(L.chimera_linear_workspace(C.byref(s), 1, C.byref(need)))
f = op.LinearForward(M, 2 * M, 3 * M, 4 * M, 5 * M, 6 * M, None, 64, 64, 32, 32, 32, 8 * M, need.value)
b = op.LinearBackward(M, 2 * M, 3 * M, 4 * M, 5 * M, None, 7 * M, 8 * M, 9 * M, 10 * M, 64, 64, 32, 32, 32, 64, 64,
                      32, 11 * M, need.value)
fwd = lambda: L.chimera_linear_forward_device(ctx.handle, C.byref(s), C.byref(f))
bwd = lambda: L.chimera_linear_backward_device(ctx.handle, C.byref(s), C.byref(b))
assert fwd() == 0 and bwd() == 0
hip.host_hip_reset_launches()
for call, args, names in ((fwd, f, ("x", "weight", "residual", "y", "saved")),
                          (bwd, b, ("x", "weight", "dy", "saved", "dx", "dweight", "dresidual"))):
    for name in names:
        for stride in (1 << 61, (1 << 63) - 1, (1 << 60) // 25):
            old = getattr(args, name + "_stride")
            setattr(args, name + "_stride", stride)
            assert call() == 1 and b"stride of " + name.encode() in L.chimera_last_error(), (name, stride)
            setattr(args, name + "_stride", old)
c = op.CacheDesc(0, 128, 128, 16, 6, codes.ptr, scales.ptr)
for stride in (1 << 61, (1 << 63) - 1):
    assert L.chimera_cache_write_device(ctx.handle, C.byref(c), C.c_void_p(M), 0, C.c_int64(stride), C.c_void_p(2 * M),
                                        C.c_int64(9)) == 1
    assert L.chimera_cache_read_device(ctx.handle, C.byref(c), C.c_void_p(M), C.c_int64(9), C.c_void_p(2 * M), 0,
                                       C.c_int64(stride)) == 1
assert hip.host_hip_launches(b"") == 0
# one row lies where it lies
s.rows, f.x_stride = 1, 1 << 59
assert fwd() == 0, L.chimera_last_error()
""")
