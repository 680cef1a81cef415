"""Arrays whose rows lie apart, given where an operator takes whole arrays:
refused, on the CPU (the library runs on a model of the HIP runtime)."""
from host_hip_child import host_hip  # noqa: F401


def test_rows_apart_where_arrays_are_whole(host_hip):  # noqa: F811
    host_hip("""
from chimera_amd import operators as op

class Apart:
    \"\"\"A view of a device array with 16 elements between rows.\"\"\"
    def __init__(self, shape, dtype):
        self.base = ctx.empty((*shape[:-1], shape[-1] + 16), dtype)
        self.ptr, self.shape, self.dtype = self.base.ptr, shape, self.base.dtype
        self.stride = shape[-1] + 16

def refuses(word, call, *args, **kw):
    hip.host_hip_reset_launches()
    try:
        call(*args, **kw)
    except ValueError as e:
        assert word in str(e), e
        assert hip.host_hip_launches(b"") == 0
        return
    raise AssertionError(word + " not refused")

ctx = context()
codes, scales = ctx.empty((64, 64), np.uint8), ctx.empty((64, 4), np.float32)
kw = dict(format="int4", dim=128, group=32)
refuses("codes", op.TokenCache, ctx, Apart((64, 64), np.uint8), scales, **kw)
refuses("scales", op.TokenCache, ctx, codes, Apart((64, 4), np.float32), **kw)
cache = op.TokenCache(ctx, codes, scales, **kw)
arrays = dict(q=((2, 32, 128), np.float32), s=((4,), np.int64), n=((4,), np.int32), p=((9,), np.int32),
              c=((2, 5), np.int32), o=((2, 5), np.float32), ti=((2, 3), np.int64), ts=((2, 3), np.float32),
              tc=((2,), np.int32))
t = {name: ctx.empty(*v) for name, v in arrays.items()}

def maxsim(**other):
    a = {**t, **other}
    cache.maxsim(a["q"], a["s"], a["n"], a["p"], 20, a["c"], a["o"], k=3, top_ids=a["ti"], top_scores=a["ts"],
                 top_counts=a["tc"])

maxsim()
for name, word in (("q", "queries"), ("c", "cand_ids"), ("o", "scores"), ("ti", "top_ids"), ("ts", "top_scores")):
    refuses(word, maxsim, **{name: Apart(*arrays[name])})
whole = Apart(*arrays["q"])
whole.stride = 32 * 128  # between queries, which follow each other
maxsim(q=whole)
# matrices of rows may lie apart, and one row is whole whatever its stride
cache.write(Apart((3, 128), np.float32), ctx.empty((3,), np.int64))
cache.read(ctx.empty((3,), np.int64), Apart((3, 128), np.float32))
one = Apart((1, 5), np.int32)
cache.maxsim(ctx.empty((1, 32, 128), np.float32), t["s"], t["n"], t["p"], 20, one, Apart((1, 5), np.float32))
""")
