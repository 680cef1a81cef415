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
