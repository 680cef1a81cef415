"""What calls that fail leave of a TokenStore, on the CPU: the library runs on
a model of the HIP runtime with failing allocations."""
from host_hip_child import host_hip  # noqa: F401

SETUP = """
from chimera_amd.store import TokenStore

ctx = context()
store = TokenStore(ctx, num_pages=20, dim=64, group=64, page_tokens=8)

def rows(n):
    return np.ones((n, 64), np.float32)

def state():
    docs = range(len(store._docs))
    return (store.free_tokens, list(store._free), [store._docs[d] and list(store._docs[d]) for d in docs],
            list(store._lens), list(store._unused), hip.host_hip_used())

def leaves_all(kind, call, *args):
    before = state()
    try:
        call(*args)
    except kind:
        assert state() == before, (before, state())
        return
    raise AssertionError("not refused")
"""


def test_a_write_that_fails_leaves_the_documents(host_hip):  # noqa: F811
    host_hip(SETUP + """
a, b, c = store.add(rows(3 + 17 + 8), [3, 17, 8])
store.remove(b)
whole = ctx.empty((5, 64), np.int32)  # not an element type
five = ctx.empty((5, 64), np.float32)
store.tables()
leaves_all(ValueError, store.append, a, whole)
leaves_all(ValueError, store.add, whole, [5])
leaves_all(ValueError, store.add, whole, [2, 3])
leaves_all(ValueError, store.add, np.ones(64, np.float32), [1])
assert store.doc_len(a) == 3
# no memory for the slots
hip.host_hip_refuse_malloc(C.c_size_t(40), C.c_size_t(40))
leaves_all(capi.ChimeraError, store.append, a, five)
leaves_all(capi.ChimeraError, store.add, five, [5])
leaves_all(capi.ChimeraError, store.append, c, five)
hip.host_hip_refuse_malloc(C.c_size_t(0), C.c_size_t(0))
store.append(a, five)
(d,) = store.add(five, [5])
assert d == b and store.doc_len(a) == 8 and store.doc_len(d) == 5
# pages are not given twice
held = [p for pages in store._docs if pages for p in pages] + store._free
assert sorted(held) == list(range(20))
""")


def test_ids_and_lengths_past_32_bits(host_hip):  # noqa: F811
    """64-bit ids, as a search returns them: those that are no document's
    are absent, not cut to another document's."""
    host_hip(SETUP + """
store.add(rows(24), [8, 8, 8])
seen = {}

def maxsim(q, start, lens, pages, longest, ids, scores, query_lens=None, **kw):
    seen.update(ids=ids.numpy(), lens=query_lens.numpy())

store.cache.maxsim = maxsim
big = 1 << 32
ids = np.array([[0, 2, -1, 1 << 31, big, big + 1, -big, 2**63 - 1]], np.int64)
store.rescore(np.zeros((1, 4, 64), np.float32), ids, 2, query_lens=np.array([big + 1], np.int64))
assert seen["ids"].tolist() == [[0, 2, -1, -1, -1, -1, -1, -1]], seen
assert seen["lens"].tolist() == [4]
store.rescore(np.zeros((1, 4, 64), np.float32), ids.astype(np.uint64), 2, query_lens=np.array([-big - 3], np.int64))
assert seen["ids"].tolist() == [[0, 2, -1, -1, -1, -1, -1, -1]] and seen["lens"].tolist() == [0]
""")


def test_allocations_that_fail_leave_no_memory(host_hip):  # noqa: F811
    """Every allocation of every call in turn."""
    host_hip(SETUP + """
empty, left = ctx.empty, [0]

def counted(shape, dtype):
    left[0] -= 1
    if left[0] < 0:
        raise capi.ChimeraError(2, "out of memory")
    return empty(shape, dtype)

def to_device(a, bf16=False):
    a = np.ascontiguousarray(a)
    d = counted(a.shape, a.dtype)
    capi.check(capi.lib().chimera_copy_to_device(ctx.handle, capi.P(d.ptr), capi._ptr(a), C.c_size_t(a.nbytes)))
    return d

def each(call, least):
    \"\"\"Lets the first, second, ... allocation of the call fail, until it ends.\"\"\"
    for n in range(100):
        left[0] = n
        used = hip.host_hip_used()
        ctx.empty, ctx.to_device = counted, to_device
        try:
            call()
        except capi.ChimeraError:
            assert hip.host_hip_used() == used, (call, n)
            continue
        finally:
            ctx.empty, ctx.to_device = empty, type(ctx).to_device.__get__(ctx)
        assert n >= least, n
        return
    raise AssertionError("does not end")

each(lambda: TokenStore(ctx, 8).close(), 2)
each(lambda: store.add(rows(11), [3, 8]), 2)
each(lambda: store.append(0, rows(9)), 2)
each(lambda: store.read(0), 2)
store.append(0, rows(1))
each(lambda: store.tables(), 3)
q = np.zeros((2, 4, 64), np.float32)
each(lambda: store.rescore(q, np.zeros((2, 5), np.int64), 2, query_lens=[1, 2]), 7)
# one document of 600 tokens, so that the cache takes a workspace
store.close()
store = TokenStore(ctx, num_pages=100, dim=64, group=64, page_tokens=8)
store.add(rows(600), [600])
store.tables()
each(lambda: store.rescore(q, np.zeros((2, 5), np.int64), 2), 7)  # the cache's too
""")
