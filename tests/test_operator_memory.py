"""Memory that the operators' objects hold, on the CPU: the library runs on a
model of the HIP runtime with a set capacity and failing allocations."""
from host_hip_child import host_hip  # noqa: F401

SETUP = """
from chimera_amd import operators as op

def fails(call, *args, **kw):
    try:
        call(*args, **kw)
    except capi.ChimeraError as e:
        return str(e)
    raise AssertionError("not refused")

def maxsim(ctx, cache, tokens, nq=1, cap=4):
    bufs = [ctx.empty(s, t) for s, t in (((nq, 32, 128), np.float32), ((4,), np.int64), ((4,), np.int32),
                                          ((9,), np.int32), ((nq, cap), np.int32), ((nq, cap), np.float32))]
    try:
        cache.maxsim(bufs[0], bufs[1], bufs[2], bufs[3], tokens, bufs[4], bufs[5])
    finally:
        for b in bufs:
            b.free()

def held(owner, args):
    \"\"\"Bytes of the workspace that a call would use, which its owner has to hold.\"\"\"
    if not args.workspace:
        return 0
    assert owner._workspace is not None and owner._workspace.ptr == args.workspace, "freed memory"
    assert owner._workspace.nbytes >= args.workspace_bytes
    return args.workspace_bytes

ctx = context()
cache = op.TokenCache(ctx, ctx.empty((64, 128), np.uint8), ctx.empty((64, 1), np.float32))
"""


def test_a_workspace_that_cannot_grow(host_hip):  # noqa: F811
    """The call that needs a larger one fails; those that fitted go on."""
    host_hip(SETUP + """
maxsim(ctx, cache, 1000)
small = held(cache, cache._args)
assert small > 0
hip.host_hip_refuse_malloc(C.c_size_t(100_000), C.c_size_t(1 << 40))  # the larger workspace alone
assert "memory" in fails(maxsim, ctx, cache, 60_000)
hip.host_hip_refuse_malloc(C.c_size_t(0), C.c_size_t(0))
maxsim(ctx, cache, 1000)
assert held(cache, cache._args) == small
maxsim(ctx, cache, 60_000)
assert held(cache, cache._args) > small
""")


def test_calls_after_close(host_hip):  # noqa: F811
    """What needs a workspace is refused; nothing points to freed memory."""
    host_hip(SETUP + """
maxsim(ctx, cache, 1000)
cache.close()
hip.host_hip_reset_launches()
assert "workspace" in fails(maxsim, ctx, cache, 1000)
assert hip.host_hip_launches(b"cache") == 0 and held(cache, cache._args) == 0
maxsim(ctx, cache, 20)  # takes none
layer = op.Linear(ctx, ctx.empty((32, 64), "bf16"), max_rows=10, training=True)
x, y = ctx.empty((10, 64), "bf16"), ctx.empty((10, 32), "bf16")
layer.forward(x, y)
layer.backward(x, y, dx=ctx.empty((10, 64), "bf16"))
layer.close()
hip.host_hip_reset_launches()
assert "workspace" in fails(layer.forward, x, y)
assert "workspace" in fails(layer.backward, x, y, dx=ctx.empty((10, 64), "bf16"))
assert hip.host_hip_launches(b"linear") == 0 and held(layer, layer._forward) == held(layer, layer._backward) == 0
""")


def test_outgrown_workspaces_stay_for_graphs(host_hip):  # noqa: F811
    """A captured call's workspace stays allocated while later calls take
    larger ones, up to close()."""
    host_hip(SETUP + """
begin = hip.host_hip_used()
kept = {}
for tokens in (600, 1000, 3000, 20_000, 60_000, 200_000):
    maxsim(ctx, cache, tokens)
    kept[cache._args.workspace] = -(-cache._workspace.nbytes // 4096) * 4096
    assert hip.host_hip_used() - begin == sum(kept.values())
assert len(kept) > 2 and sum(kept.values()) <= 2 * held(cache, cache._args) + 4096 * len(kept)
cache.close()
assert hip.host_hip_used() == begin
""")
