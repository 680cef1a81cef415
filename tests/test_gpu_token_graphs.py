"""Graphs of late interaction that are replayed after calls of other sizes."""
import ctypes as C

import numpy as np
import pytest

from chimera_amd import capi
from operator_checks import Array, Matrix, context
from test_gpu_token_cache import Cache, corpus

pytestmark = pytest.mark.gpu


def test_replays_after_a_larger_call():
    """Documents of a captured call are split, so that it has a workspace; a
    later call takes a larger one."""
    hip = C.CDLL("libamdhip64.so.7")
    rng = np.random.default_rng(21)
    ctx = context()
    page, dim = 16, 128
    lens = np.array([700, 30, 5, 9000], np.int32)
    start, pages, slots, total = corpus(rng, lens, page)
    c = Cache(ctx, total * page, "int8", dim, 128, page)
    rows, at = Matrix(ctx, rng.standard_normal((total * page, dim)), "f32"), Array(ctx, np.arange(total * page))
    c.cache.write(rows, at)
    tables = [Array(ctx, v) for v in (start, lens, pages)]
    q = Matrix(ctx, rng.standard_normal((2, 32, dim)), "f32")
    ids, all_ids = (Array(ctx, np.tile(np.arange(n, dtype=np.int32), (2, 1))) for n in (3, 4))
    scores, all_scores = (Matrix(ctx, None, "f32", shape=(2, n)) for n in (3, 4))

    def small():
        c.cache.maxsim(q, *tables, 700, ids, scores)

    small()
    want = scores.values()
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    capi.check(capi.lib().chimera_stream(ctx.handle, C.byref(stream)))
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    small()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(3):
        c.cache.maxsim(q, *tables, 9000, all_ids, all_scores)
        other = ctx.to_device(np.zeros(1 << 20, np.uint8))  # takes memory that was given back, if any was
        assert hip.hipGraphLaunch(run, stream) == 0
        ctx.synchronize()
        assert np.array_equal(scores.values(), want) and np.array_equal(all_scores.values()[:, :3], want)
        assert not other.numpy().any()
        other.free()
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    for v in (rows, at, c, *tables, q, ids, all_ids, scores, all_scores):
        v.free()
    ctx.close()
