"""Calls captured into a HIP graph and replayed between eager calls."""
import ctypes as C

import numpy as np

from chimera_amd import capi


def check_replays(ctx, calls, results, between=None):
    """`calls()` captured once gives the eager `results()` (a list of arrays)
    at each of three replays, with eager work between them."""
    hip = C.CDLL("libamdhip64.so.7")
    calls()
    want = results()
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    capi.check(capi.lib().chimera_stream(ctx.handle, C.byref(stream)))
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    calls()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(3):
        if between is not None:
            between()
        assert hip.hipGraphLaunch(run, stream) == 0
        ctx.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))
        calls()
        ctx.synchronize()
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
