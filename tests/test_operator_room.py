"""How much memory a dense layer takes, on the CPU: the library runs on a
model of the HIP runtime."""
from host_hip_child import host_hip  # noqa: F401

SETUP = """
from chimera_amd import operators as op

ctx = context()
weight = ctx.empty((96, 768), np.float32)
ROWS, ROOM = 20_000, 96 * 768 * 4  # of a weight laid out again
FULL = ROWS * 768 * 4 + ROOM

class Apart:
    \"\"\"Rows that do not start at multiples of 16 bytes.\"\"\"
    def __init__(self, rows):
        self.base = ctx.empty((rows, 769), np.float32)
        self.ptr, self.shape, self.dtype, self.stride = self.base.ptr, (rows, 768), np.dtype(np.float32), 769

x, y = ctx.empty((ROWS, 768), np.float32), ctx.empty((ROWS, 96), np.float32)
apart = Apart(ROWS)
used = hip.host_hip_used()
layer = op.Linear(ctx, weight, normalize=True, max_rows=ROWS)
taken = lambda: hip.host_hip_used() - used
"""


def test_rows_that_are_read_as_they_lie_take_no_room(host_hip):  # noqa: F811
    host_hip(SETUP + """
layer.forward(x, y)
assert taken() <= ROOM + 4096, taken()
# the first call that lays X out takes the room for all, and graphs keep theirs
layer.forward(apart, y)
assert FULL <= taken() <= FULL + ROOM + 3 * 4096, taken()
layer.forward(x, y)
layer.forward(apart, y)
assert taken() <= FULL + ROOM + 3 * 4096
layer.close()
assert taken() == 0
""")


def test_rows_are_bounded_all_the_same(host_hip):  # noqa: F811
    """max_rows says how many rows a call may have, whether or not they would
    need the room; a room that cannot be had refuses the call and no other."""
    host_hip(SETUP + """
def fails(x, y):
    try:
        layer.forward(x, y)
    except capi.ChimeraError as e:
        return str(e)
    raise AssertionError("not refused")

more = ctx.empty((ROWS + 1, 768), np.float32), ctx.empty((ROWS + 1, 96), np.float32)
hip.host_hip_reset_launches()
assert "workspace" in fails(*more)
assert hip.host_hip_launches(b"linear") == 0
hip.host_hip_refuse_malloc(C.c_size_t(FULL), C.c_size_t(1 << 40))
assert "memory" in fails(apart, y)
layer.forward(x, y)
hip.host_hip_refuse_malloc(C.c_size_t(0), C.c_size_t(0))
layer.forward(apart, y)
""")


def test_one_allocation_where_x_is_always_laid_out(host_hip):  # noqa: F811
    """Such a layer's first call may be captured: it allocates nothing."""
    host_hip(SETUP + """
odd = ctx.empty((96, 777), np.float32)
layer = op.Linear(ctx, odd, max_rows=100)
layer.forward(ctx.empty((100, 777), np.float32), y := ctx.empty((100, 96), np.float32))
assert len(layer._workspaces) == 1
training = op.Linear(ctx, weight, max_rows=100, training=True)
training.forward(x2 := Apart(100), y)
training.backward(x2, y, dx=ctx.empty((100, 768), np.float32))
assert len(training._workspaces) == 1
""")
