"""Which kernels the shapes of operator_shapes take, on the CPU: the library
runs on a model of the HIP runtime that counts launches."""
from host_hip_child import host_hip  # noqa: F401
from operator_shapes import GRADIENTS, LARGE, LAYERS, NORMALIZED, WALKS

SETUP = """
from chimera_amd import operators as op
L = capi.lib()
ctx = context()
A = 1 << 40  # arrays apart from each other; nothing reads them
NAME = {"f32": "f", "f16": "DF16_", "bf16": "DF16b"}
TILES = {"256": (256, 256, 2, 4), "128": (128, 128, 2, 2), "64": (64, 64, 2, 2), "128 x 128": (128, 128, 4, 1),
         "32 x 128": (32, 128, 1, 4), "32 x 96": (32, 96, 1, 3), "64 x 64": (64, 64, 2, 2)}
ENDS = {"layer": "Lb0ELb0ELNS0_3EndE1E", "normalized": "Lb0ELb0ELNS0_3EndE2E", "dx": "Lb0ELb1ELNS0_3EndE0E",
        "dw": "Lb1ELb1ELNS0_3EndE0E"}

def launches(part):
    return hip.host_hip_launches(part.encode())

def tile(type, end, name):
    \"\"\"Launches of the tiled product for `end` on the tile `name`.\"\"\"
    tiles = "".join(f"Li{v}E" for v in TILES[name])
    found = [s for s in ("Li3ELi2E", "Li3ELi3E") if launches(f"linear_tile_kernelI{NAME[type]}{tiles}{s}{ENDS[end]}")]
    return len(found)

def shape(rows, k, n, type, normalize=0):
    s = op.LinearShape(rows, k, n, op.TYPES[type], op.TYPES[type], 0, normalize)
    need = C.c_size_t()
    capi.check(L.chimera_linear_workspace(C.byref(s), 1, C.byref(need)))
    hip.host_hip_reset_launches()
    return s, need.value

def forward(*args, **kw):
    s, need = shape(*args, **kw)
    k, n = s.in_features, s.out_features
    f = op.LinearForward(A, 2 * A, None, None, 5 * A, None, None, k, k, n, n, n, 8 * A, need)
    capi.check(L.chimera_linear_forward_device(ctx.handle, C.byref(s), C.byref(f)))

def backward(*args, **kw):
    s, need = shape(*args, **kw)
    k, n = s.in_features, s.out_features
    b = op.LinearBackward(A, 2 * A, 3 * A, 4 * A, 5 * A, 6 * A, 7 * A, 8 * A, None, None, k, k, n, n, n, k, k, n,
                          10 * A, need)
    capi.check(L.chimera_linear_backward_device(ctx.handle, C.byref(s), C.byref(b)))
"""


def test_dense_layers(host_hip):  # noqa: F811
    host_hip(SETUP + f"""
for rows, k, n, type, kernel, _ in {LAYERS}:
    forward(rows, k, n, type)
    found = launches("linear_vector_kernel") if kernel == "vector" else tile(type, "layer", kernel)
    assert found == 1, (rows, k, n, type)
for rows, k, n, type, kernel in {NORMALIZED}:
    forward(rows, k, n, type, normalize=1)
    assert tile(type, "normalized", kernel) == 1, (rows, k, n, type)
""")


def test_gradients(host_hip):  # noqa: F811
    host_hip(SETUP + f"""
for rows, k, n, type, dx, dw, joined in {GRADIENTS}:
    backward(rows, k, n, type)
    if dx is None:
        assert launches("linear_gradients_kernel") == 1 and launches("linear_tile_kernel") == 0, (rows, k, n)
    else:
        assert tile(type, "dx", dx) == 1 and tile(type, "dw", dw) == 1, (rows, k, n)
    assert launches("linear_join_kernel") == int(joined), (rows, k, n)
""")


def test_every_tile_has_a_shape(host_hip):  # noqa: F811
    """The tiles that the rules can choose, all of them in the lists."""
    layer = {(t == "f32", kernel) for _, _, _, t, kernel, _ in LAYERS}
    assert layer >= {(False, "256"), (False, "128"), (False, "64"), (True, "128"), (True, "64"), (False, "vector")}
    dx = {(t == "f32", x) for _, _, _, t, x, _, _ in GRADIENTS}
    dw = {(t == "f32", w) for _, _, _, t, _, w, _ in GRADIENTS}
    assert dx >= {(False, s) for s in ("256", "128", "64", None)} | {(True, s) for s in ("128", "64", None)}
    assert dw >= {(False, s) for s in ("256", "128", "64", None)} | {(True, s) for s in ("128", "64", None)}
    assert {k for *_, k in NORMALIZED} == {"128 x 128", "32 x 128", "32 x 96", "64 x 64"}


def test_workspaces_grow_with_the_rows(host_hip):  # noqa: F811
    """A workspace made for some rows serves fewer, whatever tiles and parts
    those take."""
    host_hip(SETUP + """
rng = np.random.default_rng(3)
for i in range(30_000):
    k, n = (int(2 ** rng.uniform(5, 13)) for _ in range(2))
    type, training = int(rng.integers(3)), int(i % 8 != 0)
    rows = np.exp2(rng.uniform(0, 18)) * np.array([rng.uniform(0.4, 1), 1])  # near each other: parts change between them
    rows = np.maximum(1, rows.astype(np.int64))
    need = [C.c_size_t(), C.c_size_t()]
    for r, v in zip(rows, need):
        s = op.LinearShape(int(r), k, n, type, type, 0, 0)
        capi.check(L.chimera_linear_workspace(C.byref(s), training, C.byref(v)))
    assert need[0].value <= need[1].value, (rows, k, n, type, training)
""")


def test_late_interaction(host_hip):  # noqa: F811
    host_hip(SETUP + f"""
c = op.CacheDesc(0, 128, 128, 16, 50, A, 2 * A)
for _, type, nq, length, cap, items in {WALKS}:
    m = op.CacheMaxsim(queries=A, type=op.TYPES[type], nq=nq, query_len=length, page_start=A, doc_lens=A, pages=A,
                       num_docs=9, num_page_entries=20, max_doc_tokens=100, cand_ids=A, cand_cap=cap, scores=A)
    hip.host_hip_reset_launches()
    capi.check(L.chimera_cache_maxsim_device(ctx.handle, C.byref(c), C.byref(m)))
    assert hip.host_hip_blocks(b"cache_maxsim_kernel") == -(-cap // (4 * items)), (nq, cap)
""")


def test_rows_past_the_caches(host_hip):  # noqa: F811
    host_hip(SETUP + f"""
for type, format, dim, rows in {LARGE}:
    f = op.FORMATS[format]
    c = op.CacheDesc(f, dim, 128, 16, 1 << 20, A, 2 * A)
    for n, once in ((rows, 1), ((128 << 20) // dim // (4 if type == "f32" else 2), 0)):
        hip.host_hip_reset_launches()
        capi.check(L.chimera_cache_write_device(ctx.handle, C.byref(c), C.c_void_p(3 * A), op.TYPES[type], C.c_int64(dim),
                                                C.c_void_p(4 * A), C.c_int64(n)))
        capi.check(L.chimera_cache_read_device(ctx.handle, C.byref(c), C.c_void_p(4 * A), C.c_int64(n), C.c_void_p(3 * A),
                                               op.TYPES[type], C.c_int64(dim)))
        for name in ("write", "read"):
            assert launches(f"cache_{{name}}_kernelI{{NAME[type]}}Li{{f}}ELb{{once}}E") == 1, (name, type, n)
""")
