"""The launches that the dense stack's operators make, on the CPU: the library
runs on a model of the HIP runtime that refuses a launch which the runtime
refuses."""
from host_hip_child import host_hip  # noqa: F401
from test_dense_stack_dispatch import SETUP


def test_4_bit_rows_of_every_size_that_a_call_may_have(host_hip):  # noqa: F811
    """Up to 2^28 - 16 rows of up to 65,536 values: 2^31 blocks of 256 threads."""
    host_hip(SETUP + """
i64 = C.c_int64
for rows, n, parts in ((1, 1, 1), (1 << 25, 256, 1), ((1 << 25) + 1, 256, 2), ((1 << 28) - 16, 1, 8), ((1 << 27) + 33, 1024, 17),
                       ((1 << 28) - 16, 65536, 2048), (131_072, 65536, 1), (131_073, 65536, 2)):
    hip.host_hip_reset_launches()
    for type in (0, 1, 2):
        capi.check(L.chimera_mx4_quantise_device(ctx.handle, C.c_void_p(A), type, i64(n), i64(rows), n, C.c_void_p(1 << 50), C.c_void_p(1 << 52)))
        capi.check(L.chimera_mx4_read_device(ctx.handle, C.c_void_p(1 << 50), C.c_void_p(1 << 52), i64(rows), n, C.c_void_p(A), type, i64(n)))
    assert launches("mx4_quantise_kernel") == launches("mx4_read_kernel") == 3 * parts, (rows, n, launches("mx4_"))
""")


def test_4_bit_layers_of_every_size_that_a_call_may_have(host_hip):  # noqa: F811
    """Rows up to the limit of a call (2^35 / 2 values of the wider side), at each
    kernel's edge."""
    host_hip(SETUP + """
rng = np.random.default_rng(1)
for _ in range(300):
    k, n = (int(2 ** rng.uniform(0, 16)) for _ in range(2))
    normalize = int(rng.random() < 0.5)
    n = min(n, 128) if normalize else n
    rows = ((1 << 21) // -(-max(k, n) // 128)) * 128
    if k * n > 1 << 30:
        continue
    for type in (0, 1):
        s = op.LinearShape(rows, k, n, type, type, 0, normalize)
        bytes = need(L.chimera_mx4_linear_workspace, C.byref(s))
        a = op.Mx4LinearArgs(A, 1 << 50, 1 << 51, None, None, 1 << 52, k, n, n, 1 << 54 if bytes else None, bytes)
        capi.check(L.chimera_mx4_linear_device(ctx.handle, C.byref(s), C.byref(a)))
""")


def test_every_block_of_a_walk_has_work(host_hip):  # noqa: F811
    """A block for each group of columns and range of rows and none besides, as
    they go round the XCDs: idle ones would leave some of these without work.
    As many ranges as the CUs hold blocks, or as there are tiles of rows."""
    host_hip(SETUP + """
for rows, k, n, waves, units, a_cu in ((65_536, 1024, 4096, 8, 2, 1), (65_536, 1024, 2560, 8, 2, 1), (65_536, 1024, 3584, 8, 2, 1),
                                       (128, 2048, 4096, 4, 1, 2), (288, 1024, 4096, 4, 1, 2), (2048, 1024, 16384, 8, 2, 1),
                                       (1, 1024, 32768, 4, 1, 2), (32, 256, 65536, 4, 1, 2), (10_007, 777, 520, 4, 1, 2),
                                       (8200, 1500, 4096, 8, 1, 1)):
    s = op.LinearShape(rows, k, n, 2, 2, 0, 0)
    bytes = need(L.chimera_mx4_linear_workspace, C.byref(s))
    a = op.Mx4LinearArgs(A, 1 << 50, 1 << 51, None, None, 1 << 52, k, n, n, 1 << 54, bytes)
    capi.check(L.chimera_mx4_linear_device(ctx.handle, C.byref(s), C.byref(a)))
    assert launches(f"Li{waves}ELi{units}E") == launches("mx4_walk_kernel") == 1, (rows, k, n)
    groups, tiles = -(-n // (32 * waves)), -(-rows // (32 * units))
    assert hip.host_hip_blocks(b"mx4_walk_kernel") == groups * min(tiles, max(1, 256 * a_cu // groups)), (rows, k, n)
""")
