"""Shapes that reach each kernel of the operators, with the kernel that they
are meant for: run on the GPU, and checked on the CPU to take that kernel, so
that a new rule cannot leave one without a test. Sizes fill no tile."""

# rows, k, n, type, layer's kernel, rows apart and shifted
LAYERS = [
    (2999, 392, 4936, "bf16", "256", False),  # seven steps of the sum, the last of 8 values
    (3001, 328, 5000, "f16", "256", True),
    (3990, 593, 3401, "bf16", "256", False),  # X and W laid out again
    (3100, 456, 1720, "bf16", "128", True),
    (1737, 156, 3806, "f32", "128", False),  # five steps, the last of 28 values
    (1741, 129, 3807, "f32", "128", True),
    (1300, 200, 1000, "f16", "64", False),
    (700, 260, 650, "f32", "64", True),
    (3, 1000, 333, "bf16", "vector", True),
]

# rows, k, n, type, kernels of dX and dW (None: both in one launch), parts of dW's sum joined
GRADIENTS = [
    (5465, 2280, 632, "bf16", "256", "128", True),
    (7673, 1640, 104, "f16", "256", "64", True),
    (1100, 6008, 5016, "bf16", "128", "256", False),
    (4003, 2144, 1921, "f16", "128", "128", False),
    (2669, 1456, 201, "f32", "128", "64", True),
    (492, 1888, 1865, "f32", "64", "128", False),
    (552, 1968, 2617, "bf16", "64", "128", False),
    (1300, 328, 1000, "bf16", None, None, True),
    (400, 260, 333, "f32", None, None, False),
    (3000, 260, 133, "f32", None, None, True),
]

# rows, k, n, type, layer's kernel: rows of length one
NORMALIZED = [
    (24_601, 72, 128, "bf16", "128 x 128"),
    (24_670, 130, 101, "f16", "128 x 128"),
    (600, 200, 97, "bf16", "32 x 128"),
    (24_650, 40, 128, "f32", "32 x 128"),
    (70, 100, 65, "f16", "32 x 96"),
    (130, 36, 64, "bf16", "64 x 64"),
]

# format, type, queries, query length, candidates of each, documents that a wave takes
WALKS = [
    ("int8", "f32", 37, 32, 443, 2),
    ("int4", "bf16", 29, 45, 1021, 3),
    ("fp8", "f16", 64, 7, 2053, 16),
    ("int8", "f32", 24, 33, 8191, 16),  # and the largest top-k
]

# type, format, dim, rows: past the caches
LARGE = [("f32", "int8", 128, 262_145), ("bf16", "int4", 100, 700_001), ("f16", "fp8", 96, 720_000)]
