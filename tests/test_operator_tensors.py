"""PyTorch tensors as the operators' arrays, on the CPU: the library runs on a
model of the HIP runtime, the tensors are stand-ins with torch's methods."""
from host_hip_child import host_hip  # noqa: F401


def test_tensors(host_hip):  # noqa: F811
    host_hip("""
from chimera_amd import operators as op

class Tensor:
    def __init__(self, shape, dtype, stride=None, is_cuda=True):
        self.shape, self.dtype, self.is_cuda = shape, "torch." + dtype, is_cuda
        self.memory = ctx.empty(1 << 20, np.uint8)
        self._stride = stride or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))
    def data_ptr(self):
        return self.memory.ptr
    def stride(self, dim=None):
        return self._stride if dim is None else self._stride[dim]
    def dim(self):
        return len(self.shape)

def refuses(word, *args, **kw):
    try:
        op.from_torch(Tensor(*args, **kw))
    except ValueError as e:
        assert word in str(e), e
        return
    raise AssertionError(word + " not refused")

ctx = context()
assert ctx.stream != 0
t = Tensor((100, 64), "bfloat16", (80, 1))
a = op.from_torch(t)
assert (a.ptr, a.shape, a.dtype, a.stride) == (t.memory.ptr, (100, 64), "bfloat16", 80)
layer = op.Linear(ctx, op.from_torch(Tensor((32, 64), "bfloat16")), op.from_torch(Tensor((32,), "bfloat16")), max_rows=100)
layer.forward(a, op.from_torch(Tensor((100, 32), "float32")))
assert hip.host_hip_launches(b"linear") > 0
for dtype, name in (("float16", "f16"), ("float32", "f32"), ("int32", "int32"), ("int64", "int64"), ("uint8", "uint8")):
    assert op._type_name(op.from_torch(Tensor((5, 4, 3), dtype))) == name
# one row, or a column of one value, has no stride that matters
op.from_torch(Tensor((1, 64), "float32", (7, 1)))
op.from_torch(Tensor((9, 1), "float32", (5, 3)))
refuses("device", (3, 4), "float32", is_cuda=False)
refuses("stride", (3, 4), "float32", (1, 3))        # transposed
refuses("stride", (4,), "int64", (2,))               # every other value
refuses("stride", (4, 6, 8), "float32", (48, 16, 1)) # rows apart in a batch
refuses("stride", (3, 4), "float32", (0, 1))         # one row several times
""")
