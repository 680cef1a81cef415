"""The operators beside the index (include/chimera_operators.h): dense layers
that turn hidden states into token embeddings, the layer norm between them, the
update of their weights, layers served in microscaled 4-bit floating point, a
quantised cache of token embeddings and late interaction on it, and a store of
documents that come and go on top of the cache.

Arrays are device arrays: capi.DeviceArray, a PyTorch tensor through
from_torch(), or any object with `ptr`, `shape`
and `dtype` ("f32", "f16", "bf16", a numpy dtype or its name) and, for a
matrix whose rows lie apart, `stride` in elements. Calls are asynchronous on
the context's stream. An object keeps the arguments of its calls, so threads
that share one take turns; calls can be captured into a graph, which stays good
until the object is closed.
"""
from __future__ import annotations

import ctypes as C
import functools
import math

import numpy as np

from . import capi
from .capi import P, check

TYPES = {"f32": 0, "f16": 1, "bf16": 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
FORMATS = {"int8": 0, "int4": 1, "fp8": 2}
_CAPACITY = 4  # CHIMERA_ERR_CAPACITY
_NAMES = {"f32": "f32", "f16": "f16", "bf16": "bf16", "float32": "f32", "float16": "f16", "bfloat16": "bf16"}


class LinearShape(C.Structure):
    _fields_ = [("rows", C.c_int64), ("in_features", C.c_int32), ("out_features", C.c_int32), ("type", C.c_int32),
                ("out_type", C.c_int32), ("activation", C.c_int32), ("normalize", C.c_int32)]


class LinearForward(C.Structure):
    _fields_ = [("x", P), ("weight", P), ("bias", P), ("residual", P), ("y", P), ("saved", P), ("norms", P),
                ("x_stride", C.c_int64), ("weight_stride", C.c_int64), ("residual_stride", C.c_int64),
                ("y_stride", C.c_int64), ("saved_stride", C.c_int64), ("workspace", P), ("workspace_bytes", C.c_size_t)]


class LinearBackward(C.Structure):
    _fields_ = [("x", P), ("weight", P), ("dy", P), ("saved", P), ("y", P), ("norms", P), ("dx", P), ("dweight", P),
                ("dbias", P), ("dresidual", P), ("x_stride", C.c_int64), ("weight_stride", C.c_int64),
                ("dy_stride", C.c_int64), ("saved_stride", C.c_int64), ("y_stride", C.c_int64),
                ("dx_stride", C.c_int64), ("dweight_stride", C.c_int64), ("dresidual_stride", C.c_int64),
                ("workspace", P), ("workspace_bytes", C.c_size_t)]


class CacheDesc(C.Structure):
    _fields_ = [("format", C.c_int32), ("dim", C.c_int32), ("group", C.c_int32), ("page_tokens", C.c_int32),
                ("num_pages", C.c_int64), ("codes", P), ("scales", P)]


class CacheMaxsim(C.Structure):
    _fields_ = [("queries", P), ("type", C.c_int32), ("nq", C.c_int32), ("query_len", C.c_int32), ("query_lens", P),
                ("page_start", P), ("doc_lens", P), ("pages", P), ("num_docs", C.c_int64),
                ("num_page_entries", C.c_int64), ("max_doc_tokens", C.c_int32), ("cand_ids", P), ("cand_counts", P),
                ("cand_cap", C.c_int32), ("scores", P), ("k", C.c_int32), ("top_ids", P), ("top_scores", P),
                ("top_counts", P), ("workspace", P), ("workspace_bytes", C.c_size_t)]


class NormShape(C.Structure):
    _fields_ = [("rows", C.c_int64), ("features", C.c_int32), ("type", C.c_int32), ("out_type", C.c_int32), ("eps", C.c_float)]


class NormForward(C.Structure):
    _fields_ = [("x", P), ("weight", P), ("bias", P), ("y", P), ("mean", P), ("rstd", P), ("x_stride", C.c_int64),
                ("y_stride", C.c_int64)]


class NormBackward(C.Structure):
    _fields_ = [("x", P), ("weight", P), ("dy", P), ("mean", P), ("rstd", P), ("dx", P), ("dweight", P), ("dbias", P),
                ("x_stride", C.c_int64), ("dy_stride", C.c_int64), ("dx_stride", C.c_int64), ("workspace", P),
                ("workspace_bytes", C.c_size_t)]


class Mx4LinearArgs(C.Structure):
    _fields_ = [("x", P), ("codes", P), ("scales", P), ("bias", P), ("residual", P), ("y", P), ("x_stride", C.c_int64),
                ("residual_stride", C.c_int64), ("y_stride", C.c_int64), ("workspace", P), ("workspace_bytes", C.c_size_t)]


class OrthogonalShape(C.Structure):
    _fields_ = [("rows", C.c_int32), ("cols", C.c_int32), ("type", C.c_int32), ("out_type", C.c_int32), ("steps", C.c_int32),
                ("a", C.c_float), ("b", C.c_float), ("c", C.c_float)]


class OrthogonalArgs(C.Structure):
    _fields_ = [("gradient", P), ("momentum", P), ("new_momentum", P), ("mu", C.c_float), ("nesterov", C.c_int32), ("out", P),
                ("weight", P), ("new_weight", P), ("rounded", P), ("rate", C.c_float), ("decay", C.c_float),
                ("gradient_stride", C.c_int64), ("momentum_stride", C.c_int64), ("new_momentum_stride", C.c_int64),
                ("out_stride", C.c_int64), ("weight_stride", C.c_int64), ("new_weight_stride", C.c_int64),
                ("rounded_stride", C.c_int64), ("workspace", P), ("workspace_bytes", C.c_size_t)]


_NUMPY = {np.dtype(np.float32): "f32", np.dtype(np.float16): "f16", np.dtype(np.int32): "int32",
          np.dtype(np.int64): "int64", np.dtype(np.uint8): "uint8"}


def _type_name(a) -> str:
    d = a.dtype
    if d.__class__ is str:
        return _NAMES.get(d, d)
    if getattr(a, "bf16", False):
        return "bf16"
    d = np.dtype(d)
    return _NUMPY.get(d) or d.name


def _type(a, what: str) -> int:
    t = TYPES.get(_type_name(a))
    if t is None:
        raise ValueError(f"{what} must be f32, f16 or bf16, not {_type_name(a)}")
    return t


def _expect(a, what: str, shape: tuple, type_name: str) -> None:
    if a.shape != shape and tuple(a.shape) != shape:
        raise ValueError(f"{what} must have shape {shape}, not {tuple(a.shape)}")
    if _type_name(a) != type_name:
        raise ValueError(f"{what} must be {type_name}, not {_type_name(a)}")


def _expect_whole(a, what: str, shape: tuple, type_name: str) -> None:
    _expect(a, what, shape, type_name)
    _whole(a, what)


def _whole(a, what: str) -> None:
    """Refuses rows that lie apart where the call takes no stride."""
    s = getattr(a, "stride", None)
    if s is None or len(a.shape) < 2 or s == a.shape[-1]:
        return
    if s != math.prod(a.shape[1:]) and any(n != 1 for n in a.shape[:-1]):  # between first indices, of more than two
        raise ValueError(f"the rows of {what} must follow each other")


@functools.lru_cache(maxsize=None)
def _function(name: str, *argtypes):
    """An entry point with its argument types set: plain integers and struct
    references go through without wrapping."""
    f = capi.lib()[name]
    f.argtypes = argtypes
    f.restype = C.c_int
    return f


def _stride(a) -> int:
    s = getattr(a, "stride", None)
    return a.shape[-1] if s is None else s


def _ptr(a):
    return None if a is None else a.ptr


class TensorArray:
    """A device array that is a PyTorch tensor's memory (from_torch)."""

    def __init__(self, tensor, ptr: int, shape: tuple, dtype: str, stride: int | None):
        self.tensor, self.ptr, self.shape, self.dtype, self.stride = tensor, ptr, shape, dtype, stride


def from_torch(tensor) -> TensorArray:
    """A PyTorch tensor as an array that the operators take: its memory, not
    a copy; rows of a matrix may lie apart. torch has to be imported before
    this package loads its library, so that both share torch's HIP runtime, and
    its work is not ordered against the context's stream: run it there
    (torch.cuda.ExternalStream(ctx.stream)), or synchronize between the two."""
    if not tensor.is_cuda:
        raise ValueError("the tensor is not on the device")
    shape, strides = tuple(tensor.shape), tuple(tensor.stride())
    follow = 1  # elements from one index to the next without gaps
    for i in range(len(shape) - 1, -1, -1):
        rows = len(shape) == 2 and i == 0 and strides[0] >= shape[1]
        if shape[i] > 1 and strides[i] != follow and not rows:
            raise ValueError(f"a tensor with strides {strides} is no matrix of rows; call contiguous()")
        follow *= shape[i]
    apart = strides[0] if len(shape) == 2 and shape[0] > 1 else None
    return TensorArray(tensor, tensor.data_ptr(), shape, str(tensor.dtype).rpartition(".")[2], apart)


class Linear:
    """One dense layer, Y = act(X W^T + b) + R, divided row by row by its
    length with `normalize` (at most 128 outputs). weight [out, in] and bias
    [out] stay the caller's arrays and may change between calls. The object
    holds the workspace for calls of up to max_rows rows, and with `training`
    for the backward pass; close it before its context. Where in_features fill
    whole 16 bytes it allocates the room to lay out x again, without `training`,
    at the first call whose rows do not start at multiples of 16 bytes: make
    one before such a call is captured into a graph."""

    def __init__(self, ctx: capi.Context, weight, bias=None, activation: str = "none", normalize: bool = False,
                 max_rows: int = 1, training: bool = False):
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        if len(weight.shape) != 2:
            raise ValueError("weight must be [out_features, in_features]")
        self.ctx = ctx
        self.weight, self.bias = weight, bias
        self.out_features, self.in_features = weight.shape
        self.type = _type_name(weight)
        t = _type(weight, "weight")
        if bias is not None:
            _expect(bias, "bias", (self.out_features,), self.type)
        self.training = training
        self._shape = LinearShape(0, self.in_features, self.out_features, t, t, ACTIVATIONS[activation], int(normalize))
        self._forward = LinearForward(weight=weight.ptr, bias=_ptr(bias), weight_stride=_stride(weight))
        self._backward = LinearBackward(weight=weight.ptr, weight_stride=_stride(weight))
        self._shape_ref = C.byref(self._shape)
        self._forward_ref, self._backward_ref = C.byref(self._forward), C.byref(self._backward)
        self._call_forward = _function("chimera_linear_forward_device", P, P, P)
        self._call_backward = _function("chimera_linear_backward_device", P, P, P)
        self._workspaces = []  # the last one is in use, and holds `capacity` bytes when a call needed them
        self.max_rows = max_rows
        self._capacity = self._need(max_rows, training)
        # rows that do not end at a multiple of 16 bytes are always laid out again
        whole = self.in_features * (4 if self.type == "f32" else 2) % 16 == 0
        self._allocate(self._need(0, False) if whole and not training else self._capacity)

    def _need(self, rows: int, training: bool) -> int:
        need = C.c_size_t()
        self._shape.rows = rows
        check(capi.lib().chimera_linear_workspace(self._shape_ref, int(training), C.byref(need)))
        return need.value

    @property
    def _workspace(self):
        return self._workspaces[-1] if self._workspaces else None

    def _allocate(self, nbytes: int) -> None:
        self._workspaces.append(self.ctx.empty(nbytes, np.uint8))
        for args in (self._forward, self._backward):
            args.workspace, args.workspace_bytes = self._workspace.ptr, nbytes

    def _run(self, call, args) -> None:
        code = call(self.ctx.handle, self._shape_ref, args)
        if code == _CAPACITY and self._workspaces and self._workspace.nbytes < self._capacity:
            self._allocate(self._capacity)
            code = call(self.ctx.handle, self._shape_ref, args)
        check(code)

    def close(self) -> None:
        """Frees the workspace; calls after it are refused."""
        workspaces = getattr(self, "_workspaces", None)
        if workspaces:
            for args in (self._forward, self._backward):
                args.workspace, args.workspace_bytes = None, 0
            self.ctx.synchronize()
            while workspaces:
                workspaces.pop().free()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _rows(self, x, y, what: str, training: bool) -> int:
        rows = x.shape[0]
        if rows > self.max_rows:
            need = self._need(rows, training)
            if need > self._capacity:
                raise capi.ChimeraError(_CAPACITY, f"the workspace is for {self.max_rows} rows, the call has {rows}")
        if tuple(y.shape) != (rows, self.out_features):
            raise ValueError(f"{what} must have shape {(rows, self.out_features)}, not {tuple(y.shape)}")
        self._shape.rows, self._shape.out_type = rows, _type(y, what)
        return rows

    def forward(self, x, y, residual=None, saved=None, norms=None) -> None:
        """y [rows, out] (the layer's type or f32) from x [rows, in]. For the
        backward pass, `saved` [rows, out] gets the sums before the activation
        and `norms` [rows] f32 the lengths."""
        rows = self._rows(x, y, "y", False)
        _expect(x, "x", (rows, self.in_features), self.type)
        a = self._forward
        a.x, a.x_stride, a.y, a.y_stride = x.ptr, _stride(x), y.ptr, _stride(y)
        a.residual = a.saved = a.norms = None
        if residual is not None:
            _expect(residual, "residual", (rows, self.out_features), self.type)
            a.residual, a.residual_stride = residual.ptr, _stride(residual)
        if saved is not None:
            _expect(saved, "saved", (rows, self.out_features), self.type)
            a.saved, a.saved_stride = saved.ptr, _stride(saved)
        if norms is not None:
            _expect(norms, "norms", (rows,), "f32")
            a.norms = norms.ptr
        self._run(self._call_forward, self._forward_ref)

    def backward(self, x, dy, saved=None, y=None, norms=None, dx=None, dweight=None, dbias=None,
                 dresidual=None) -> None:
        """Gradients from dy [rows, out]; those left out are not computed.
        `saved` is read with an activation, `y` and `norms` with normalize, as
        forward() left them."""
        if not self.training:
            raise ValueError("the layer was made without training")
        rows = self._rows(x, dy, "dy", True)
        n, k, t = self.out_features, self.in_features, self.type
        _expect(x, "x", (rows, k), t)
        a = self._backward
        a.x, a.x_stride, a.dy, a.dy_stride = x.ptr, _stride(x), dy.ptr, _stride(dy)
        for name, v, shape, kind in (("saved", saved, (rows, n), t), ("y", y, (rows, n), _type_name(dy)),
                                     ("norms", norms, (rows,), "f32"), ("dx", dx, (rows, k), t),
                                     ("dweight", dweight, (n, k), t), ("dbias", dbias, (n,), t),
                                     ("dresidual", dresidual, (rows, n), t)):
            if v is not None:
                _expect(v, name, shape, kind)
                if len(shape) == 2:
                    setattr(a, name + "_stride", _stride(v))
            setattr(a, name, _ptr(v))
        self._run(self._call_backward, self._backward_ref)


def _int32(value: int, what: str) -> int:
    """The value, which ctypes would cut to 32 bits without a word."""
    if not -(1 << 31) <= value < 1 << 31:
        raise ValueError(f"{what} must fit 32 bits, not {value}")
    return value


class _Workspace:
    """What an object's calls need of memory, for calls of up to a number of
    rows: freed by close(), after which calls that need it are refused."""

    def __init__(self, ctx: capi.Context):
        self.ctx = ctx
        self._workspace = None

    def _allocate(self, nbytes: int, *args) -> None:
        self._holders = args
        self._bytes = nbytes
        if nbytes:
            self._workspace = self.ctx.empty(nbytes, np.uint8)
        for a in args:
            a.workspace, a.workspace_bytes = _ptr(self._workspace), nbytes

    def close(self) -> None:
        """Frees the workspace; calls after it that need it are refused."""
        workspace, self._workspace = getattr(self, "_workspace", None), None
        if workspace is not None:
            for a in self._holders:
                a.workspace, a.workspace_bytes = None, 0
            self.ctx.synchronize()
            workspace.free()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _room(self, rows: int, need) -> None:
        if rows > self.max_rows and need(rows) > self._bytes:
            raise capi.ChimeraError(_CAPACITY, f"the workspace is for {self.max_rows} rows, the call has {rows}")


class LayerNorm(_Workspace):
    """y = (x - mean) / sqrt(var + eps) * weight + bias, row by row. weight and
    bias [features] stay the caller's arrays and may change between calls; a
    bias of None is zeros. For ones, leave the weight out and give `features`
    and `type`. With `training` the object holds the workspace for backward
    passes of up to max_rows rows; close it before its context."""

    def __init__(self, ctx: capi.Context, weight=None, bias=None, eps: float = 1e-5, max_rows: int = 1,
                 training: bool = False, features: int | None = None, type: str | None = None):
        super().__init__(ctx)
        if weight is None and bias is None and (features is None or type is None):
            raise ValueError("a layer norm without weight and bias needs features and type")
        given = weight if weight is not None else bias
        if given is not None:
            if len(given.shape) != 1:
                raise ValueError("weight and bias must be [features]")
            features, type = given.shape[0], _type_name(given)
        if type not in TYPES:
            raise ValueError(f"the type must be f32, f16 or bf16, not {type}")
        for v, what in ((weight, "weight"), (bias, "bias")):
            if v is not None:
                _expect(v, what, (features,), type)
        self.weight, self.bias, self.features, self.type = weight, bias, features, type
        self.training, self.max_rows = training, max_rows
        self._shape = NormShape(0, _int32(features, "features"), TYPES[type], TYPES[type], eps)
        self._forward = NormForward(weight=_ptr(weight), bias=_ptr(bias))
        self._backward = NormBackward(weight=_ptr(weight))
        self._shape_ref = C.byref(self._shape)
        self._forward_ref, self._backward_ref = C.byref(self._forward), C.byref(self._backward)
        self._call_forward = _function("chimera_norm_forward_device", P, P, P)
        self._call_backward = _function("chimera_norm_backward_device", P, P, P)
        need = self._need(max_rows)
        self._allocate(need if training else 0, self._backward)

    def _need(self, rows: int) -> int:
        need = C.c_size_t()
        self._shape.rows, self._shape.out_type = rows, self._shape.type  # a refused call may have left another
        check(capi.lib().chimera_norm_workspace(self._shape_ref, C.byref(need)))
        return need.value

    def forward(self, x, y, mean=None, rstd=None) -> None:
        """y [rows, features] (the norm's type or f32) from x [rows, features].
        For the backward pass `mean` and `rstd` [rows] f32 get the rows'
        statistics."""
        rows = x.shape[0]
        _expect(x, "x", (rows, self.features), self.type)
        if tuple(y.shape) != (rows, self.features):
            raise ValueError(f"y must have shape {(rows, self.features)}, not {tuple(y.shape)}")
        self._shape.rows, self._shape.out_type = rows, _type(y, "y")
        a = self._forward
        a.x, a.x_stride, a.y, a.y_stride = x.ptr, _stride(x), y.ptr, _stride(y)
        for name, v in (("mean", mean), ("rstd", rstd)):
            if v is not None:
                _expect(v, name, (rows,), "f32")
            setattr(a, name, _ptr(v))
        check(self._call_forward(self.ctx.handle, self._shape_ref, self._forward_ref))

    def backward(self, x, dy, mean, rstd, dx=None, dweight=None, dbias=None) -> None:
        """Gradients from dy [rows, features] and what forward() left in `mean`
        and `rstd`; those left out are not computed. The weight's is that of the
        factor, also where it is ones."""
        if not self.training:
            raise ValueError("the layer norm was made without training")
        rows, n, t = x.shape[0], self.features, self.type
        _expect(x, "x", (rows, n), t)
        if tuple(dy.shape) != (rows, n):
            raise ValueError(f"dy must have shape {(rows, n)}, not {tuple(dy.shape)}")
        _expect(mean, "mean", (rows,), "f32")
        _expect(rstd, "rstd", (rows,), "f32")
        self._room(rows, self._need)
        self._shape.rows, self._shape.out_type = rows, _type(dy, "dy")
        a = self._backward
        a.x, a.x_stride, a.dy, a.dy_stride, a.mean, a.rstd = x.ptr, _stride(x), dy.ptr, _stride(dy), mean.ptr, rstd.ptr
        if dx is not None:
            _expect(dx, "dx", (rows, n), t)
            a.dx_stride = _stride(dx)
        a.dx = _ptr(dx)
        for name, v in (("dweight", dweight), ("dbias", dbias)):
            if v is not None:
                _expect(v, name, (n,), t)
            setattr(a, name, _ptr(v))
        check(self._call_backward(self.ctx.handle, self._shape_ref, self._backward_ref))


def mx4_row(features: int) -> tuple[int, int]:
    """(bytes of codes, bytes of scales) of a row of 4-bit values."""
    row, scales = C.c_int32(), C.c_int32()
    check(capi.lib().chimera_mx4_row(_int32(features, "features"), C.byref(row), C.byref(scales)))
    return row.value, scales.value


def _expect_mx4(codes, scales, rows: int, features: int) -> None:
    row, blocks = mx4_row(features)
    _expect_whole(codes, "codes", (rows, row), "uint8")
    _expect_whole(scales, "scales", (rows, blocks), "uint8")


def mx4_quantise(ctx: capi.Context, rows, codes, scales) -> None:
    """Rows [n, features] as codes of 4 bits [n, row bytes] uint8 and a power of
    two for each 32 values, scales [n, row scales] uint8 (mx4_row)."""
    n, features = rows.shape
    _expect_mx4(codes, scales, n, features)
    call = _function("chimera_mx4_quantise_device", P, P, C.c_int32, C.c_int64, C.c_int64, C.c_int32, P, P)
    check(call(ctx.handle, rows.ptr, _type(rows, "rows"), _stride(rows), n, features, codes.ptr, scales.ptr))


def mx4_read(ctx: capi.Context, codes, scales, out) -> None:
    """out [n, features] = the values of rows that mx4_quantise wrote."""
    n, features = out.shape
    _expect_mx4(codes, scales, n, features)
    call = _function("chimera_mx4_read_device", P, P, P, C.c_int64, C.c_int32, P, C.c_int32, C.c_int64)
    check(call(ctx.handle, codes.ptr, scales.ptr, n, features, out.ptr, _type(out, "out"), _stride(out)))


class Mx4Linear(_Workspace):
    """A dense layer on a weight in microscaled 4-bit floating point, codes
    [out, row bytes] and scales [out, row scales] as mx4_quantise writes them of
    a weight [out, in_features]. x is quantised the same way within the call;
    what follows the product is as in Linear. `type` is that of x, the bias and
    the residual. The object holds the workspace for calls of up to max_rows
    rows; close it before its context."""

    def __init__(self, ctx: capi.Context, codes, scales, in_features: int, bias=None, type: str = "bf16",
                 activation: str = "none", normalize: bool = False, max_rows: int = 1):
        super().__init__(ctx)
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        if type not in TYPES:
            raise ValueError(f"the type must be f32, f16 or bf16, not {type}")
        n = codes.shape[0]
        _expect_mx4(codes, scales, n, in_features)
        if bias is not None:
            _expect(bias, "bias", (n,), type)
        self.codes, self.scales, self.bias = codes, scales, bias
        self.in_features, self.out_features, self.type, self.max_rows = in_features, n, type, max_rows
        t = TYPES[type]
        self._shape = LinearShape(0, in_features, n, t, t, ACTIVATIONS[activation], int(normalize))
        self._args = Mx4LinearArgs(codes=codes.ptr, scales=scales.ptr, bias=_ptr(bias))
        self._shape_ref, self._args_ref = C.byref(self._shape), C.byref(self._args)
        self._call = _function("chimera_mx4_linear_device", P, P, P)
        self._allocate(self._need(max_rows), self._args)

    def _need(self, rows: int) -> int:
        need = C.c_size_t()
        self._shape.rows, self._shape.out_type = rows, self._shape.type  # a refused call may have left another
        check(capi.lib().chimera_mx4_linear_workspace(self._shape_ref, C.byref(need)))
        return need.value

    def forward(self, x, y, residual=None) -> None:
        """y [rows, out] (the layer's type or f32) from x [rows, in]."""
        rows = x.shape[0]
        _expect(x, "x", (rows, self.in_features), self.type)
        if tuple(y.shape) != (rows, self.out_features):
            raise ValueError(f"y must have shape {(rows, self.out_features)}, not {tuple(y.shape)}")
        self._room(rows, self._need)
        self._shape.rows, self._shape.out_type = rows, _type(y, "y")
        a = self._args
        a.x, a.x_stride, a.y, a.y_stride = x.ptr, _stride(x), y.ptr, _stride(y)
        if residual is not None:
            _expect(residual, "residual", (rows, self.out_features), self.type)
            a.residual_stride = _stride(residual)
        a.residual = _ptr(residual)
        check(self._call(self.ctx.handle, self._shape_ref, self._args_ref))


class OrthogonalUpdate(_Workspace):
    """The update of a weight [rows, cols]: its gradient (of `type`), with
    momentum or without, is divided by its size and made near orthogonal by
    `steps` steps X <- a X + (b A + c A^2) X with A = X X^T. The object holds
    the workspace; close it before its context."""

    def __init__(self, ctx: capi.Context, rows: int, cols: int, type: str = "f32", steps: int = 5,
                 coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315)):
        super().__init__(ctx)
        if type not in TYPES:
            raise ValueError(f"the type must be f32, f16 or bf16, not {type}")
        a, b, c = coefficients
        self.rows, self.cols, self.type = _int32(rows, "rows"), _int32(cols, "cols"), type
        self._shape = OrthogonalShape(rows, cols, TYPES[type], TYPES[type], _int32(steps, "steps"), a, b, c)
        self._args = OrthogonalArgs()
        self._shape_ref, self._args_ref = C.byref(self._shape), C.byref(self._args)
        self._call = _function("chimera_orthogonal_update_device", P, P, P)
        need = C.c_size_t()
        check(capi.lib().chimera_orthogonal_workspace(self._shape_ref, C.byref(need)))
        self._allocate(need.value, self._args)

    def _set(self, name: str, v, kind: str) -> None:
        if v is not None:
            _expect(v, name, (self.rows, self.cols), kind)
            setattr(self._args, name + "_stride", _stride(v))
        setattr(self._args, name, _ptr(v))

    def _run(self, gradient, out, momentum, new_momentum, mu, nesterov) -> None:
        a = self._args
        self._set("gradient", gradient, self.type)
        self._set("momentum", momentum, "f32")
        self._set("new_momentum", new_momentum if new_momentum is not None else momentum, "f32")
        if momentum is None and new_momentum is not None:
            raise ValueError("new_momentum needs momentum")
        a.mu, a.nesterov = mu, int(nesterov)
        self._shape.out_type = self._shape.type
        if out is not None:
            _expect(out, "out", (self.rows, self.cols), _type_name(out))
            self._shape.out_type, a.out_stride = _type(out, "out"), _stride(out)
        a.out = _ptr(out)
        check(self._call(self.ctx.handle, self._shape_ref, self._args_ref))

    def orthogonalize(self, gradient, out, momentum=None, new_momentum=None, mu: float = 0.95, nesterov: bool = True) -> None:
        """out [rows, cols] (the gradient's type or f32) = the orthogonal
        update alone."""
        for name in ("weight", "new_weight", "rounded"):
            self._set(name, None, "f32")
        self._args.rate = self._args.decay = 0.0
        self._run(gradient, out, momentum, new_momentum, mu, nesterov)

    def step(self, gradient, weight, new_weight=None, rate: float = 0.02, decay: float = 0.0, momentum=None,
             new_momentum=None, mu: float = 0.95, nesterov: bool = True, rounded=None, out=None) -> None:
        """new_weight = (1 - decay) weight - rate * update, and the momentum
        mu * momentum + gradient; weights and momentum are f32 and change in
        their place where no new array is given. `rounded` gets the weight in
        the gradient's type, as a 16-bit layer reads it."""
        self._set("weight", weight, "f32")
        self._set("new_weight", new_weight if new_weight is not None else weight, "f32")
        self._set("rounded", rounded, self.type)
        self._args.rate, self._args.decay = rate, decay
        self._run(gradient, out, momentum, new_momentum, mu, nesterov)


def cache_row(format: str, dim: int, group: int, page_tokens: int = 1) -> tuple[int, int]:
    """(bytes of codes, number of scales) of one slot of a cache."""
    if format not in FORMATS:
        raise ValueError(f"unknown cache format {format!r}")
    row, scales = C.c_int32(), C.c_int32()
    desc = CacheDesc(FORMATS[format], _int32(dim, "dim"), _int32(group, "group"), _int32(page_tokens, "page_tokens"), 0,
                     None, None)
    check(capi.lib().chimera_cache_row(C.byref(desc), C.byref(row), C.byref(scales)))
    return row.value, scales.value


class TokenCache:
    """Quantised token embeddings in pages of page_tokens slots: codes [slots,
    row bytes] uint8 and scales [slots, scales] f32, the caller's arrays. A
    call's workspace is kept for the next one; where one needs a larger one, it
    allocates (so it cannot be captured: make a call of that size first), and
    the smaller ones stay until close() for the graphs that hold their
    addresses. Each is at least twice the one before it, the last below 32 MiB.
    Close the cache before its context."""

    def __init__(self, ctx: capi.Context, codes, scales, format: str = "int8", dim: int = 128, group: int = 128,
                 page_tokens: int = 16):
        row, groups = cache_row(format, dim, group)
        slots = codes.shape[0]
        if tuple(codes.shape) != (slots, row) or tuple(scales.shape) != (slots, groups):
            raise ValueError(f"the cache needs codes [slots, {row}] and scales [slots, {groups}]")
        if _type_name(codes) != "uint8" or _type_name(scales) != "f32":
            raise ValueError("codes must be uint8 and scales f32")
        _whole(codes, "codes")
        _whole(scales, "scales")
        if page_tokens < 1 or slots % page_tokens:
            raise ValueError("the slots must fill whole pages")
        cache_row(format, dim, group, page_tokens)
        self.ctx, self.codes, self.scales = ctx, codes, scales
        self.format, self.dim, self.group, self.page_tokens = format, dim, group, page_tokens
        self.slots = slots
        self._desc = CacheDesc(FORMATS[format], dim, group, page_tokens, slots // page_tokens, codes.ptr, scales.ptr)
        self._desc_ref = C.byref(self._desc)
        self._call_write = _function("chimera_cache_write_device", P, P, P, C.c_int32, C.c_int64, P, C.c_int64)
        self._call_read = _function("chimera_cache_read_device", P, P, P, C.c_int64, P, C.c_int32, C.c_int64)
        self._call_maxsim = _function("chimera_cache_maxsim_device", P, P, P)
        self._workspaces = []  # the last one is in use
        self._closed = False
        self._sizes = None  # of the call that the workspace was last found large enough for
        self._args = CacheMaxsim()
        self._args_ref = C.byref(self._args)

    def close(self) -> None:
        """Frees the workspaces; calls after it that need one are refused."""
        self._closed = True
        workspaces = getattr(self, "_workspaces", None)
        if workspaces:
            self._args.workspace, self._args.workspace_bytes = None, 0
            self.ctx.synchronize()
            while workspaces:
                workspaces.pop().free()

    @property
    def _workspace(self):
        return self._workspaces[-1] if self._workspaces else None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def write(self, rows, slots) -> None:
        """Quantises rows [n, dim] into slots [n] (int64; entries outside the
        cache are skipped, the others must differ)."""
        n = rows.shape[0]
        if tuple(rows.shape) != (n, self.dim):
            raise ValueError(f"rows must be [n, {self.dim}]")
        _expect(slots, "slots", (n,), "int64")
        check(self._call_write(self.ctx.handle, self._desc_ref, rows.ptr, _type(rows, "rows"), _stride(rows), slots.ptr, n))

    def read(self, slots, out) -> None:
        """out [n, dim] = the values in slots [n], zeros for a slot outside
        the cache."""
        n = out.shape[0]
        if tuple(out.shape) != (n, self.dim):
            raise ValueError(f"out must be [n, {self.dim}]")
        _expect(slots, "slots", (n,), "int64")
        check(self._call_read(self.ctx.handle, self._desc_ref, slots.ptr, n, out.ptr, _type(out, "out"), _stride(out)))

    def maxsim(self, queries, page_start, doc_lens, pages, max_doc_tokens: int, cand_ids, scores, query_lens=None,
               cand_counts=None, k: int = 0, top_ids=None, top_scores=None, top_counts=None) -> None:
        """scores [nq, cap] f32 of the documents cand_ids [nq, cap] int32 for
        queries [nq, query_len, dim]; token t of document d is in slot t %
        page_tokens of page pages[page_start[d] + t / page_tokens] (int32,
        int64), t < doc_lens[d] (int32). With k the best k of each query
        too."""
        nq, query_len, dim = queries.shape
        if dim != self.dim:
            raise ValueError(f"queries must have {self.dim} dimensions")
        docs, cap = doc_lens.shape[0], cand_ids.shape[1]
        a = self._args
        t = _type(queries, "queries")
        _whole(queries, "queries")
        _expect(page_start, "page_start", (docs,), "int64")
        _expect(doc_lens, "doc_lens", (docs,), "int32")
        _expect(pages, "pages", (pages.shape[0],), "int32")
        _expect_whole(cand_ids, "cand_ids", (nq, cap), "int32")
        _expect_whole(scores, "scores", (nq, cap), "f32")
        a.page_start, a.doc_lens, a.pages = page_start.ptr, doc_lens.ptr, pages.ptr
        a.cand_ids, a.scores = cand_ids.ptr, scores.ptr
        a.query_lens = a.cand_counts = a.top_ids = a.top_scores = a.top_counts = None
        if query_lens is not None:
            _expect(query_lens, "query_lens", (nq,), "int32")
            a.query_lens = query_lens.ptr
        if cand_counts is not None:
            _expect(cand_counts, "cand_counts", (nq,), "int32")
            a.cand_counts = cand_counts.ptr
        if k:
            for name, v, shape, kind in (("top_ids", top_ids, (nq, k), "int64"),
                                         ("top_scores", top_scores, (nq, k), "f32"),
                                         ("top_counts", top_counts, (nq,), "int32")):
                if v is not None:
                    _expect_whole(v, name, shape, kind)
                    setattr(a, name, v.ptr)
        a.queries, a.type, a.nq, a.query_len = queries.ptr, t, nq, query_len
        a.num_docs, a.num_page_entries = docs, pages.shape[0]
        a.max_doc_tokens, a.cand_cap, a.k = _int32(max_doc_tokens, "max_doc_tokens"), cap, _int32(k, "k")
        sizes = (nq, query_len, cap, max_doc_tokens)
        if sizes != self._sizes and not self._closed:
            need = C.c_size_t()
            check(capi.lib().chimera_cache_maxsim_workspace(C.byref(a), C.byref(need)))
            have = 0 if self._workspace is None else self._workspace.nbytes
            if need.value > have:
                larger = self.ctx.empty(max(need.value, 2 * have), np.uint8)
                self._workspaces.append(larger)
                a.workspace, a.workspace_bytes = larger.ptr, larger.nbytes
            self._sizes = sizes
        check(self._call_maxsim(self.ctx.handle, self._desc_ref, self._args_ref))
