"""The linear layer over the update step's quantised weights, on
libodyssey_mp.so (extensions; the reference's linear layer works on float
tensors).

    y  = fp4_linear(x, w)             y  = x W^T    W in 4 bits, in the step's bytes
    dx = fp4_linear_dgrad(dy, w)      dx = dy W
    a  = save_activation8(x)          x kept in 8 bits for the backward pass
    x' = load_activation8(a)
    dW = linear_wgrad8(dy, a)         dW = dy^T x'

Weights are QuantizedTensors of the 4-bit kinds (to_mxfp4, to_nvfp4,
to_nvfp4_tensor_scaled, to_mxfp4_ocp, or the copy that
MixedPrecisionStep.get_quant makes of the step's), read in place. Activations
and gradients are float32, float16 or bfloat16 arrays whose last axis is the
feature axis; leading axes are tokens. CUDA tensors run on torch's current
stream of their device without waiting, host arrays (numpy, or torch on the
CPU; bfloat16 numpy data as uint16 with dtype='bfloat16') are staged and the
call returns when done. A result may not share memory with an operand
(linear_wgrad8's add=out apart); such a call is refused. The gradients are
calls of their own: no autograd graph is recorded, and a product of a tensor
that requires one is refused while gradients are on.
"""
import ctypes as C
from dataclasses import dataclass
from functools import lru_cache
from math import prod

import numpy as np

from . import _lib as L
from .quant import QuantizedTensor

FORMATS8 = {"e4m3": L.A8_E4M3, "e5m2": L.A8_E5M2}
_NAMES = ("float32", "float16", "bfloat16")
_CODES = {"float32": L.F32, "float16": L.F16, "bfloat16": L.BF16, L.F32: L.F32, L.F16: L.F16, L.BF16: L.BF16}
_BLOCK = {L.Q_MXFP4: (32, 17), L.Q_NVFP4: (16, 9), L.Q_NVFP4_TENSOR: (16, 9), L.Q_MXFP4_OCP: (32, 17)}
_TORCH = {}  # torch dtype -> code and back, once torch is there


def _torch_dtypes():
    t = L._torch()
    if not _TORCH and t is not None:
        _TORCH.update({t.float32: L.F32, t.float16: L.F16, t.bfloat16: L.BF16,
                       L.F32: t.float32, L.F16: t.float16, L.BF16: t.bfloat16})
    return _TORCH


def _code(dtype):
    """F32/F16/BF16 code of a dtype given by name, code or torch dtype."""
    c = _CODES.get(dtype) if isinstance(dtype, (str, int)) else _torch_dtypes().get(dtype)
    if c is None:
        raise L.OdysseyError(f"unsupported dtype {dtype}", L.ERR_DTYPE)
    return c


def _count_bytes(b, what):
    """The bytes of a buffer of bytes."""
    if L.is_torch(b):
        n, size = b.numel(), b.element_size()
    else:
        b = np.asarray(b)
        n, size = b.size, b.itemsize
    if size != 1:
        raise L.OdysseyError(f"{what} must be uint8", L.ERR_DTYPE)
    return n


def _no_graph(name, tensor):
    """Refuses a tensor whose gradient would be lost: nothing here records one."""
    if getattr(tensor, "requires_grad", False) and L._torch().is_grad_enabled():
        raise L.OdysseyError(f"{name} records no gradient: detach its tensors or call it under torch.no_grad() "
                             "(the layer's gradients are fp4_linear_dgrad and linear_wgrad8)", L.ERR_ARG)


@dataclass
class Activation8:
    """An activation in 8 bits: codes [rows, 32 * groups] and one scale byte
    per row and 32 columns, uint8; `shape` and `dtype` are the saved tensor's
    (None: [rows, cols] and bfloat16)."""
    codes: object
    scales: object
    rows: int
    cols: int
    format: str = "e4m3"
    shape: tuple = None
    dtype: object = None

    def check(self):
        g = (self.cols + 31) // 32
        if self.format not in FORMATS8:
            raise L.OdysseyError(f"unknown 8-bit activation format {self.format!r}", L.ERR_ARG)
        if self.rows <= 0 or self.cols <= 0:
            raise L.OdysseyError("cannot save an empty activation", L.ERR_SHAPE)
        for b, n in ((self.codes, self.rows * g * 32), (self.scales, self.rows * g)):
            if _count_bytes(b, "codes and scales") != n:
                raise L.OdysseyError("codes and scales do not have the bytes of the activation's rows and columns",
                                     L.ERR_SHAPE)


class _Rows:
    """An array as rows of its last axis: the code of its type and its pitch."""
    __slots__ = ("a", "code", "rows", "cols", "ld", "cuda", "ptr", "lead", "grad")

    def __init__(self, x, dtype, what):
        if L.is_torch(x):
            code = _torch_dtypes().get(x.dtype)
            if code is None:
                raise L.OdysseyError(f"unsupported dtype {x.dtype}", L.ERR_DTYPE)
            shape = x.shape
            if len(shape) == 0 or x.numel() == 0:
                raise L.OdysseyError(f"{what} is empty", L.ERR_SHAPE)
            self.cuda, self.grad = x.is_cuda, x.requires_grad
            if len(shape) != 2:
                x = x.reshape(-1, shape[-1])
            rows, cols = x.shape
            ld, step = x.stride()
            # rows of any pitch are read in place; anything else is copied
            if (step != 1 and cols > 1) or (rows > 1 and ld < cols) or not self.cuda:
                x = x.contiguous()
                ld = cols
            self.ld = ld if rows > 1 else cols
            self.ptr = x.data_ptr()
        else:
            code = L.dtype_code(x, dtype)
            shape = np.shape(x)
            x = np.ascontiguousarray(x)
            if len(shape) == 0 or x.size == 0:
                raise L.OdysseyError(f"{what} is empty", L.ERR_SHAPE)
            self.cuda = self.grad = False
            x = x.reshape(-1, shape[-1])
            rows, cols = x.shape
            self.ld = cols
            self.ptr = x.ctypes.data
        self.a, self.code, self.lead, self.rows, self.cols = x, code, shape[:-1], rows, cols


class _Place:
    """Where a buffer lies (what _same_place and _out ask of _Rows)."""

    def __init__(self, a):
        self.a, self.cuda, self.code = a, L.is_torch(a) and a.is_cuda, None


def _same_place(x, *others):
    """Buffers of one call live on one device (or all on the host)."""
    for o in others:
        t = getattr(o, "is_cuda", False)
        if t != x.cuda or (t and o.get_device() != x.a.get_device()):
            raise L.OdysseyError("the buffers of a call must be on one device", L.ERR_ARG)


def _out(x, out, shape, code, what):
    """The result buffer: new, or the caller's after its checks."""
    if out is None:
        if L.is_torch(x.a):
            return x.a.new_empty(shape) if code == x.code else x.a.new_empty(shape, dtype=_torch_dtypes()[code])
        return np.empty(shape, (np.float32, np.float16, np.uint16)[code])
    _same_place(x, out)
    have = _torch_dtypes().get(out.dtype) if L.is_torch(out) else \
        {np.dtype(np.float32): L.F32, np.dtype(np.float16): L.F16, np.dtype(np.uint16): L.BF16}.get(out.dtype)
    if have != code:
        raise L.OdysseyError(f"{what} must be {_NAMES[code]}", L.ERR_DTYPE)
    if tuple(out.shape) != tuple(shape):
        raise L.OdysseyError(f"{what} has shape {tuple(out.shape)}, expected {tuple(shape)}", L.ERR_SHAPE)
    L.ptr(out)  # contiguous
    return out


def _flat(a):
    return a if a.is_contiguous() else a.contiguous()


def _enqueue(index, fn, *args):
    """fn(*args, stream) with that CUDA device current and torch's stream on
    it; raises on a non-zero status."""
    t = L._torch_module
    if index != t.cuda.current_device():
        with t.cuda.device(index):
            rc = fn(*args, t.cuda.current_stream(index).cuda_stream)
    else:
        raw = getattr(t._C, "_cuda_getCurrentRawStream", None)  # the handle without a Stream object around it
        rc = fn(*args, raw(index) if raw is not None else t.cuda.current_stream(index).cuda_stream)
    if rc:
        L.check(rc)


@lru_cache(maxsize=4096)
def _workspace_bytes(device_index, op, kind, rows, out, inn, code):
    return int(L.lib().ody_linear_workspace_of(op, kind, rows, out, inn, code))


def _workspace(a, n):
    """(tensor or None, its address, n) for one call on a's device."""
    if n <= 0:
        return None, None, 0
    ws = a.new_empty(n, dtype=L._torch().uint8)
    return ws, ws.data_ptr(), n


@lru_cache(maxsize=4096)
def _weight(name, op, kind, numel, features):
    """(the operand's other features, out features, in features, the weight's
    bytes) of a weight of so many elements that meets so many features."""
    other = numel // features
    if numel <= 0 or other * features != numel:
        raise L.OdysseyError(f"{name}: a weight of {numel} elements has no rows of {features}" if op == L.LINEAR_FORWARD
                             else f"{name}: a weight of {numel} elements does not have {features} rows", L.ERR_SHAPE)
    block, size = _BLOCK[kind]
    nout, nin = (other, features) if op == L.LINEAR_FORWARD else (features, other)
    return other, nout, nin, (numel + block - 1) // block * size


def _product(name, op, x, w, out, out_dtype, dtype, what):
    if not isinstance(w, QuantizedTensor) or w.kind not in _BLOCK:
        raise L.OdysseyError(f"{name} takes a weight of the 4-bit kinds", L.ERR_ARG)
    r = _Rows(x, dtype, what)
    if r.grad:
        _no_graph(name, x)
    if out is not None:
        _no_graph(name, out)
    other, nout, nin, need = _weight(name, op, w.kind, w.original_numel, r.cols)
    data = w.data
    if _count_bytes(data, "the weight's buffer") != need:
        raise L.OdysseyError(f"quantised buffer has {L.numel(data)} bytes, expected {need}", L.ERR_SHAPE)
    code = r.code if out_dtype is None else _code(out_dtype)
    y = _out(r, out, (*r.lead, other), code, "out")
    lib = L.lib()
    _same_place(r, data)
    if not r.cuda:
        fn = lib.ody_fp4_linear if op == L.LINEAR_FORWARD else lib.ody_fp4_linear_dgrad
        data = L.contiguous(data)  # a copy of a strided buffer has to outlive the call
        L.check(fn(w.kind, L.ptr(data), float(w.tensor_scale), nout, nin, r.ptr, r.code, r.rows, L.ptr(y), code))
        return y
    data = _flat(data)
    ts, alpha = None, 1.0
    if w.kind == L.Q_NVFP4_TENSOR:
        if L.is_torch(w.tensor_scale):  # a device float: read by the kernel, no synchronisation
            _same_place(r, w.tensor_scale)
            _no_graph(name, w.tensor_scale)
            if w.tensor_scale.numel() != 1 or w.tensor_scale.dtype != L._torch().float32:
                raise L.OdysseyError("the tensor scale must be one float32", L.ERR_DTYPE)
            ts = w.tensor_scale.data_ptr()
        else:
            alpha = w.tensor_scale
    index = r.a.get_device()
    ws, at, n = _workspace(r.a, _workspace_bytes(index, op, w.kind, r.rows, nout, nin, r.code))
    _enqueue(index, lib.ody_fp4_linear_on_stream if op == L.LINEAR_FORWARD else lib.ody_fp4_linear_dgrad_on_stream, w.kind,
             data.data_ptr(), ts, alpha, nout, nin, r.ptr, r.code, r.rows, r.ld, y.data_ptr(), code, other, at, n)
    return y


def fp4_linear(x, w, out=None, out_dtype=None, dtype=None):
    """y[..., out_features] = x[..., in_features] W^T with W the 4-bit weight
    [w.original_numel / in_features, in_features].  out_dtype: x's by default."""
    return _product("fp4_linear", L.LINEAR_FORWARD, x, w, out, out_dtype, dtype, "x")


def fp4_linear_dgrad(dy, w, out=None, out_dtype=None, dtype=None):
    """dx[..., in_features] = dy[..., out_features] W, the input gradient of
    fp4_linear.  out_dtype: dy's by default."""
    return _product("fp4_linear_dgrad", L.LINEAR_DGRAD, dy, w, out, out_dtype, dtype, "dy")


def save_activation8(x, format="e4m3", dtype=None):
    """x[..., cols] in 8 bits ('e4m3' or 'e5m2') with a power of two per 32
    columns, the least that keeps the group's largest finite element in range."""
    fmt = FORMATS8.get(format)
    if fmt is None:
        raise L.OdysseyError(f"unknown 8-bit activation format {format!r}", L.ERR_ARG)
    r = _Rows(x, dtype, "x")
    g = (r.cols + 31) // 32
    if L.is_torch(r.a):
        u8 = L._torch().uint8
        codes, scales = r.a.new_empty((r.rows, g * 32), dtype=u8), r.a.new_empty((r.rows, g), dtype=u8)
    else:
        codes, scales = np.empty((r.rows, g * 32), np.uint8), np.empty((r.rows, g), np.uint8)
    lib = L.lib()
    if r.cuda:
        _enqueue(r.a.get_device(), lib.ody_act8_save_on_stream, fmt, r.ptr, r.code, r.rows, r.cols, r.ld,
                 codes.data_ptr(), scales.data_ptr())
    else:
        L.check(lib.ody_act8_save(fmt, r.ptr, r.code, r.rows, r.cols, L.ptr(codes), L.ptr(scales)))
    return Activation8(codes, scales, r.rows, r.cols, format, r.lead + (r.cols,), _NAMES[r.code])


def load_activation8(a, dtype=None, out=None):
    """The values an Activation8 stands for, in the saved shape and type (or `dtype`)."""
    a.check()
    code = _code(dtype if dtype is not None else a.dtype if a.dtype is not None else L.BF16)
    shape = a.shape if a.shape is not None else (a.rows, a.cols)
    if prod(shape) != a.rows * a.cols:
        raise L.OdysseyError(f"the activation's shape {tuple(shape)} does not have the {a.rows * a.cols} elements of its rows "
                             "and columns", L.ERR_SHAPE)
    codes, scales = L.contiguous(a.codes), L.contiguous(a.scales)
    r = _Place(codes)
    _same_place(r, scales)
    y = _out(r, out, shape, code, "out")
    lib, fmt = L.lib(), FORMATS8[a.format]
    if r.cuda:
        _enqueue(codes.get_device(), lib.ody_act8_load_on_stream, fmt, codes.data_ptr(), scales.data_ptr(), a.rows, a.cols,
                 y.data_ptr(), code, a.cols)
    else:
        L.check(lib.ody_act8_load(fmt, L.ptr(codes), L.ptr(scales), a.rows, a.cols, L.ptr(y), code))
    return y


def linear_wgrad8(dy, a, add=None, alpha=1.0, out=None, out_dtype=None, dtype=None):
    """dW[out_features, in_features] = alpha dy^T x' (+ add) from dy[...,
    out_features] and the activation saved in the forward pass.  add: of the
    result's type; it may be `out` (accumulation in place).  out_dtype: add's,
    out's or dy's."""
    a.check()
    r = _Rows(dy, dtype, "dy")
    for b in (dy, add, out):
        if b is not None:
            _no_graph("linear_wgrad8", b)
    if r.rows != a.rows:
        raise L.OdysseyError(f"dy has {r.rows} rows, the saved activation {a.rows}", L.ERR_SHAPE)
    _same_place(r, a.codes, a.scales)
    if out_dtype is not None:
        code = _code(out_dtype)
    else:
        like = out if out is not None else add
        code = r.code if like is None else \
            (L.BF16 if not L.is_torch(like) and like.dtype == np.uint16 else L.dtype_code(like))
    shape = (r.cols, a.cols)
    y = _out(r, out, shape, code, "out")
    if add is not None:
        add = _out(r, add, shape, code, "add")
    codes, scales = L.contiguous(a.codes), L.contiguous(a.scales)
    fmt, lib = FORMATS8[a.format], L.lib()
    if r.cuda:
        index = r.a.get_device()
        ws, at, n = _workspace(r.a, _workspace_bytes(index, L.LINEAR_WGRAD, fmt, r.rows, r.cols, a.cols, r.code))
        _enqueue(index, lib.ody_linear_wgrad8_on_stream, fmt, codes.data_ptr(), scales.data_ptr(), a.rows, a.cols, r.ptr,
                 r.code, r.cols, r.ld, alpha, None if add is None else add.data_ptr(), y.data_ptr(), code, at, n)
    else:
        L.check(lib.ody_linear_wgrad8(fmt, L.ptr(codes), L.ptr(scales), a.rows, a.cols, r.ptr, r.code, r.cols,
                                      C.c_float(alpha), None if add is None else L.ptr(add), L.ptr(y), code))
    return y


def linear_status(device=None):
    """Waits for torch's current stream of the device and raises if a bounded
    wait inside a linear kernel ran out there since the last query (the CUDA
    calls above do not wait, so they cannot say so themselves)."""
    t = L._torch()
    index = None if device is None else t.device(device).index
    _enqueue(t.cuda.current_device() if index is None else index, L.lib().ody_linear_status)
