"""Operators over a forest's leaves and over many classes, on device memory.

A forest grows one tree per class and round, so a problem of hundreds of
classes or more is modelled on its leaves instead: every row has one leaf a
tree (``Forest.predict_margin_device`` writes their ids on the device), each
leaf a vector, and the sum of a row's vectors is scored against every class::

    # off[t]: the table rows before tree t's own, ascending
    hb.leaf_embedding(table, ids, h, offset=off)          # h[r] = sum of its leaves' vectors
    ws = empty(hb.softmax_head_workspace(n, k, dim, "bfloat16"))
    hb.softmax_head(h, w, labels=y, loss=loss, dh=dh, dw=dw, grad_scale=1 / n, workspace=ws)
    hb.leaf_embedding_grad(dh, ids, dtable, offset=off, workspace=ws2)
    hb.clip_gradients([dtable, dw], 1.0, norm=norm, workspace=ws3)

Every array is device memory: a torch tensor on a GPU, or a ``DeviceArray``
over a ``DeviceBuffer``. A call queues its work on ``stream`` (a hipStream_t
as an int, or an object with a ``cuda_stream``; None: torch's current stream
of the tensors' device, the default stream for DeviceArrays) and returns; it
allocates nothing and waits for nothing, so it can be captured into a graph
(behind a first call outside one). Outputs are written into the caller's
arrays and must not overlap inputs, each other or the workspace, except where
an argument says so. A workspace holds what one call needs while it runs: one
named for the largest batch serves smaller ones of the same other sizes, and
calls, or replayed graphs, that may run at the same time need one each. The
arrays have to live until the queued work is done: torch tensors handed to a stream other than their
own want ``record_stream``.

Vectors and inputs are shorter than 2^20 elements; strides are free as long
as a row's elements lie side by side.
"""
from __future__ import annotations

import ctypes as C
import operator
import struct
import sys

from . import _capi as A

_SIZE = {"float32": 4, "bfloat16": 2, "int32": 4, "uint8": 1, "float8_e4m3fn": 1}
_CODE = {"float32": A.F32, "bfloat16": A.BF16}
_names: dict = {}


class DeviceArray:
    """A typed view of device memory the library allocated: the first
    elements of a DeviceBuffer (from ``byte_offset`` on) as an array of
    ``shape``, its rows ``stride`` elements apart (contiguous when None)."""

    def __init__(self, buffer, dtype, shape, stride=None, byte_offset=0):
        self.buffer = buffer
        self.dtype = _dtype(dtype)
        self.shape = (int(shape),) if isinstance(shape, int) else tuple(int(s) for s in shape)
        if len(self.shape) > 2 or min(self.shape, default=0) < 0:
            raise ValueError("a DeviceArray has one or two axes")
        row = self.shape[-1] if stride is None else int(stride)
        self._stride = (row, 1) if len(self.shape) == 2 else (1,)
        self.ordinal = buffer.ordinal
        self._ptr = buffer.ptr + byte_offset
        rows = self.shape[0] if len(self.shape) == 2 else 1
        end = ((rows - 1) * row + self.shape[-1]) * _SIZE[self.dtype] if rows and self.shape[-1] else 0
        if byte_offset < 0 or byte_offset + end > buffer.nbytes or row < 0:
            raise ValueError("the array does not fit its buffer")

    def data_ptr(self):
        return self._ptr

    def get_device(self):
        return self.ordinal

    def numel(self):
        return self.shape[0] * (self.shape[1] if len(self.shape) == 2 else 1)

    def is_contiguous(self):
        return len(self.shape) == 1 or self.shape[0] <= 1 or self._stride[0] == self.shape[1]

    def stride(self):
        return self._stride


def _dtype(d):
    """A type's name: a string, or torch's or numpy's type object."""
    name = _names.get(d)
    if name is None:
        name = str(getattr(d, "name", None) or getattr(d, "__name__", d)).rsplit(".", 1)[-1]
        if name not in _SIZE:
            raise ValueError(f"unsupported type {d}: the operators take float32 or bfloat16 arrays and int32 ids")
        _names[d] = name
    return name


def _code(d):
    code = _CODE.get(_dtype(d))
    if code is None:
        raise ValueError(f"float32 or bfloat16 is needed, not {_dtype(d)}")
    return code


def _size(v, what, bits=32):
    """A size that its field holds (the record's fields would cut it off)."""
    v = operator.index(v)
    if not 0 <= v < 1 << bits:
        raise ValueError(f"{what}: {v} is not from 0 to 2^{bits} - 1")
    return v


class _Call:
    """One call's arrays: their device must be one, and names its stream."""

    def __init__(self):
        self.ordinal = None
        self.torch = False
        self.kind = None  # the class of the last array whose device was looked at

    def device(self, a, what):
        if isinstance(a, DeviceArray):
            ordinal = a.ordinal
        else:
            ordinal = a.get_device()
            if ordinal < 0:
                raise ValueError(f"{what}: not in device memory")
            if not self.torch:
                _one_runtime()
                self.torch = True
        if self.ordinal is None:
            self.ordinal = ordinal
        elif self.ordinal != ordinal:
            raise ValueError(f"{what}: on device {ordinal}, the others on {self.ordinal}")
        self.kind = a.__class__

    def array(self, a, what, ndim, dtypes, shape=None):
        """(address, shape, row stride) of an array whose last axis is contiguous."""
        dims = a.shape
        if len(dims) != ndim:
            raise ValueError(f"{what}: {ndim} axes are needed, not {len(dims)}")
        if (_names.get(a.dtype) or _dtype(a.dtype)) not in dtypes:
            raise ValueError(f"{what}: {' or '.join(dtypes)} is needed, not {_dtype(a.dtype)}")
        if shape is not None and dims != shape:
            raise ValueError(f"{what}: the shape {shape} is needed, not {tuple(dims)}")
        if a.__class__ is not self.kind or a.get_device() != self.ordinal:
            self.device(a, what)
        st = a.stride()
        if dims[-1] > 1 and st[-1] != 1:
            raise ValueError(f"{what}: the elements of a row must be contiguous")
        if ndim == 1:
            return a.data_ptr(), dims, 1
        row = st[0]
        if dims[0] <= 1 or dims[1] == 0:
            row = dims[1]  # no second row: whatever the stride says
        elif row < dims[1]:
            raise ValueError(f"{what}: the rows overlap")
        return a.data_ptr(), dims, row

    def pointer(self, a, what, dtype, n):
        """An optional vector's address."""
        return None if a is None else self.array(a, what, 1, (dtype,), (n,))[0]

    def memory(self, a):
        """A workspace's address and bytes."""
        if a is None:
            return None, 0
        p, dims, _ = self.array(a, "workspace", 1, tuple(_SIZE))
        return p, dims[0] * _SIZE[_dtype(a.dtype)]

    def stream(self, stream):
        if stream is None:
            if not self.torch:
                return None
            return _current_stream(self.ordinal)
        return getattr(stream, "cuda_stream", stream)


_raw_stream = None


def _current_stream(ordinal):
    """torch's current stream, without an object for it where torch has such a call."""
    global _raw_stream
    if _raw_stream is None:
        torch = sys.modules["torch"]
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda o: torch.cuda.current_stream(o).cuda_stream)
    return _raw_stream(ordinal)


_runtime_checked = False


def _one_runtime():
    """torch brings a HIP runtime of its own, which this library shares when
    torch is imported first. Loaded the other way round the process holds
    two, and a stream of the one means nothing to the other."""
    global _runtime_checked
    if _runtime_checked:
        return
    A.lib()
    with open("/proc/self/maps") as f:
        paths = {line.split(None, 5)[5].strip() for line in f if "libamdhip64" in line}
    if len(paths) > 1:
        raise RuntimeError("two HIP runtimes are loaded: import torch before the first call of hessboost_amd")
    _runtime_checked = True


_FLOATS = ("float32", "bfloat16")


def _lookup(call, ids, offset, scale, dtype, dim, table_rows, table_stride, out_stride):
    p, (n, columns), stride = call.array(ids, "ids", 2, ("int32",))
    return A.Lookup(_CODE[dtype], _size(dim, "dim"), n, _size(columns, "columns"), 0, table_rows, table_stride, stride, out_stride, p,
                    call.pointer(offset, "offset", "int32", columns), call.pointer(scale, "scale", "float32", columns))


def leaf_embedding(table, ids, out, *, offset=None, scale=None, stream=None):
    """out[r] = sum over columns t of scale[t] * table[offset[t] + ids[r, t]].

    ``table`` [rows, dim] and ``out`` [n, dim] are float32 or bfloat16 alike,
    ``ids`` [n, columns] int32, ``offset`` int32 and ``scale`` float32 (None:
    1) one entry a column. ``offset`` (each tree's first table row, ascending)
    gives every column its own rows, up to the next column's; with None every
    column has the whole table. An id below 0, or one that leads out of its
    column's rows, adds nothing. Sums are float32, in the order of the
    columns (of float32 vectors eight columns by themselves, then the
    eights)."""
    call = _Call()
    tp, (rows, dim), ts = call.array(table, "table", 2, _FLOATS)
    dtype = _dtype(table.dtype)
    op, _, os = call.array(out, "out", 2, (dtype,), (ids.shape[0], dim))
    p = _lookup(call, ids, offset, scale, dtype, dim, rows, ts, os)
    A.check(A.lib().hbr_leaf_embedding(call.ordinal, C.byref(p), tp, op, call.stream(stream)))


def leaf_embedding_grad_workspace(n, columns, table_rows, dim, dtype):
    """The bytes leaf_embedding_grad needs for n x columns ids, or for fewer
    rows of them."""
    out = C.c_uint64()
    dim, columns = _size(dim, "dim"), _size(columns, "columns")
    p = A.Lookup(_code(dtype), dim, _size(n, "n", 64), columns, 0, _size(table_rows, "table_rows", 64), dim, columns, dim,
                 None, None, None)
    A.check(A.lib().hbr_leaf_embedding_grad_workspace(C.byref(p), C.byref(out)))
    return out.value


def leaf_embedding_grad(dout, ids, dtable, *, offset=None, scale=None, workspace=None, stream=None):
    """The gradient of leaf_embedding in its table: dtable[v] = the sum of
    scale[t] * dout[r] over every (r, t) that leads to row v, zeros where
    none does. ``dout`` [n, dim] and ``dtable`` [rows, dim] are float32 or
    bfloat16 alike; ids, offset and scale as for leaf_embedding. Sums are
    float32, in an order that the ids alone decide."""
    call = _Call()
    tp, (rows, dim), ts = call.array(dtable, "dtable", 2, _FLOATS)
    dtype = _dtype(dtable.dtype)
    op, _, os = call.array(dout, "dout", 2, (dtype,), (ids.shape[0], dim))
    p = _lookup(call, ids, offset, scale, dtype, dim, rows, ts, os)
    w, nbytes = call.memory(workspace)
    A.check(A.lib().hbr_leaf_embedding_grad(call.ordinal, C.byref(p), op, tp, w, nbytes, call.stream(stream)))


def softmax_head_workspace(n, classes, dim, dtype, gradient=True):
    """The bytes softmax_head needs for n rows or fewer, with gradients (that
    serves calls without, too) or without."""
    out = C.c_uint64()
    A.check(A.lib().hbr_softmax_head_workspace(_size(n, "n", 64), _size(classes, "classes"), _size(dim, "dim"), _code(dtype),
                                               int(bool(gradient)), C.byref(out)))
    return out.value


def softmax_head(h, w, *, bias=None, labels=None, weight=None, grad_scale=1.0, loss=None, lse=None, best=None,
                 dh=None, dw=None, db=None, workspace=None, stream=None):
    """The softmax cross entropy of the linear layer z = h w^T + bias over
    many classes, the scores never kept, and its gradients.

    ``h`` [n, dim] and ``w`` [classes, dim] are float32 or bfloat16 alike,
    ``bias`` float32 (-inf shuts a class), ``labels`` int32, ``weight``
    float32, one entry a row. Outputs, each optional: ``lse`` [n] = log sum
    exp z; ``loss`` [n] = weight * (lse - z of the label), 0 for a row whose
    label is below 0, or without labels lse less the largest z; ``best`` [n]
    (int32) = the first class of the largest z; ``dh``, ``dw`` (the inputs'
    type) and ``db`` (float32) = the gradients of grad_scale * sum(loss).
    Rows whose label is below 0 take no part in any gradient, whatever they
    hold. A label of ``classes`` or more makes the row's lse and loss, and the
    gradients, NaN.

    bfloat16 inputs: the scores' gradients (probability less one-hot, times
    the row's weight) are rounded once to bfloat16 before the products that
    make ``dh`` and ``dw``, half a step each beside the outputs' own rounding;
    ``db`` is summed from the float32 values. With float32 inputs all of them
    stay float32."""
    call = _Call()
    hp, (n, dim), hs = call.array(h, "h", 2, _FLOATS)
    dtype = _dtype(h.dtype)
    classes = w.shape[0]
    wp, _, ws = call.array(w, "w", 2, (dtype,), (classes, dim))
    hgp = wgp = None
    hgs = wgs = dim
    if dh is not None:
        hgp, _, hgs = call.array(dh, "dh", 2, (dtype,), (n, dim))
    if dw is not None:
        wgp, _, wgs = call.array(dw, "dw", 2, (dtype,), (classes, dim))
    p = A.Softmax(_CODE[dtype], _size(dim, "dim"), n, _size(classes, "classes"), grad_scale, hs, ws, hgs, wgs, hp, wp,
                  call.pointer(bias, "bias", "float32", classes), call.pointer(labels, "labels", "int32", n),
                  call.pointer(weight, "weight", "float32", n), call.pointer(loss, "loss", "float32", n),
                  call.pointer(lse, "lse", "float32", n), call.pointer(best, "best", "int32", n), hgp, wgp,
                  call.pointer(db, "db", "float32", classes))
    m, nbytes = call.memory(workspace)
    A.check(A.lib().hbr_softmax_head(call.ordinal, C.byref(p), m, nbytes, call.stream(stream)))


def clip_gradients_workspace(n_tensors):
    """The bytes clip_gradients needs for a set of n_tensors or fewer."""
    out = C.c_uint64()
    A.check(A.lib().hbr_clip_gradients_workspace(_size(n_tensors, "n_tensors", 64), C.byref(out)))
    return out.value


def clip_gradients(grads, max_norm, *, norm=None, out=None, workspace=None, stream=None):
    """The set's 2-norm into ``norm`` (float32 [1]), and each tensor times
    min(1, max_norm / (norm + 1e-6)) into ``out`` (a list of arrays like the
    grads; None: in place). The tensors are contiguous, float32 or bfloat16,
    of any shape, and each is given once; squares are summed in float64."""
    call = _Call()
    grads = list(grads)
    out = grads if out is None or out is grads else list(out)
    if len(out) != len(grads):
        raise ValueError("out: one array a gradient is needed")
    data, sizes, codes = _whole(call, grads, "grads")
    to = data
    if out is not grads:
        to, *others = _whole(call, out, "out")
        if others != [sizes, codes]:
            raise ValueError("out: arrays of the gradients' sizes and types are needed")
    words = [w for record in zip(data, to, sizes, codes) for w in record]  # data, out, len, dtype
    records = struct.pack(f"{len(words)}Q", *words)
    np_ = call.pointer(norm, "norm", "float32", 1)
    w, nbytes = call.memory(workspace)
    if call.ordinal is None:
        return
    A.check(A.lib().hbr_clip_gradients(call.ordinal, C.cast(C.c_char_p(records), C.POINTER(A.Tensor)), len(grads), float(max_norm), np_,
                                       w, nbytes, call.stream(stream)))


def _whole(call, arrays, what):
    """Contiguous arrays of any shape as (addresses, elements, types' codes)."""
    if not all([a.is_contiguous() for a in arrays]):
        raise ValueError(f"{what}: contiguous arrays are needed")
    codes = {d: _CODE.get(_dtype(d)) for d in {a.dtype for a in arrays}}
    for d, code in codes.items():
        if code is None:
            raise ValueError(f"{what}: float32 or bfloat16 is needed, not {_dtype(d)}")
    for a in {(a.__class__, a.get_device()): a for a in arrays}.values():  # one of each kind and device
        call.device(a, what)
    return [a.data_ptr() for a in arrays], [a.numel() for a in arrays], [codes[a.dtype] for a in arrays]
