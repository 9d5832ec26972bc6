"""Operators of the layers between leaf vectors and classes, on device memory.

A row's sum of leaf vectors (``leaf_embedding``) goes through a norm and a
projection before it is scored (``softmax_head``); what the backward pass reads
of it can be kept in 8 bits::

    hb.rms_norm(h, y, weight=g, residual=r, total=r, inv=inv, codes=c, scales=s, normed=True)
    hb.linear(y, w, z, bias=b, workspace=ws)
    hb.softmax_head(z, v, labels=labels, loss=loss, dh=dz, dw=dv, grad_scale=1 / n, workspace=ws2)
    hb.linear_grad(dz, w, codes=c, scales=s, weight=g, dx=dy, dw=dw, db=db, workspace=ws3)
    hb.rms_norm_grad(dy, dh, codes=c, scales=s, inv=inv, weight=g, dweight=dg, workspace=ws4)

One projection serves many customers by low-rank adapters beside it, each row
its own (``linear``'s ``down``, ``up`` and ``ids``).

Rows in 8 bits are two arrays: ``codes`` [n, dim] (torch.float8_e4m3fn, or
uint8 of the same bits) and ``scales`` [n, packed_scales(dim)] uint8, a power of
two for every 32 columns of a row: a code stands for its e4m3 value times
2^(scale - 127). The power is the smallest, 2^-109 at least, under which no
finite element of the 32 is above 448; the values are bfloat16 exactly, off by
half of e4m3's step (2^-4 relative, or 2^-10 of the power). Infinite elements are
held as NaN.

Arrays, streams, workspaces and errors are those of the operators over leaves
(``hessboost_amd.leafops``)."""
from __future__ import annotations

import ctypes as C

from . import _capi as A
from .leafops import _CODE, _FLOATS, _Call, _code, _dtype, _size

_BYTES = ("uint8", "float8_e4m3fn")
_ALIKE = {d: (d,) for d in _FLOATS}
_UINT8, _INT32, _FLOAT32 = ("uint8",), ("int32",), ("float32",)
_packed_record, _norm_record, _norm_grad_record, _linear_record, _linear_grad_record = (
    A.packer(r) for r in (A.Packed, A.Norm, A.NormGrad, A.Linear, A.LinearGrad))


def packed_scales(dim):
    """The scales of a row of dim elements in 8 bits."""
    return -(-_size(dim, "dim") // A.PACK_BLOCK)


def _rows(call, a, what, dtypes, shape):
    """An optional array of rows: its address and row stride."""
    if a is None:
        return 0, 0
    p, _, stride = call.array(a, what, 2, dtypes, shape)
    return p, stride


def _vector(call, a, what, n, dtypes=_FLOAT32):
    """An optional vector's address."""
    return 0 if a is None else call.array(a, what, 1, dtypes, (n,))[0]


def _packed(call, codes, scales, shape):
    """Rows in 8 bits: (codes, stride, scales, stride)."""
    if (codes is None) != (scales is None):
        raise ValueError("codes and scales go together")
    if codes is None:
        return 0, 0, 0, 0
    return (*_rows(call, codes, "codes", _BYTES, shape),
            *_rows(call, scales, "scales", _UINT8, (shape[0], packed_scales(shape[1]))))


def pack_rows(x, codes, scales, *, stream=None):
    """The rows of ``x`` [n, dim] (float32 or bfloat16) in 8 bits."""
    call = _Call()
    xp, (n, dim), xs = call.array(x, "x", 2, _FLOATS)
    cp, cs, sp, ss = _packed(call, codes, scales, (n, dim))
    p = _packed_record(_CODE[_dtype(x.dtype)], _size(dim, "dim"), n, xs, cs, ss)
    A.check(A.lib().hbr_pack_rows(call.ordinal, p, xp, cp, sp, call.stream(stream)))


def unpack_rows(codes, scales, out, *, weight=None, stream=None):
    """What rows in 8 bits stand for, times ``weight`` (float32 [dim], one a
    column; None: 1), into ``out`` [n, dim] (float32 or bfloat16)."""
    call = _Call()
    op, (n, dim), os = call.array(out, "out", 2, _FLOATS)
    cp, cs, sp, ss = _packed(call, codes, scales, (n, dim))
    p = _packed_record(_CODE[_dtype(out.dtype)], _size(dim, "dim"), n, os, cs, ss)
    A.check(A.lib().hbr_unpack_rows(call.ordinal, p, cp, sp, _vector(call, weight, "weight", dim), op,
                                    call.stream(stream)))


def rms_norm(x, out=None, *, weight=None, eps=1e-6, residual=None, total=None, inv=None, codes=None, scales=None,
             normed=False, stream=None):
    """The root-mean-square norm of each row of ``x`` [n, dim], the residual
    added first: with s = x + residual, inv = 1 / sqrt(mean s^2 + eps) and
    normed = s * inv, out = normed * weight.

    ``x``, ``residual``, ``out`` and ``total`` are float32 or bfloat16 alike,
    ``weight`` [dim] and ``inv`` [n] float32. Outputs, each optional: ``out``;
    ``total`` = s; ``inv``; ``codes`` and ``scales`` = out in 8 bits, or with
    ``normed`` the normed rows, which is what the gradients read. ``out`` and
    ``total`` may each be ``x`` or ``residual`` itself. Sums are float32
    (float64 for rows beyond its range), every output is rounded once."""
    call = _Call()
    xp, (n, dim), xs = call.array(x, "x", 2, _FLOATS)
    dtype, shape = _dtype(x.dtype), (n, dim)
    alike = _ALIKE[dtype]
    rp, rs = _rows(call, residual, "residual", alike, shape)
    op, os = _rows(call, out, "out", alike, shape)
    tp, ts = _rows(call, total, "total", alike, shape)
    cp, cs, sp, ss = _packed(call, codes, scales, shape)
    p = _norm_record(_CODE[dtype], _size(dim, "dim"), n, xs, rs, os, ts, cs, ss, xp, rp,
               _vector(call, weight, "weight", dim), op, tp, _vector(call, inv, "inv", n), cp, sp,
               eps, int(bool(normed)))
    A.check(A.lib().hbr_rms_norm(call.ordinal, p, call.stream(stream)))


def rms_norm_grad_workspace(n, dim, dtype):
    """The bytes rms_norm_grad needs for dweight of n rows or fewer."""
    out = C.c_uint64()
    A.check(A.lib().hbr_rms_norm_grad_workspace(_size(n, "n", 64), _size(dim, "dim"), _code(dtype), C.byref(out)))
    return out.value


def rms_norm_grad(dout, dx=None, *, x=None, codes=None, scales=None, inv=None, weight=None, eps=1e-6, dtotal=None,
                  dweight=None, workspace=None, stream=None):
    """The gradient of rms_norm: with g = dout * weight, dx = inv * (g -
    normed * mean(g * normed)) + dtotal, and dweight = the sum over rows of
    dout * normed (float32 [dim]; needs the workspace).

    The rows are ``x`` as the norm saw it (its ``total`` where there was a
    residual; ``inv`` may be None and is made of ``x`` and ``eps`` then), or
    the normed rows in 8 bits (``inv`` is needed). ``dtotal`` is the gradient
    that reaches the total by other ways. dx is the gradient of x and of the
    residual alike, and may be ``dout`` or ``dtotal`` itself."""
    call = _Call()
    gp, (n, dim), gs = call.array(dout, "dout", 2, _FLOATS)
    dtype, shape = _dtype(dout.dtype), (n, dim)
    alike = _ALIKE[dtype]
    xp, xs = _rows(call, x, "x", alike, shape)
    cp, cs, sp, ss = _packed(call, codes, scales, shape)
    tp, ts = _rows(call, dtotal, "dtotal", alike, shape)
    dp, ds = _rows(call, dx, "dx", alike, shape)
    p = _norm_grad_record(_CODE[dtype], _size(dim, "dim"), n, gs, xs, cs, ss, ts, ds, gp, xp, cp, sp,
                   _vector(call, inv, "inv", n), _vector(call, weight, "weight", dim), tp, dp,
                   _vector(call, dweight, "dweight", dim), eps, 0)
    m, nbytes = call.memory(workspace)
    A.check(A.lib().hbr_rms_norm_grad(call.ordinal, p, m, nbytes, call.stream(stream)))


def linear_workspace(n, outs, dim, dtype, rank=0):
    """The bytes linear needs for n rows or fewer, with adapters of the rank
    or less (a few rows without adapters need none)."""
    out = C.c_uint64()
    A.check(A.lib().hbr_linear_workspace(_size(n, "n", 64), _size(outs, "outs"), _size(dim, "dim"), _size(rank, "rank"),
                                         _code(dtype), C.byref(out)))
    return out.value


def _flat(call, a, what, dtypes, rows, cols):
    """An adapters' array of ``rows`` rows an adapter, [adapters, rows, cols]
    or [adapters * rows, cols]: its address, its rows' stride and how many
    adapters there are."""
    dims = a.shape
    if len(dims) == 3 and dims[1] == rows and dims[2] == cols and a.is_contiguous():
        p, _, _ = call.array(a, what, 3, dtypes)
        return p, cols, dims[0]
    if len(dims) == 3:
        if dims[1:] != (rows, cols):
            raise ValueError(f"{what}: the shape ({dims[0]}, {rows}, {cols}) is needed, not {tuple(dims)}")
        a = _joined(a, what)
        dims = a.shape
    if len(dims) != 2 or dims[1] != cols or (rows and dims[0] % rows):
        raise ValueError(f"{what}: {rows} rows of {cols} an adapter are needed, not {tuple(dims)}")
    p, _, stride = call.array(a, what, 2, dtypes)
    return p, stride, dims[0] // rows if rows else 0


def _joined(a, what):
    try:
        return a.view(a.shape[0] * a.shape[1], a.shape[2])
    except RuntimeError:
        raise ValueError(f"{what}: the adapters' rows must lie at one stride") from None


def linear(x, w, out, *, bias=None, down=None, up=None, ids=None, scale=None, workspace=None, stream=None):
    """out[r] = x[r] w^T + bias + scale[a] * ((x[r] down[a]^T) up[a]^T), a =
    ids[r]: a projection, and beside it each row's low-rank adapter.

    ``x`` [n, dim], ``w`` [outs, dim], ``out`` [n, outs], ``down`` [adapters,
    rank, dim] and ``up`` [adapters, outs, rank] are float32 or bfloat16 alike
    (down and up also as [adapters * rank, dim] and [adapters * outs, rank]),
    ``bias`` [outs] and ``scale`` [adapters] float32 (None: 0 and 1), ``ids``
    [n] int32. A row whose id is below 0, or no adapter's, has none. Rows come
    in any order; those of one adapter take the least time next to each other.
    Elements of an adapter that are no finite numbers reach its own rows alone,
    whose outputs are then infinite or NaN, as the formula has it for any number
    of rows.

    Sums are float32, the ``rank`` values between down and up (the scale in
    them) too, and the outputs are rounded once."""
    call = _Call()
    xp, (n, dim), xs = call.array(x, "x", 2, _FLOATS)
    dtype, outs = _dtype(x.dtype), w.shape[0]
    alike = _ALIKE[dtype]
    wp, _, ws = call.array(w, "w", 2, alike, (outs, dim))
    op, _, os = call.array(out, "out", 2, alike, (n, outs))
    if len({a is None for a in (down, up, ids)}) > 1:
        raise ValueError("down, up and ids go together")
    dp = up_ = ip = sp = rank = adapters = ds = us = 0
    if down is not None:
        rank = up.shape[-1]
        dp, ds, adapters = _flat(call, down, "down", alike, rank, dim)
        up_, us, more = _flat(call, up, "up", alike, outs, rank)
        if rank and more != adapters:
            raise ValueError(f"up: {adapters} adapters are needed, not {more}")
        ip = _vector(call, ids, "ids", n, _INT32)
        sp = _vector(call, scale, "scale", adapters)
    elif scale is not None:
        raise ValueError("scale: there are no adapters")
    p = _linear_record(_CODE[dtype], _size(dim, "dim"), n, _size(outs, "outs"), _size(rank, "rank"), _size(adapters, "adapters"), 0,
                 xs, ws, os, ds, us, xp, wp, _vector(call, bias, "bias", outs), dp, up_, ip, sp, op)
    m, nbytes = call.memory(workspace)
    A.check(A.lib().hbr_linear(call.ordinal, p, m, nbytes, call.stream(stream)))


def linear_grad_workspace(n, outs, dim, dtype):
    """The bytes linear_grad needs for n rows or fewer."""
    out = C.c_uint64()
    A.check(A.lib().hbr_linear_grad_workspace(_size(n, "n", 64), _size(outs, "outs"), _size(dim, "dim"), _code(dtype), C.byref(out)))
    return out.value


def linear_grad(dout, w=None, *, x=None, codes=None, scales=None, weight=None, dx=None, dw=None, db=None, workspace=None,
                stream=None):
    """The gradients of out = x w^T + bias (adapters have none here): ``dx``
    [n, dim] = dout w, ``dw`` [outs, dim] = dout^T x, ``db`` (float32 [outs]) =
    the sum of dout's rows, each optional.

    ``dout`` [n, outs], ``w`` [outs, dim] (for dx), ``x`` [n, dim] (for dw),
    ``dx`` and ``dw`` are float32 or bfloat16 alike. In x's place may stand
    rows in 8 bits, and ``weight`` (float32 [dim]) as a factor of x's columns:
    with the normed rows and the weight of a norm, x is what the norm gave.
    Sums are float32 and rounded once."""
    call = _Call()
    gp, (n, outs), gs = call.array(dout, "dout", 2, _FLOATS)
    dtype = _dtype(dout.dtype)
    alike = _ALIKE[dtype]
    dim = next((a.shape[1] for a in (w, x, codes, dx, dw) if a is not None and len(a.shape) == 2), None)
    if dim is None:  # db alone
        dim = 1
    wp, ws = _rows(call, w, "w", alike, (outs, dim))
    xp, xs = _rows(call, x, "x", alike, (n, dim))
    cp, cs, sp, ss = _packed(call, codes, scales, (n, dim))
    xgp, xgs = _rows(call, dx, "dx", alike, (n, dim))
    wgp, wgs = _rows(call, dw, "dw", alike, (outs, dim))
    p = _linear_grad_record(_CODE[dtype], _size(dim, "dim"), n, _size(outs, "outs"), 0, gs, ws, xs, cs, ss, xgs, wgs, gp, wp, xp, cp, sp,
                     _vector(call, weight, "weight", dim), xgp, wgp, _vector(call, db, "db", outs))
    m, nbytes = call.memory(workspace)
    A.check(A.lib().hbr_linear_grad(call.ordinal, p, m, nbytes, call.stream(stream)))
