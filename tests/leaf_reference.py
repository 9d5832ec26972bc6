"""Plain 64-bit forms of the operators over leaves and many classes, and the
bounds of what a right f32 computation may be off by."""
import numpy as np

EPS32 = 2.0 ** -24   # half a step of f32, relative
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


def to_bf16(x):
    """f32 rounded to bf16 (nearest, ties to even), as its 16 bits."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(np.asarray(x, np.float32))
    return np.where(nan, np.uint16(0x7FC0), r).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def rounded(x, dtype):
    """The values of x that the type holds, in f64."""
    x = np.asarray(x, np.float32)
    return (from_bf16(to_bf16(x)) if dtype == "bfloat16" else x).astype(np.float64)


def places(ids, offset, table_rows):
    """Each id's table row, -1 where it adds nothing."""
    ids = np.asarray(ids, np.int64)
    if offset is None:
        return np.where((ids >= 0) & (ids < table_rows), ids, -1)
    row = ids + np.asarray(offset, np.int64)[None, :]
    end = np.append(np.asarray(offset, np.int64)[1:], table_rows)[None, :]
    return np.where((ids >= 0) & (row >= 0) & (row < np.minimum(end, table_rows)), row, -1)


def embedding(table, ids, offset, scale, dtype):
    """(out, bound): one product and one addition a column, one rounding."""
    n, columns = ids.shape
    s = np.ones(columns) if scale is None else np.asarray(scale, np.float64)
    at = places(ids, offset, len(table))
    out, size = np.zeros((n, table.shape[1])), np.zeros((n, table.shape[1]))
    for t in range(columns):
        ok = at[:, t] >= 0
        part = s[t] * table[at[ok, t]]
        out[ok] += part
        size[ok] += np.abs(part)
    return out, (columns + 1) * EPS32 * size + HALF[dtype] * np.abs(out) + 1e-37


def embedding_grad(dout, ids, offset, scale, table_rows, dtype):
    """(dtable, bound): a product and an addition an id, the parts' sums
    after them (no more additions than ids), one rounding."""
    n, columns = ids.shape
    s = np.ones(columns) if scale is None else np.asarray(scale, np.float64)
    at = places(ids, offset, table_rows)
    out, size = np.zeros((table_rows, dout.shape[1])), np.zeros((table_rows, dout.shape[1]))
    count = np.zeros((table_rows, 1))
    for t in range(columns):
        ok = at[:, t] >= 0
        np.add.at(out, at[ok, t], s[t] * dout[ok])
        np.add.at(size, at[ok, t], np.abs(s[t] * dout[ok]))
        np.add.at(count, at[ok, t], 1.0)
    return out, (2 * count + 1) * EPS32 * size + HALF[dtype] * np.abs(out) + 1e-37


def head(h, w, bias, labels, weight, scale, dtype):
    """The softmax head in f64 with each output's bound, as name ->
    (value, bound). Bounds, in half steps e of f32:
    z: dim + 4 roundings of its products' sizes (a product made of the parts
      of its factors is off by less than two more);
    lse: the largest bound of its z, and K + 16 roundings of the sum of its
      exponentials, each off by the argument's rounding (|z - max| e) and two
      steps of its own;
    loss: those of lse and z, and two roundings;
    pair: p (bound of z + bound of lse + (|z - lse| + 8) e) c a, one more of
      its own and one to the type that the products take;
    gradients: their pairs' bounds, one rounding a term, one to the type."""
    n, dim = h.shape
    k = len(w)
    z, zs = h @ w.T, np.abs(h) @ np.abs(w.T)
    if bias is not None:
        z, zs = z + bias, zs + np.abs(np.where(np.isfinite(bias), bias, 0.0))
    ez = (dim + 4) * EPS32 * zs
    top = z.max(1, keepdims=True)
    e = np.exp(z - np.where(np.isfinite(top), top, 0.0))
    lse = np.where(np.isfinite(top), top, 0.0)[:, 0] + np.log(e.sum(1))
    share = e / e.sum(1, keepdims=True)
    gap = np.where(np.isfinite(z), np.abs(z - top), 0.0)
    elz = (ez.max(1) + (k + 16) * EPS32 + (share * (gap + 4)).sum(1) * EPS32 + 2 * EPS32 * np.abs(lse))
    out = {"lse": (lse, elz), "best": (z.argmax(1), None)}
    if labels is None:
        out["loss"] = (lse - z.max(1), elz + ez.max(1) + 2 * EPS32 * np.abs(lse))
        return out
    a = np.where(labels < 0, 0.0, np.ones(n) if weight is None else weight)
    y = np.maximum(labels, 0)
    zy, ezy = z[np.arange(n), y], ez[np.arange(n), y]
    loss = np.where(labels < 0, 0.0, a * (lse - zy))
    out["loss"] = (loss, np.where(labels < 0, 0.0, np.abs(a) * (elz + ezy + 2 * EPS32 * (np.abs(lse) + np.abs(zy)))
                                  + 2 * EPS32 * np.abs(loss)))
    one = np.zeros((n, k))
    one[np.arange(n), y] = 1.0
    c = (scale * a)[:, None]
    live = labels >= 0
    far = np.where(np.isfinite(z), np.abs(z - lse[:, None]), 0.0)
    g = np.where(live[:, None], c * (share - one), 0.0)
    eg = np.where(live[:, None], np.abs(c) * share * (ez + elz[:, None] + (far + 8) * EPS32), 0.0)
    eg = eg + 2 * EPS32 * np.abs(g)
    out["db"] = (g.sum(0), eg.sum(0) + (n + 1) * EPS32 * np.abs(g).sum(0) + 1e-37)
    eg = eg + HALF[dtype] * np.abs(g)
    hz = np.where(live[:, None], h, 0.0)
    for name, value, err, size, terms in (("dh", g @ w, eg @ np.abs(w), np.abs(g) @ np.abs(w), k),
                                          ("dw", g.T @ hz, eg.T @ np.abs(hz), np.abs(g.T) @ np.abs(hz), n)):
        out[name] = (value, err + (terms + 4) * EPS32 * size + HALF[dtype] * (np.abs(value) + err) + 1e-37)
    return out
