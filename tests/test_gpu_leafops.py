"""The operators over leaves and many classes against their plain forms in
64 bits, at the sizes, masks and layouts where they can go wrong."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import hessboost_amd as hb
import leaf_reference as R
from hessboost_amd import _capi as A
from hessboost_amd.leafops import DeviceArray

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16")
_BITS = {"float32": np.uint32, "bfloat16": np.uint16, "int32": np.uint32, "uint8": np.uint8}


def dev(values, dtype, pad=0, lead=0):
    """The values on the device, rows `pad` elements apart beyond their own,
    `lead` elements into the buffer; the gaps hold NaN bits."""
    v = np.asarray(values)
    if dtype == "bfloat16":
        bits = R.to_bf16(v)
    elif dtype == "float32":
        bits = np.ascontiguousarray(v, np.float32).view(np.uint32)
    else:
        bits = np.ascontiguousarray(v, np.int32).view(np.uint32)
    rows, cols = (1, v.shape[0]) if v.ndim == 1 else v.shape
    stride = cols + pad
    whole = np.full(lead + rows * stride, 0x7FC0 if dtype == "bfloat16" else 0x7FC00000, _BITS[dtype])
    for r in range(rows):
        whole[lead + r * stride: lead + r * stride + cols] = bits.reshape(rows, cols)[r]
    buf = hb.DeviceBuffer(max(16, whole.nbytes))
    if whole.nbytes:
        buf.upload(whole)
    size = whole.itemsize
    a = DeviceArray(buf, dtype, v.shape, stride=stride if v.ndim == 2 else None, byte_offset=lead * size)
    a.lead, a.pad = lead, pad
    return a


def like(shape, dtype, pad=0, lead=0):
    """An output array: every element, and the gaps, NaN bits."""
    a = dev(np.full(shape, np.nan) if dtype != "int32" else np.full(shape, 0x7FC00000), dtype, pad, lead)
    return a


def back(a):
    """The array's values (f64, or int32); the gaps must still hold their bits."""
    bits = _BITS[a.dtype]
    whole = a.buffer.download(bits, a.buffer.nbytes // np.dtype(bits).itemsize)
    rows, cols = (1, a.shape[0]) if len(a.shape) == 1 else a.shape
    stride = cols + a.pad
    body = whole[a.lead: a.lead + rows * stride].reshape(rows, stride)
    gap = 0x7FC0 if a.dtype == "bfloat16" else 0x7FC00000
    assert np.all(whole[:a.lead] == gap) and np.all(body[:, cols:] == gap), "written outside the array"
    v = np.ascontiguousarray(body[:, :cols]).reshape(a.shape)
    if a.dtype == "bfloat16":
        return R.from_bf16(v).astype(np.float64)
    if a.dtype == "float32":
        return v.view(np.float32).astype(np.float64)
    return v.view(np.int32)


def work(nbytes):
    """A workspace of just the bytes asked for, full of NaN bits."""
    buf = hb.DeviceBuffer(max(16, nbytes))
    buf.upload(np.full(max(16, nbytes) // 4 + 1, 0x7FC00001, np.uint32).view(np.uint8)[:max(16, nbytes)])
    return DeviceArray(buf, "uint8", nbytes)


def close(got, want, what=""):
    value, bound = want
    both = np.isnan(value) & np.isnan(got)
    same = (got == value) | both  # infinities
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, np.abs(got - value))
    worst = np.max(np.where(same, 0.0, off / bound)) if off.size else 0.0
    assert np.all(same | (off <= bound)), f"{what}: {worst} times the bound"


# ---- leaf vectors ------------------------------------------------------------------

# rows, columns, table rows a column, dim, dtype, offsets, scale, padded share, stride gaps, lead
LOOKUPS = [
    (1, 1, 1, 1, "float32", False, False, 0.0, 0, 0),
    (1, 1, 5, 8, "bfloat16", False, True, 0.0, 0, 0),
    (3, 2, 7, 5, "float32", True, True, 0.3, 3, 1),
    (3, 2, 7, 5, "bfloat16", True, True, 0.3, 2, 1),
    (33, 9, 15, 16, "float32", True, True, 0.0, 0, 0),
    (257, 17, 31, 50, "float32", True, False, 0.1, 0, 0),
    (257, 17, 31, 50, "bfloat16", True, False, 0.1, 0, 0),
    (1000, 100, 127, 64, "bfloat16", True, True, 0.0, 0, 0),
    (1000, 23, 127, 32, "float32", True, True, 0.0, 8, 4),
    (4097, 3, 511, 24, "bfloat16", True, True, 0.5, 8, 8),
    (5000, 1, 9001, 96, "bfloat16", False, True, 0.02, 0, 0),
    (300, 1, 70_001, 257, "float32", False, True, 0.02, 0, 0),
    (130, 2, 40, 1030, "bfloat16", True, False, 0.0, 2, 0),
    (64, 5, 12, 3, "float32", True, True, 1.0, 0, 0),        # nothing adds
    (20_000, 4, 3, 8, "float32", True, True, 0.0, 0, 0),     # a few rows hold every id
    (9000, 1, 2, 40, "bfloat16", False, False, 0.0, 0, 0),
    (300, 100, 9, 8, "bfloat16", True, True, 0.1, 0, 0),     # several passes over the columns
    (9, 2100, 3, 2056, "bfloat16", True, True, 0.1, 0, 0),   # and over the vectors
    (7, 1300, 3, 1028, "float32", True, False, 0.0, 4, 0),
    (0, 3, 4, 8, "float32", True, True, 0.0, 0, 0),
    (5, 0, 4, 8, "float32", False, False, 0.0, 0, 0),
]


def lookup_case(case, seed=0):
    n, columns, rows, dim, dtype, offsets, scaled, padded, gap, lead = case
    rng = np.random.default_rng([seed, n, columns, dim])
    table_rows = rows * max(1, columns) if offsets else rows
    ids = np.minimum((rng.random((n, columns)) ** 2 * rows).astype(np.int32), rows - 1)
    drop = rng.random((n, columns)) < padded
    # ids that add nothing: negative ones, and ones past the table's end
    ids = np.where(drop, np.where(rng.random((n, columns)) < 0.5, -1 - ids, 2_000_000_000 + ids), ids).astype(np.int32)
    off = (np.arange(columns) * rows).astype(np.int32) if offsets else None
    s = (rng.random(columns) + 0.5).astype(np.float32) if scaled else None
    return dict(n=n, columns=columns, table_rows=table_rows, dim=dim, dtype=dtype, ids=ids, offset=off, scale=s,
                gap=gap, lead=lead, rng=rng)


def vec(v, dtype):
    return None if v is None else dev(v, dtype)


@pytest.mark.parametrize("case", LOOKUPS)
def test_leaf_embedding_sums_the_rows_of_its_ids(case):
    c = lookup_case(case)
    table = R.rounded(c["rng"].standard_normal((c["table_rows"], c["dim"])), c["dtype"])
    out = like((c["n"], c["dim"]), c["dtype"], c["gap"], c["lead"])
    hb.leaf_embedding(dev(table, c["dtype"], c["gap"], c["lead"]), dev(c["ids"], "int32", c["gap"]), out,
                      offset=vec(c["offset"], "int32"), scale=vec(c["scale"], "float32"))
    close(back(out), R.embedding(table, c["ids"], c["offset"], c["scale"], c["dtype"]), "out")


@pytest.mark.parametrize("case", LOOKUPS)
def test_leaf_embedding_grad_sums_the_rows_that_lead_to_each_place(case):
    c = lookup_case(case, 1)
    dout = R.rounded(c["rng"].standard_normal((c["n"], c["dim"])), c["dtype"])
    dtable = like((c["table_rows"], c["dim"]), c["dtype"], c["gap"], c["lead"])
    args = (dev(dout, c["dtype"], c["gap"], c["lead"]), dev(c["ids"], "int32", c["gap"]), dtable)
    kw = dict(offset=vec(c["offset"], "int32"), scale=vec(c["scale"], "float32"),
              workspace=work(hb.leaf_embedding_grad_workspace(c["n"], c["columns"], c["table_rows"], c["dim"],
                                                              c["dtype"])))
    hb.leaf_embedding_grad(*args, **kw)
    got = back(dtable)
    want = R.embedding_grad(dout, c["ids"], c["offset"], c["scale"], c["table_rows"], c["dtype"])
    close(got, want, "dtable")
    assert np.all(got[want[0].any(1) == 0] == 0)
    hb.leaf_embedding_grad(*args, **kw)  # the same bits on a used workspace
    assert np.array_equal(back(dtable), got)


def test_sums_of_many_columns_lose_no_more_than_a_few_steps():
    """One vector of 1 and 127 of a little less than half a step of it. Eight
    columns are summed by themselves, then added: a product and seven
    additions, then one addition for each eight columns, each off by half a
    step of the sum at most."""
    columns, dim = 128, 8
    table = np.full((2, dim), 0.9 * 2.0 ** -24)
    table[0] = 1.0
    table = R.rounded(table, "float32")
    ids = np.ones((3, columns), np.int32)
    ids[0, 0] = ids[1, columns // 2] = ids[2, 7] = 0
    out = like((3, dim), "float32")
    hb.leaf_embedding(dev(table, "float32"), dev(ids, "int32"), out)
    want, _ = R.embedding(table, ids, None, None, "float32")
    close(back(out), (want, (8 + columns / 8) * R.EPS32 * want))


# table rows few and many against the ids, so that either way of the gradient runs
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offsets", [None, (0, 0, 5, 6, 30, 41), (3, 9, 20, 30, 40, 50), (-7, -2, 0, 600, 1000, 1500),
                                     (0, 100, 200, 300, 400, 5000)])
@pytest.mark.parametrize("rows", [50, 2000, 40_000])
def test_columns_hold_the_table_rows_up_to_the_next(offsets, rows, dtype):
    """Columns that share the table, empty ones, ones that begin before or
    behind it, ids past a column's end, and the same id twice in a row."""
    rng = np.random.default_rng(3)
    n, columns, dim = 700, 6, 12
    ids = rng.integers(-3, 40, (n, columns)).astype(np.int32)
    ids[::7] = rng.integers(0, 3000, ids[::7].shape)
    off = None if offsets is None else np.array(offsets, np.int32)
    s = rng.standard_normal(columns).astype(np.float32)
    table = R.rounded(rng.standard_normal((rows, dim)), dtype)
    out, dtable = like((n, dim), dtype), like((rows, dim), dtype)
    d = dict(offset=vec(off, "int32"), scale=dev(s, "float32"))
    hb.leaf_embedding(dev(table, dtype), dev(ids, "int32"), out, **d)
    close(back(out), R.embedding(table, ids, off, s, dtype))
    dout = R.rounded(rng.standard_normal((n, dim)), dtype)
    hb.leaf_embedding_grad(dev(dout, dtype), dev(ids, "int32"), dtable,
                           workspace=work(hb.leaf_embedding_grad_workspace(n, columns, rows, dim, dtype)), **d)
    close(back(dtable), R.embedding_grad(dout, ids, off, s, rows, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, rows, columns, dim, few", [
    (16_384, 512, 1, 8, 512),       # one block, one round of keys
    (16_385, 513, 1, 24, 513),      # a row more, a key more
    (40_000, 1200, 1, 130, 3),      # three rounds of keys; three rows hold all ids
    (5_000, 3, 1, 300, 3),          # fewer rows than waves, several slices
    (700, 700, 20, 65, 1),          # every id of a column alike
    (50_001, 31, 7, 20, 31),
])
def test_many_ids_a_table_row(n, rows, columns, dim, few, dtype):
    """Blocks of rows, rounds of keys, slices of the vectors, and keys that
    reach over several waves' shares."""
    rng = np.random.default_rng(n)
    ids = rng.integers(0, few, (n, columns)).astype(np.int32)
    off = (np.arange(columns) * rows).astype(np.int32) if columns > 1 else None
    total = rows * columns
    dout = R.rounded(rng.standard_normal((n, dim)), dtype)
    dtable = like((total, dim), dtype)
    hb.leaf_embedding_grad(dev(dout, dtype), dev(ids, "int32"), dtable, offset=vec(off, "int32"),
                           workspace=work(hb.leaf_embedding_grad_workspace(n, columns, total, dim, dtype)))
    close(back(dtable), R.embedding_grad(dout, ids, off, None, total, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim", [(3_000, 65), (3_000, 127), (400, 193), (20_000, 129)])
def test_columns_of_odd_widths_take_slices_of_single_elements(n, dim, dtype):
    """Vectors that no wider load divides: 64 elements a slice and not 128."""
    c = lookup_case((n, 9, 15, dim, dtype, True, True, 0.1, 0, 0), 5)
    dout = R.rounded(c["rng"].standard_normal((n, dim)), dtype)
    dtable = like((c["table_rows"], dim), dtype)
    hb.leaf_embedding_grad(dev(dout, dtype), dev(c["ids"], "int32"), dtable, offset=dev(c["offset"], "int32"),
                           scale=dev(c["scale"], "float32"),
                           workspace=work(hb.leaf_embedding_grad_workspace(n, 9, c["table_rows"], dim, dtype)))
    close(back(dtable), R.embedding_grad(dout, c["ids"], c["offset"], c["scale"], c["table_rows"], dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_no_id_leads_to_is_not_read(dtype):
    """NaN and infinities in table rows, or in rows of dout, that no id leads
    to or from; a NaN that one leads to reaches its sums alone."""
    rng = np.random.default_rng(4)
    n, rows, dim = 300, 20, 10
    ids = (2 * rng.integers(0, rows // 2, (n, 3))).astype(np.int32)
    ids[5] = -1
    ids[7] = [4, -2, rows]
    table = R.rounded(rng.standard_normal((rows, dim)), dtype)
    table[1::2] = np.nan
    table[3] = np.inf
    out = like((n, dim), dtype)
    hb.leaf_embedding(dev(table, dtype), dev(ids, "int32"), out)
    clean = np.where(np.isfinite(table), table, 0.0)
    close(back(out), R.embedding(clean, ids, None, None, dtype))
    dout = R.rounded(rng.standard_normal((n, dim)), dtype)
    dout[5] = np.nan
    dout[7] = np.inf
    dtable = like((rows, dim), dtype)
    hb.leaf_embedding_grad(dev(dout, dtype), dev(ids, "int32"), dtable,
                           workspace=work(hb.leaf_embedding_grad_workspace(n, 3, rows, dim, dtype)))
    got, rest = back(dtable), ids.copy()
    assert np.all(np.isinf(got[4]))
    rest[7] = -1
    want, bound = R.embedding_grad(np.where(np.isfinite(dout), dout, 0.0), rest, None, None, rows, dtype)
    keep = np.arange(rows) != 4
    close(got[keep], (want[keep], bound[keep]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, rows", [(3, 9), (700, 9), (3000, 900)])
@pytest.mark.parametrize("bad", [np.inf, np.nan, -2.0])
def test_a_scale_reaches_only_what_its_column_leads_to(bad, n, rows, dtype):
    """By columns, in one block and several, and by sorting."""
    rng = np.random.default_rng(n)
    dim = 12
    ids = rng.integers(0, rows // 2, (n, 3)).astype(np.int32)  # half of a column's rows have none
    ids[::2, 1] = -1
    off, s = np.arange(3, dtype=np.int32) * rows, np.float32([0.5, bad, 1.5])
    table = R.rounded(rng.random((3 * rows, dim)) + 0.5, dtype)
    d = dict(offset=dev(off, "int32"), scale=dev(s, "float32"))
    out, finite = like((n, dim), dtype), np.where(np.isfinite(s), s, 1.0).astype(np.float32)
    hb.leaf_embedding(dev(table, dtype), dev(ids, "int32"), out, **d)
    got, want = back(out), R.embedding(table, ids, off, finite, dtype)
    close(got[::2], (want[0][::2], want[1][::2]))
    if not np.isfinite(bad):
        assert not np.isfinite(got[1::2]).any()
    dout, dtable = R.rounded(rng.random((n, dim)) + 0.5, dtype), like((3 * rows, dim), dtype)
    hb.leaf_embedding_grad(dev(dout, dtype), dev(ids, "int32"), dtable, **d,
                           workspace=work(hb.leaf_embedding_grad_workspace(n, 3, 3 * rows, dim, dtype)))
    got, (want, bound) = back(dtable), R.embedding_grad(dout, ids, off, finite, 3 * rows, dtype)
    hit = np.zeros(3 * rows, bool)
    hit[rows + ids[1::2, 1]] = not np.isfinite(bad)
    close(got[~hit], (want[~hit], bound[~hit]))
    assert not np.isfinite(got[hit]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, columns, rows, dim", [
    (600_000, 1, 90_001, 4),       # the sort's large tiles, two passes
    (300_001, 3, 1 << 18, 3),      # and three, tiles that end inside, no offsets
    (5_000, 1, (1 << 18) + 9, 20), # three passes of small tiles
    (1_100, 1, 1 << 19, 8)])
def test_sorts_of_many_ids_and_of_large_tables(n, columns, rows, dim, dtype):
    rng = np.random.default_rng(n)
    ids = np.minimum((rng.random((n, columns)) ** 2 * rows).astype(np.int32), rows - 1)
    ids[rng.random((n, columns)) < 0.02] = -1
    ids[::5000] = rows - 1
    s = (rng.random(columns) + 0.5).astype(np.float32)
    dout = R.rounded(rng.standard_normal((n, dim)), dtype)
    dtable = like((rows, dim), dtype)
    hb.leaf_embedding_grad(dev(dout, dtype), dev(ids, "int32"), dtable, scale=dev(s, "float32"),
                           workspace=work(hb.leaf_embedding_grad_workspace(n, columns, rows, dim, dtype)))
    got = back(dtable)
    want = R.embedding_grad(dout, ids, None, s, rows, dtype)
    close(got, want)
    assert np.all(got[want[0].any(1) == 0] == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [300, 40_000])
def test_rows_that_no_id_leads_from_are_not_read_by_columns(n, dtype):
    """NaN in rows of dout whose ids add nothing, with columns of their own."""
    rng = np.random.default_rng(n)
    rows, columns, dim = 9, 3, 20
    ids = rng.integers(0, rows, (n, columns)).astype(np.int32)
    dead = rng.random(n) < 0.1
    ids[dead] = np.where(rng.random((dead.sum(), columns)) < 0.5, -1, 5 * rows)
    off = np.arange(columns, dtype=np.int32) * rows
    dout = R.rounded(rng.standard_normal((n, dim)), dtype)
    want = R.embedding_grad(dout, ids, off, None, rows * columns, dtype)
    dout[dead] = np.where(rng.random((dead.sum(), dim)) < 0.5, np.nan, np.inf)
    dtable = like((rows * columns, dim), dtype)
    hb.leaf_embedding_grad(dev(dout, dtype), dev(ids, "int32"), dtable, offset=dev(off, "int32"),
                           workspace=work(hb.leaf_embedding_grad_workspace(n, columns, rows * columns, dim, dtype)))
    close(back(dtable), want)


def test_an_embedding_gradient_is_the_differences_of_its_sum():
    """<out, dout> is linear in the table: a step along any direction changes
    it by <dtable, direction>, up to both sides' rounding bounds."""
    c = lookup_case((500, 7, 31, 20, "float32", True, True, 0.1, 0, 0), 2)
    rng = c["rng"]
    table = R.rounded(rng.standard_normal((c["table_rows"], c["dim"])), "float32")
    step = R.rounded(rng.standard_normal(table.shape), "float32")
    dout = R.rounded(rng.standard_normal((c["n"], c["dim"])), "float32")
    d = dict(offset=dev(c["offset"], "int32"), scale=dev(c["scale"], "float32"))
    ids, sums, slack = dev(c["ids"], "int32"), [], 0.0
    for t in (R.rounded(table + step, "float32"), R.rounded(table - step, "float32")):
        out = like((c["n"], c["dim"]), "float32")
        hb.leaf_embedding(dev(t, "float32"), ids, out, **d)
        sums.append(np.sum(back(out) * dout))
        slack += np.sum(R.embedding(t, c["ids"], c["offset"], c["scale"], "float32")[1] * np.abs(dout))
    moved = R.rounded(table + step, "float32") - R.rounded(table - step, "float32")
    dtable = like(table.shape, "float32")
    hb.leaf_embedding_grad(dev(dout, "float32"), ids, dtable, **d,
                           workspace=work(hb.leaf_embedding_grad_workspace(c["n"], c["columns"], c["table_rows"],
                                                                           c["dim"], "float32")))
    slack += np.sum(R.embedding_grad(dout, c["ids"], c["offset"], c["scale"], c["table_rows"], "float32")[1]
                    * np.abs(moved))
    assert abs((sums[0] - sums[1]) - np.sum(back(dtable) * moved)) <= slack


def test_leaf_ids_of_a_forest_are_looked_up_where_they_lie():
    """The ids that a forest writes on the device, with its trees' offsets and
    weights and the leaf values as vectors of one element: its margins."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3_000, 6)).astype(np.float32)
    b = hb.train({"objective": "reg:squarederror", "max_depth": 5}, hb.DMatrix(x, label=x[:, 0] * x[:, 1]), 12)
    f = b.forest()
    dx, margins = hb.DeviceBuffer(x.nbytes), hb.DeviceBuffer(4 * len(x))
    leaves = hb.DeviceBuffer(4 * len(x) * f.n_trees)
    dx.upload(x)
    f.predict_margin_device(dx.ptr, len(x), x.shape[1], margins.ptr, leaves.ptr)
    values = f.arrs["leaf_value"].astype(np.float64)[:, None]
    out = like((len(x), 1), "float32")
    ids = DeviceArray(leaves, "int32", (len(x), f.n_trees))
    offset = f.arrs["tree_offset"][:-1].astype(np.int32)
    hb.leaf_embedding(dev(values, "float32"), ids, out, offset=dev(offset, "int32"))
    host_ids = leaves.download(np.int32, len(x) * f.n_trees).reshape(len(x), -1)
    want, bound = R.embedding(values, host_ids, offset, None, "float32")
    close(back(out), (want, bound))
    m = margins.download(np.float32, len(x)).astype(np.float64)
    base = float(b.base_score[0])
    assert np.all(np.abs(back(out)[:, 0] + base - m) <= 2 * bound[:, 0] + (f.n_trees + 2) * R.EPS32 * (np.abs(m) + abs(base)) * 2)


# ---- the softmax head ---------------------------------------------------------------------

# rows, classes, dim, ignored share, weights, bias, stride gap, lead
HEADS = [
    (1, 1, 1, 0.0, False, False, 0, 0),
    (1, 2, 3, 0.0, False, True, 1, 1),
    (5, 7, 8, 0.0, True, True, 0, 0),
    (64, 10, 50, 0.1, True, True, 0, 0),
    (129, 65, 33, 0.0, False, True, 3, 1),
    (300, 16, 64, 0.0, True, False, 0, 0),
    (257, 17, 40, 0.2, True, True, 0, 0),
    (70, 300, 128, 0.1, True, True, 8, 8),
    (513, 513, 96, 0.0, False, True, 0, 0),
    (33, 1000, 257, 0.5, True, True, 0, 0),
    (1025, 129, 72, 0.0, True, True, 16, 0),
    (40, 90, 20, 1.0, True, True, 0, 0),      # no row takes part
    (600, 31, 1, 0.0, False, True, 0, 0),
    (2000, 3, 12, 0.1, True, True, 0, 0),
    (0, 5, 8, 0.0, True, True, 0, 0),
    (0, 500, 300, 0.0, False, True, 0, 0),
    (600, 200, 136, 0.1, True, True, 0, 0),   # long inputs, read where they lie
    (600, 200, 136, 0.1, False, False, 24, 8),
    (33, 700, 1000, 0.0, True, True, 8, 0),
    (1030, 260, 140, 0.1, True, True, 0, 0),  # laid out first
    (2050, 129, 129, 0.0, False, True, 1, 1),
    (128, 4000, 64, 0.0, False, True, 0, 0),  # short inputs, classes shared out
    (5000, 70, 9, 0.1, True, True, 0, 0),     # and rows
    (900, 1100, 65, 0.3, False, True, 0, 0),
    (4100, 130, 136, 0.1, True, True, 0, 0),  # enough rows to lay out the classes too
    (300, 200, 97, 0.0, False, True, 0, 0),
    (2000, 64, 7, 0.2, True, True, 0, 0),     # vectors shorter than a load
    (40, 33, 515, 0.2, True, True, 5, 3),
]


def head_case(case, dtype, seed=0):
    n, classes, dim, ignored, weighted, biased, gap, lead = case
    rng = np.random.default_rng([seed, n, classes, dim])
    w = R.rounded(rng.standard_normal((classes, dim)) * 2 / np.sqrt(dim), dtype)
    h = R.rounded(rng.standard_normal((n, dim)), dtype)
    bias = R.rounded(rng.standard_normal(classes) * 0.5, "float32") if biased else None
    labels = rng.integers(0, classes, n).astype(np.int32)
    labels[rng.random(n) < ignored] = -1 - rng.integers(0, 3)
    weight = R.rounded(rng.random(n) + 0.5, "float32") if weighted else None
    return dict(n=n, classes=classes, dim=dim, w=w, h=h, bias=bias, labels=labels, weight=weight, gap=gap, lead=lead,
                dtype=dtype, scale=float(np.float32(1.0 / max(1, n))))


def run_head(c, outputs=("loss", "lse", "best", "dh", "dw", "db"), labels=True, workspace=None):
    n, classes, dim, dtype = c["n"], c["classes"], c["dim"], c["dtype"]
    shapes = dict(loss=((n,), "float32"), lse=((n,), "float32"), best=((n,), "int32"), dh=((n, dim), dtype),
                  dw=((classes, dim), dtype), db=((classes,), "float32"))
    out = {k: like(*shapes[k], *((c["gap"], c["lead"]) if k in ("dh", "dw") else ())) for k in outputs}
    gradient = any(k in out for k in ("dh", "dw", "db"))
    if workspace is None:
        workspace = work(hb.softmax_head_workspace(n, classes, dim, dtype, gradient))
    hb.softmax_head(dev(c["h"], dtype, c["gap"], c["lead"]), dev(c["w"], dtype, c["gap"], c["lead"]),
                    bias=vec(c["bias"], "float32"), labels=vec(c["labels"], "int32") if labels else None,
                    weight=vec(c["weight"], "float32"), grad_scale=c["scale"], workspace=workspace, **out)
    return {k: back(v) for k, v in out.items()}


def check_head(got, want, h_dim=None):
    for k, v in got.items():
        if k != "best":
            close(v, want[k], k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", HEADS)
def test_softmax_head_and_its_gradients(case, dtype):
    c = head_case(case, dtype)
    got = run_head(c)
    if c["n"] == 0:
        assert not got["dw"].any() and not got["db"].any()
        return
    want = R.head(c["h"], c["w"], c["bias"], c["labels"], c["weight"], c["scale"], dtype)
    check_head(got, want)
    z = c["h"] @ c["w"].T + (0 if c["bias"] is None else c["bias"])
    second = np.sort(z, 1)[:, -2] if c["classes"] > 1 else np.full(c["n"], -np.inf)
    clear = z.max(1) - second > 2 * (c["dim"] + 4) * R.EPS32 * (np.abs(c["h"]) @ np.abs(c["w"].T) + 2).max(1)
    assert np.array_equal(got["best"][clear], want["best"][0][clear])
    again = run_head(c)
    assert all(np.array_equal(got[k], again[k]) for k in got)
    for k in got:  # each alone: the gradients' bits, and scores within their bounds
        alone = run_head(c, (k,))[k]
        if k in ("dh", "dw", "db"):
            assert np.array_equal(alone, got[k]), k
        elif k == "best":
            assert np.array_equal(alone[clear], got[k][clear])
        else:
            close(alone, want[k], k)


@pytest.mark.parametrize("dtype, n, classes", [("float32", 40_000, 5_000), ("bfloat16", 90_000, 6_200)])
def test_classes_taken_in_pieces(dtype, n, classes):
    """More pairs than are held at once: some rows' loss and gradient against
    all of their classes, and some classes' (the first and last of each piece
    among them) against all rows, whose lse the first check stands for."""
    c = head_case((n, classes, 130, 0.05, True, True, 0, 0), dtype, 9)
    got = run_head(c, ("loss", "lse", "dh", "dw", "db"))
    rows = np.r_[0:40, n // 2:n // 2 + 40, n - 40:n]
    part = dict(c, h=c["h"][rows])
    want = R.head(part["h"], c["w"], c["bias"], c["labels"][rows], c["weight"][rows], c["scale"], dtype)
    for k in ("loss", "lse", "dh"):
        close(got[k][rows], want[k], k)
    some = np.r_[0:20, classes // 2 - 160:classes // 2 + 160, classes - 20:classes]
    z = c["h"] @ c["w"][some].T + c["bias"][some]
    p = np.exp(z - got["lse"][:, None])
    live = c["labels"] >= 0
    g = np.where(live[:, None], c["scale"] * c["weight"][:, None] * (p - (c["labels"][:, None] == some[None, :])), 0.0)
    # a score's and the lse's bounds, and the pair's roundings, as in R.head
    size = np.abs(c["h"]) @ np.abs(c["w"][some].T) + np.abs(c["bias"][some])
    elz = want["lse"][1].max() * 2
    eg = c["scale"] * c["weight"][:, None] * p * ((c["dim"] + 4) * R.EPS32 * size + elz + (np.abs(z - got["lse"][:, None]) + 8) * R.EPS32)
    eg = np.where(live[:, None], eg, 0.0) + 2 * R.EPS32 * np.abs(g)
    close(got["db"][some], (g.sum(0), eg.sum(0) + (n + 1) * R.EPS32 * np.abs(g).sum(0)), "db")
    eg = eg + R.HALF[dtype] * np.abs(g)
    value, err = g.T @ c["h"], eg.T @ np.abs(c["h"])
    close(got["dw"][some], (value, err + (n + 4) * R.EPS32 * (np.abs(g).T @ np.abs(c["h"])) + R.HALF[dtype] * (np.abs(value) + err)), "dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, classes, dim", [(1, 5, 16), (1, 4099, 64), (7, 1000, 33), (16, 70_000, 24), (50, 257, 512)])
def test_rows_answered_without_labels(n, classes, dim, dtype):
    c = head_case((n, classes, dim, 0.0, False, True, 0, 0), dtype, 1)
    got = run_head(c, ("loss", "lse", "best"), labels=False)
    want = R.head(c["h"], c["w"], c["bias"], None, None, 1.0, dtype)
    check_head(got, want)
    z = c["h"] @ c["w"].T + c["bias"]
    assert np.all(z[np.arange(n), got["best"]] >= z.max(1) - 2 * (dim + 4) * R.EPS32 * (
        np.abs(c["h"]) @ np.abs(c["w"].T) + np.abs(c["bias"])).max(1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, classes, dim", [(4_100, 2_050, 24), (8_193, 1_030, 64), (130_000, 65, 33)])
def test_many_rows_of_short_inputs_scored_alone(n, classes, dim, dtype):
    """Without gradients, on a workspace that was named for them."""
    c = head_case((n, classes, dim, 0.1, True, True, 0, 0), dtype, 17)
    ws = work(hb.softmax_head_workspace(n, classes, dim, dtype))
    want = R.head(c["h"], c["w"], c["bias"], c["labels"], c["weight"], 1.0, dtype)
    check_head(run_head(c, ("loss", "lse"), workspace=ws), want)
    got = run_head(c, ("loss", "lse", "best"), labels=False, workspace=ws)
    check_head(got, R.head(c["h"], c["w"], c["bias"], None, None, 1.0, dtype))
    z = c["h"] @ c["w"].T + c["bias"]
    assert np.all(z[np.arange(n), got["best"]] >= z.max(1) - 2 * (dim + 4) * R.EPS32 * (
        np.abs(c["h"]) @ np.abs(c["w"].T) + np.abs(c["bias"])).max(1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, classes", [(70, 9), (5, 3000), (200, 700)])
def test_the_first_of_equal_classes_is_the_best(n, classes, dtype):
    """Every class alike, and a later pair above the others."""
    c = head_case((n, classes, 16, 0.0, False, False, 0, 0), dtype, 2)
    c["w"][:] = c["w"][0]
    assert np.all(run_head(c, ("best",), labels=False)["best"] == 0)
    c["bias"] = np.zeros(classes)
    c["bias"][[classes - 1, classes // 2]] = 3.0
    assert np.all(run_head(c, ("best",), labels=False)["best"] == classes // 2)


# few classes, tiles of products, short inputs (whose kernels give gradients alone)
WAYS = [(9, 24), (60, 24), (300, 24), (300, 136)]


def scored(values, n, dim, dtype):
    """A case whose scores are exactly the values, whatever the types: inputs of zeros."""
    classes = len(values)
    return dict(n=n, classes=classes, dim=dim, w=np.ones((classes, dim)), h=np.zeros((n, dim)),
                bias=np.asarray(values, np.float32).astype(np.float64), labels=np.zeros(n, np.int32), weight=None, gap=0,
                lead=0, dtype=dtype, scale=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes, dim", WAYS)
def test_the_best_class_has_the_largest_score_to_the_last_bit(classes, dim, dtype):
    """Scores one step of f32 apart, the larger one of the later class."""
    rng = np.random.default_rng(classes)
    for low in (1.4, 1.9, 0.7, 11.3, 22.9, -0.36, -1.42, -23.0, 1.2e7):
        low = np.float32(low)
        high = np.nextafter(low, np.float32(np.inf))
        values = np.full(classes, low - np.float32(abs(low)) / 2 - 1, np.float32)
        first, second = np.sort(rng.choice(classes, 2, replace=False))
        values[first], values[second] = low, high
        c = scored(values, 3, dim, dtype)
        for outputs in (("best",), ("best", "dh")):
            assert np.all(run_head(c, outputs, labels=len(outputs) > 1)["best"] == second), (low, outputs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes, dim", WAYS)
@pytest.mark.parametrize("far", [0.0, 5e4, -3e6])
def test_a_loss_is_made_of_differences_of_scores(far, classes, dim, dtype):
    """Of scores held exactly, a loss is off by the rounding of their
    differences, of the exponentials' sum and of its logarithm, however far
    from zero they lie: (gap + classes + 16) half steps for the logarithm of
    the sum, one of it and two of the loss. The exponentials are off by the
    rounding of their arguments, at most (gap + 3) half steps."""
    rng = np.random.default_rng(7)
    values = np.float32(far) + rng.integers(-24, 25, classes).astype(np.float32) / 4
    c = scored(values, 40, dim, dtype)
    c["labels"] = rng.integers(0, classes, 40).astype(np.int32)
    z = c["bias"]
    tail = np.log(np.exp(z - z.max()).sum())
    loss = z.max() - z[c["labels"]] + tail
    gap = z.max() - z.min()
    bound = (2 * gap + classes + 20 + 2 * tail + 2 * loss) * R.EPS32
    for outputs in (("loss",), ("loss", "dh")):
        close(run_head(c, outputs)["loss"], (loss, bound), outputs)
    answer = run_head(c, ("loss",), labels=False)["loss"]
    close(answer, (np.full(40, tail), (2 * gap + classes + 20 + 2 * tail) * R.EPS32), "answer")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, classes, dim", [(90, 12, 20), (90, 300, 64), (90, 300, 160), (1100, 300, 136)])
def test_shut_classes_and_rows_that_take_no_part(n, classes, dim, dtype):
    """Biases of -infinity; NaN, infinities and a NaN weight in rows whose
    label is below 0: the others' results are those without them."""
    c = head_case((n, classes, dim, 0.3, True, True, 0, 0), dtype, 3)
    c["bias"][::3] = -np.inf
    open_ = np.flatnonzero(np.isfinite(c["bias"]))
    live = c["labels"] >= 0
    c["labels"][live] = open_[c["labels"][live] % len(open_)]
    want = R.head(c["h"], c["w"], c["bias"], c["labels"], c["weight"], c["scale"], dtype)
    dead = np.flatnonzero(~live)
    c["h"][dead[0]] = np.nan
    c["h"][dead[1]] = np.inf
    c["h"][dead[2], 0] = -np.inf
    c["weight"][dead[3]] = np.nan
    got = run_head(c)
    assert not got["dh"][dead].any() and not got["loss"][dead].any()
    assert not got["dw"][::3].any() and not got["db"][::3].any()
    for k in ("loss", "dh", "lse"):
        close(got[k][live], (want[k][0][live], want[k][1][live]), k)
    for k in ("dw", "db"):
        close(got[k], want[k], k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes, dim", WAYS + [(300, 33)])
def test_rows_that_take_no_part_keep_their_lse_and_reach_no_gradient(classes, dim, dtype):
    """Finite inputs of any size in rows whose label is below 0: their lse is
    that of any row, and scores past f32's range reach no gradient."""
    c = head_case((90, classes, dim, 0.3, True, True, 0, 0), dtype, 16)
    live = c["labels"] >= 0
    dead = np.flatnonzero(~live)
    c["h"][dead[0]] = R.rounded(c["h"][dead[0]] * 1e17, dtype)
    want = R.head(c["h"], c["w"], c["bias"], c["labels"], c["weight"], c["scale"], dtype)
    close(run_head(c, ("lse", "dw"))["lse"], want["lse"], "lse")
    c["h"][dead[1]] = R.rounded(np.where(c["h"][dead[1]] < 0, -3e38, 3e38), dtype)
    c["w"][:, 2] = R.rounded(c["w"][:, 2] * 64, dtype)
    c["h"][live, 2] = 0.0
    want = R.head(np.where(live[:, None], c["h"], 0.0), c["w"], c["bias"], c["labels"], c["weight"], c["scale"], dtype)
    got = run_head(c, ("loss", "dh", "dw", "db"))
    assert not got["dh"][dead].any() and not got["loss"][dead].any()
    for k in ("dw", "db"):
        close(got[k], want[k], k)
    for k in ("loss", "dh"):
        close(got[k][live], (want[k][0][live], want[k][1][live]), k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes, dim", WAYS)
def test_infinite_inputs_give_infinite_scores(classes, dim, dtype):
    """An infinity in a class's weights, against inputs of one sign there:
    a score of -infinity, which shuts the class as its bias does."""
    c = head_case((70, classes, dim, 0.2, True, True, 0, 0), dtype, 14)
    c["h"][:, 5] = R.rounded(np.abs(c["h"][:, 5]) + 0.25, dtype)
    c["labels"] = np.where(c["labels"] >= 0, 1 + c["labels"] % (classes - 2), c["labels"]).astype(np.int32)
    shut = dict(c, w=c["w"].copy(), bias=c["bias"].copy())
    c["w"][0, 5] = c["w"][classes - 1, 5] = -np.inf
    shut["w"][[0, classes - 1]] = 0.0
    shut["bias"][[0, classes - 1]] = -np.inf
    want = R.head(shut["h"], shut["w"], shut["bias"], c["labels"], c["weight"], c["scale"], dtype)
    for outputs in (("loss", "lse"), ("loss", "lse", "dw", "db")):
        check_head(run_head(c, outputs), want)
    # and in an input: every score infinite, of its weight's sign
    c = head_case((70, classes, dim, 0.0, False, True, 0, 0), dtype, 15)
    c["w"][:, 3] = R.rounded(-np.abs(c["w"][:, 3]) - 0.25, dtype)
    c["h"][7, 3] = np.inf
    lse = run_head(c, ("lse",))["lse"]
    assert np.isneginf(lse[7]) and np.isfinite(np.delete(lse, 7)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes, dim", [(6, 24), (200, 24), (200, 160)])
def test_a_label_in_a_shut_class_has_an_infinite_loss(classes, dim, dtype):
    c = head_case((40, classes, dim, 0.0, False, True, 0, 0), dtype, 4)
    c["bias"][0] = -np.inf
    c["labels"][:] = np.maximum(c["labels"], 1)
    c["labels"][3] = 0
    got = run_head(c)
    assert np.isposinf(got["loss"][3]) and np.isfinite(np.delete(got["loss"], 3)).all()
    want = R.head(c["h"], c["w"], c["bias"], c["labels"], None, c["scale"], dtype)
    for k in ("dh", "dw", "db"):
        close(got[k], want[k], k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes, dim", [(4, 8), (130, 8), (130, 136)])
def test_rows_with_no_open_class_and_labels_that_are_no_class(classes, dim, dtype):
    c = head_case((30, classes, dim, 0.0, False, True, 0, 0), dtype, 5)
    shut = dict(c, bias=np.full(classes, -np.inf))
    got = run_head(shut, ("loss", "lse"))
    assert np.all(np.isneginf(got["lse"])) and np.all(np.isnan(got["loss"]))
    shut["labels"] = np.full(30, -1, np.int32)
    got = run_head(shut)
    assert not got["loss"].any() and not got["dh"].any() and not got["dw"].any() and not got["db"].any()
    c["labels"][4] = classes
    got = run_head(c)
    assert np.isnan(got["loss"][4]) and np.isnan(got["lse"][4]) and np.isnan(got["dh"][4]).all()
    assert np.isfinite(np.delete(got["loss"], 4)).all() and np.isnan(got["dw"]).all()


@pytest.mark.parametrize("classes", [5, 150])
def test_scores_far_from_zero_keep_their_loss(classes):
    """Scores of thousands: exponentials are taken of differences alone."""
    c = head_case((50, classes, 16, 0.0, False, True, 0, 0), "float32", 6)
    c["h"] = R.rounded(c["h"] * 1000, "float32")
    c["bias"] = R.rounded(c["bias"] - 5e4, "float32")
    got = run_head(c)
    check_head(got, R.head(c["h"], c["w"], c["bias"], c["labels"], None, c["scale"], "float32"))


@pytest.mark.parametrize("n, classes, dim", [(6, 5, 8), (20, 150, 12), (20, 150, 132)])
def test_head_gradients_are_the_differences_of_the_loss(n, classes, dim):
    """A central difference along a direction in h, w and bias at once. With
    step e the difference is off by e^2/6 times the loss's third derivative
    (a third moment of the scores' slopes u_k and, through the product of
    the two moving factors, of their bends) and by the loss's bound over e."""
    c = head_case((n, classes, dim, 0.0, True, True, 0, 0), "float32", 7)
    rng = np.random.default_rng(8)
    e = 2.0 ** -7
    g = run_head(c, ("dh", "dw", "db"))
    total, slack, moved = [], 0.0, []
    sides = []
    dh, dw, db = (rng.standard_normal(c[k].shape) for k in ("h", "w", "bias"))
    for sign in (1, -1):
        s = dict(c, h=R.rounded(c["h"] + sign * e * dh, "float32"), w=R.rounded(c["w"] + sign * e * dw, "float32"),
                 bias=R.rounded(c["bias"] + sign * e * db, "float32"))
        loss = run_head(s, ("loss",))["loss"]
        want = R.head(s["h"], s["w"], s["bias"], s["labels"], s["weight"], 1.0, "float32")["loss"]
        total.append(loss.sum())
        slack += want[1].sum()
        sides.append(s)
    moved = {k: sides[0][k] - sides[1][k] for k in ("h", "w", "bias")}
    slope = np.sum(g["dh"] * moved["h"]) + np.sum(g["dw"] * moved["w"]) + np.sum(g["db"] * moved["bias"])
    # z(t) = z + t u + t^2 v: the third derivative of lse is the third central
    # moment of u plus three times the covariance of u and 2 v
    u = dh @ c["w"].T + c["h"] @ dw.T + db
    v = dh @ dw.T
    span_u = np.ptp(np.abs(u) + 2 * e * np.abs(v), axis=1) + 2 * (np.abs(u) + 2 * e * np.abs(v)).max(1)
    span_v = 2 * np.abs(2 * v).max(1)
    third = span_u ** 3 + 3 * span_u * span_v
    slack += np.sum(c["weight"] * third) * e ** 3 / 3
    want = R.head(c["h"], c["w"], c["bias"], c["labels"], c["weight"], c["scale"], "float32")
    slack += sum(np.sum(want[k][1] * np.abs(moved[m])) for k, m in (("dh", "h"), ("dw", "w"), ("db", "bias"))) / c["scale"]
    slack += 1e-12 * abs(total[0]) + 1e-5 * e  # the sides' own rounding of the step
    assert abs((total[0] - total[1]) - slope / c["scale"]) <= slack


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride", [0, 3, 1 << 40])
def test_the_stride_of_a_single_row_counts_nothing(stride, dtype):
    """A record of one row, or of one class or table row, may hold any stride
    there: the results are those of its own length."""
    L = A.lib()
    for classes, dim in ((1, 24), (9, 128), (70, 128), (200, 128), (200, 500), (200, 40)):
        c = head_case((1, classes, dim, 0.0, True, True, 0, 0), dtype, 12)
        want = run_head(c)
        out = {k: like((1,), "float32" if k != "best" else "int32") for k in ("loss", "lse", "best")}
        out.update(dh=like((1, dim), dtype), dw=like((classes, dim), dtype), db=like((classes,), "float32"))
        held = {k: dev(c[k], t) for k, t in (("h", dtype), ("w", dtype), ("bias", "float32"), ("labels", "int32"),
                                             ("weight", "float32"))}
        ws = work(hb.softmax_head_workspace(1, classes, dim, dtype))
        one = stride if classes == 1 else dim
        p = A.Softmax(A.F32 if dtype == "float32" else A.BF16, dim, 1, classes, c["scale"], stride, one, stride, one,
                      *(held[k].data_ptr() for k in ("h", "w", "bias", "labels", "weight")),
                      *(out[k].data_ptr() for k in ("loss", "lse", "best", "dh", "dw", "db")))
        A.check(L.hbr_softmax_head(0, C.byref(p), ws.data_ptr(), ws.shape[0], None))
        for k, v in out.items():
            assert np.array_equal(back(v), want[k]), (classes, dim, k)
    rng = np.random.default_rng(13)
    table, dim = R.rounded(rng.standard_normal((1, 40)), dtype), 40
    ids, out, dtable = dev(np.zeros((1, 3)), "int32"), like((1, dim), dtype), like((1, dim), dtype)
    ws = work(hb.leaf_embedding_grad_workspace(1, 3, 1, dim, dtype))
    p = A.Lookup(A.F32 if dtype == "float32" else A.BF16, dim, 1, 3, 0, 1, stride, stride, stride, ids.data_ptr(), None, None)
    A.check(L.hbr_leaf_embedding(0, C.byref(p), dev(table, dtype).data_ptr(), out.data_ptr(), None))
    A.check(L.hbr_leaf_embedding_grad(0, C.byref(p), dev(table, dtype).data_ptr(), dtable.data_ptr(), ws.data_ptr(), ws.shape[0], None))
    one = R.embedding(table, np.zeros((1, 3), np.int32), None, None, dtype)
    close(back(out), one)
    close(back(dtable), one)


# ---- arrays of more than 4 GiB ----------------------------------------------------------

FAR = 9 << 30


def upload(address, values):
    A.check(A.lib().hbr_device_upload(0, C.c_void_p(address), A.ptr(values), values.nbytes))


def far(rows, cols, dtype, stride, values=None):
    """An array whose rows lie `stride` elements apart over more than 4 GiB,
    with nothing known between them."""
    size = 2 if dtype == "bfloat16" else 4
    assert FAR > (rows - 1) * stride * size > 1 << 32
    a = DeviceArray(hb.DeviceBuffer(FAR), dtype, (rows, cols), stride=stride)
    if values is not None:
        bits = R.to_bf16(values) if dtype == "bfloat16" else np.ascontiguousarray(values, np.float32)
        for r in range(rows):
            upload(a.data_ptr() + r * stride * size, bits[r])
    return a


def far_back(a):
    size, (rows, cols) = (2 if a.dtype == "bfloat16" else 4), a.shape
    bits = np.empty((rows, cols), _BITS[a.dtype])
    for r in range(rows):
        A.check(A.lib().hbr_device_download(0, A.ptr(bits[r]), C.c_void_p(a.data_ptr() + r * a.stride()[0] * size), cols * size))
    return (R.from_bf16(bits) if a.dtype == "bfloat16" else bits.view(np.float32)).astype(np.float64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 37])
def test_lookups_over_more_than_4_gib(dim, dtype):
    rng = np.random.default_rng(dim)
    rows, columns, n = 8, 3, 500
    gap = (1 << 30) // (2 if dtype == "bfloat16" else 4) + 16
    table = R.rounded(rng.standard_normal((rows, dim)), dtype)
    ids = rng.integers(-1, rows + 1, (n, columns)).astype(np.int32)
    out = like((n, dim), dtype)
    hb.leaf_embedding(far(rows, dim, dtype, gap, table), dev(ids, "int32"), out)
    close(back(out), R.embedding(table, ids, None, None, dtype), "the table far")
    out = far(rows, dim, dtype, gap)
    hb.leaf_embedding(dev(table, dtype), dev(ids[:rows], "int32"), out)
    close(far_back(out), R.embedding(table, ids[:rows], None, None, dtype), "the vectors far")
    dout = R.rounded(rng.standard_normal((n, dim)), dtype)
    for t, what in ((columns, "the gradient far, by sorting"), (1, "by column")):
        mine, dtable = ids[:, :t].copy(), far(rows, dim, dtype, gap)
        hb.leaf_embedding_grad(dev(dout, dtype), dev(mine, "int32"), dtable,
                               workspace=work(hb.leaf_embedding_grad_workspace(n, t, rows, dim, dtype)))
        close(far_back(dtable), R.embedding_grad(dout, mine, None, None, rows, dtype), what)
    dtable = like((rows, dim), dtype)
    hb.leaf_embedding_grad(far(rows, dim, dtype, gap, dout[:rows]), dev(ids[:rows], "int32"), dtable,
                           workspace=work(hb.leaf_embedding_grad_workspace(rows, columns, rows, dim, dtype)))
    close(back(dtable), R.embedding_grad(dout[:rows], ids[:rows], None, None, rows, dtype), "the rows far")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, classes, dim", [(1100, 20, 24), (1100, 70, 24), (1100, 70, 136), (9, 1100, 136), (70, 1100, 40)])
def test_a_head_over_more_than_4_gib(n, classes, dim, dtype):
    """The longer side's rows, and their gradients, near the largest stride."""
    c = head_case((n, classes, dim, 0.1, True, True, 0, 0), dtype, 5)
    gap = (1 << 21) - 8
    rows = max(n, classes)
    by_rows = n == rows
    x, y = (c["h"], c["w"]) if by_rows else (c["w"], c["h"])
    x, dx = far(rows, dim, dtype, gap, x), far(rows, dim, dtype, gap)
    y, dy = dev(y, dtype), like(y.shape, dtype)
    h, w, dh, dw = (x, y, dx, dy) if by_rows else (y, x, dy, dx)
    lse = like((n,), "float32")
    hb.softmax_head(h, w, bias=dev(c["bias"], "float32"), labels=dev(c["labels"], "int32"),
                    weight=dev(c["weight"], "float32"), grad_scale=c["scale"], lse=lse, dh=dh, dw=dw,
                    workspace=work(hb.softmax_head_workspace(n, classes, dim, dtype)))
    want = R.head(c["h"], c["w"], c["bias"], c["labels"], c["weight"], c["scale"], dtype)
    close(back(lse), want["lse"], "lse")
    close(far_back(dx), want["dh" if by_rows else "dw"], "the far gradient")
    close(back(dy), want["dw" if by_rows else "dh"], "the near gradient")


def test_clipping_a_tensor_of_more_than_4_gib():
    n = (1 << 30) + 1027
    buf, out = hb.DeviceBuffer(4 * n), hb.DeviceBuffer(4 * n)
    g, to = DeviceArray(buf, "float32", n), DeviceArray(out, "float32", n)
    # zeros: the gradient of a table that no id leads to
    hb.leaf_embedding_grad(dev(np.zeros((1, 1027)), "float32"), dev(np.full((1, 1), -1), "int32"),
                           DeviceArray(buf, "float32", (n // 1027, 1027)),
                           workspace=work(hb.leaf_embedding_grad_workspace(1, 1, n // 1027, 1027, "float32")))
    at, held = [0, 5, 1 << 29, (1 << 30) - 1, 1 << 30, n - 1], np.float32([3, -1, 2, 5, -4, 6])
    tail = n // 1027 * 1027
    upload(g.data_ptr() + 4 * tail, np.zeros(n - tail, np.float32))
    for i, v in zip(at, held):
        upload(g.data_ptr() + 4 * i, np.float32([v]))
    norm = like((1,), "float32")
    hb.clip_gradients([g], 0.5, norm=norm, out=[to], workspace=work(hb.clip_gradients_workspace(1)))
    true = np.sqrt(np.sum(held.astype(np.float64) ** 2))
    assert abs(back(norm)[0] - true) <= R.EPS32 * true
    one = np.empty(1, np.float32)
    for i, v in zip(at, held):
        A.check(A.lib().hbr_device_download(0, A.ptr(one), C.c_void_p(to.data_ptr() + 4 * i), 4))
        # the factor's and the product's roundings
        assert abs(one[0] - v * 0.5 / (true + 1e-6)) <= 2.01 * R.EPS32 * abs(v)
    A.check(A.lib().hbr_device_download(0, A.ptr(one), C.c_void_p(to.data_ptr() + 4 * (n - 2)), 4))
    assert one[0] == 0.0


# ---- clipping ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [0], [], [7, 0, 8192, 8193], [5] * 97, [100_003, 3, 16_384 * 3 + 5],
                                   [1] * 300 + [5_000_001]])
def test_clipping_scales_a_set_to_its_largest_norm(sizes, dtype):
    rng = np.random.default_rng(len(sizes))
    grads = [R.rounded(rng.standard_normal(s), dtype) for s in sizes]
    true = np.sqrt(sum(float(np.sum(g * g)) for g in grads))
    for most in (0.0, 0.25 * true, 4.0 * true + 1.0, np.inf):
        arrays = [dev(g, dtype, lead=i % 3) for i, g in enumerate(grads)]
        outs = [like(g.shape, dtype, lead=(i // 2) % 3) for i, g in enumerate(grads)]
        norm = like((1,), "float32")
        kw = dict(norm=norm, workspace=work(hb.clip_gradients_workspace(len(grads))))
        hb.clip_gradients(arrays, most, out=outs, **kw)
        # f64 sums, one rounding of the norm
        assert abs(back(norm)[0] - true) <= true * (2 * R.EPS32)
        by = min(1.0, most / (true + 1e-6))
        for g, o, a in zip(grads, outs, arrays):
            want = g * by
            close(back(o), (want, (4 * R.EPS32 + R.HALF[dtype]) * np.abs(want) + 1e-38))
            assert np.array_equal(back(a), g)
        hb.clip_gradients(arrays, most, **kw)  # in place
        for o, a in zip(outs, arrays):
            assert np.array_equal(back(o), back(a))


def test_clipping_of_mixed_types_and_huge_values():
    a, b = np.array([1e30, -3e38], np.float32).astype(np.float64), R.rounded(np.array([2e38, 1.0]), "bfloat16")
    x, y, norm = dev(a, "float32"), dev(b, "bfloat16"), like((1,), "float32")
    w = work(hb.clip_gradients_workspace(2))
    hb.clip_gradients([x, y], 1.0, norm=norm, workspace=w)
    # the norm is past f32's range, the factor is not
    true = np.sqrt(np.sum(a * a) + np.sum(b * b))
    assert np.isposinf(back(norm)[0])
    # each factor is a denormal f32 here: half its smallest step
    close(back(x), (a / true, np.abs(a) * (2.0 ** -150 + 4 * R.EPS32 / true)))
    close(back(y), (b / true, np.abs(b) * (2.0 ** -150 + 4 * R.EPS32 / true) + R.HALF["bfloat16"] * np.abs(b / true) + 1e-40))


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_norm_that_is_none_shows_in_every_tensor(bad):
    x, y, norm = dev(np.array([1.0, bad]), "float32"), dev(np.ones(5), "float32"), like((1,), "float32")
    hb.clip_gradients([x, y], 1.0, norm=norm, workspace=work(hb.clip_gradients_workspace(2)))
    if np.isnan(bad):
        assert np.isnan(back(norm)[0]) and np.isnan(back(x)).all() and np.isnan(back(y)).all()
    else:  # 1 / infinity: zeros, and infinity times zero
        assert np.isposinf(back(norm)[0]) and not back(y).any() and back(x)[0] == 0 and np.isnan(back(x)[1])


# ---- together, on streams and in graphs ---------------------------------------------------------

class Step:
    """One training step of a model on leaves: look-up, head, gradients, clip."""

    def __init__(self, dtype, seed, n=700, columns=12, rows=31, dim=40, classes=130):
        rng = np.random.default_rng(seed)
        self.dtype, self.n, self.dim, self.classes, self.rows = dtype, n, dim, classes, rows * columns
        self.ids_v = rng.integers(0, rows, (n, columns)).astype(np.int32)
        self.off_v = (np.arange(columns) * rows).astype(np.int32)
        self.s_v = R.rounded(rng.random(columns) + 0.5, "float32")
        self.table_v = R.rounded(rng.standard_normal((self.rows, dim)) * 0.3, dtype)
        self.w_v = R.rounded(rng.standard_normal((classes, dim)) * 0.2, dtype)
        self.b_v = R.rounded(rng.standard_normal(classes) * 0.1, "float32")
        self.y_v = rng.integers(-1, classes, n).astype(np.int32)
        self.ids, self.off, self.s = dev(self.ids_v, "int32"), dev(self.off_v, "int32"), dev(self.s_v, "float32")
        self.table, self.w, self.b = dev(self.table_v, dtype), dev(self.w_v, dtype), dev(self.b_v, "float32")
        self.y = dev(self.y_v, "int32")
        self.h, self.dh = like((n, dim), dtype), like((n, dim), dtype)
        self.loss, self.norm = like((n,), "float32"), like((1,), "float32")
        self.grads = [like((self.rows, dim), dtype), like((classes, dim), dtype), like((classes,), "float32")]
        self.ws = [work(b) for b in (hb.softmax_head_workspace(n, classes, dim, dtype),
                                     hb.leaf_embedding_grad_workspace(n, columns, self.rows, dim, dtype),
                                     hb.clip_gradients_workspace(3))]

    def run(self, stream=None):
        kw = dict(offset=self.off, scale=self.s, stream=stream)
        hb.leaf_embedding(self.table, self.ids, self.h, **kw)
        hb.softmax_head(self.h, self.w, bias=self.b, labels=self.y, loss=self.loss, dh=self.dh, dw=self.grads[1],
                        db=self.grads[2], grad_scale=1.0 / self.n, workspace=self.ws[0], stream=stream)
        hb.leaf_embedding_grad(self.dh, self.ids, self.grads[0], workspace=self.ws[1], **kw)
        hb.clip_gradients(self.grads, 0.01, norm=self.norm, workspace=self.ws[2], stream=stream)

    def outputs(self):
        return [back(a) for a in (self.h, self.loss, self.norm, *self.grads)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_training_step_runs_through_all_of_them(dtype):
    s = Step(dtype, 11)
    s.run()
    h, loss, norm, *grads = s.outputs()
    close(h, R.embedding(s.table_v, s.ids_v, s.off_v, s.s_v, dtype))
    want = R.head(h, s.w_v, s.b_v, s.y_v, None, float(np.float32(1 / s.n)), dtype)
    close(loss, want["loss"])
    dh = back(s.dh)
    close(dh, want["dh"])
    full = [R.embedding_grad(dh, s.ids_v, s.off_v, s.s_v, s.rows, dtype), want["dw"], want["db"]]
    true = np.sqrt(sum(np.sum(v * v) for v, _ in full))
    slack = np.sqrt(sum(np.sum(e * e) for _, e in full))
    assert abs(norm[0] - true) <= slack + 2 * R.EPS32 * true and true > 0.01
    by = 0.01 / (true + 1e-6)
    for g, (v, e), t in zip(grads, full, (dtype, dtype, "float32")):
        close(g, (v * by, (e + np.abs(v) * (slack / true + 6 * R.EPS32)) * by * 1.01 + R.HALF[t] * 1.01 * (np.abs(v) + e) * by + 1e-38))


def hip():
    L = C.CDLL("libamdhip64.so.7")
    for name in ("hipStreamCreateWithFlags", "hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate",
                 "hipGraphLaunch", "hipStreamSynchronize", "hipDeviceSynchronize", "hipGetDevice", "hipStreamDestroy",
                 "hipGraphExecDestroy", "hipGraphDestroy"):
        getattr(L, name).restype = C.c_int
    return L


def ok(status):
    assert status == 0, f"HIP error {status}"


def test_steps_on_several_streams_give_the_same_bits():
    L = hip()
    steps = [Step("bfloat16", 21), Step("bfloat16", 22), Step("float32", 23)]
    want = []
    for s in steps:
        s.run()
        want.append(s.outputs())
    streams = []
    for _ in steps:
        st = C.c_void_p()
        ok(L.hipStreamCreateWithFlags(C.byref(st), 1))
        streams.append(st)
    again = [Step("bfloat16", 21), Step("bfloat16", 22), Step("float32", 23)]
    for _ in range(3):
        for s, st in zip(again, streams):
            s.run(st.value)
    ok(L.hipDeviceSynchronize())
    for s, w in zip(again, want):
        for a, b in zip(s.outputs(), w):
            assert np.array_equal(a, b)
    for st in streams:
        ok(L.hipStreamDestroy(st))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step_replays_with_the_eager_bits(dtype):
    """Captured once; replayed on other inputs with eager work between."""
    L = hip()
    st = C.c_void_p()
    ok(L.hipStreamCreateWithFlags(C.byref(st), 1))
    s = Step(dtype, 31)
    other = Step(dtype, 32)
    other.run()
    ok(L.hipStreamBeginCapture(st, 2))
    s.run(st.value)
    graph, run = C.c_void_p(), C.c_void_p()
    ok(L.hipStreamEndCapture(st, C.byref(graph)))
    ok(L.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
    for seed in (31, 41, 42, 31):
        t = Step(dtype, seed)
        for mine, its in ((s.ids, t.ids), (s.table, t.table), (s.w, t.w), (s.b, t.b), (s.y, t.y), (s.s, t.s)):
            mine.buffer.copy_from(its.buffer)
        ok(L.hipDeviceSynchronize())
        ok(L.hipGraphLaunch(run, st))
        ok(L.hipStreamSynchronize(st))
        got = s.outputs()
        t.run()
        for a, b in zip(got, t.outputs()):
            assert np.array_equal(a, b)
        other.run()
    ok(L.hipGraphExecDestroy(run))
    ok(L.hipGraphDestroy(graph))
    ok(L.hipStreamDestroy(st))


def test_a_stream_of_no_such_device_is_invalid():
    s = Step("float32", 1, n=5)
    p = A.Lookup(A.F32, 4, 1, 1, 0, 1, 4, 1, 4, s.ids.data_ptr(), None, None)
    n = C.c_int()
    A.check(A.lib().hbr_device_count(C.byref(n)))
    assert A.lib().hbr_leaf_embedding(n.value, C.byref(p), s.table.data_ptr(), s.h.data_ptr(), None) == A.INVALID


TORCH = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import numpy as np
import torch
import hessboost_amd as hb
import leaf_reference as R

torch.manual_seed(0)
n, t, rows, dim, classes = 500, 6, 15, 48, 300
for dtype, name in ((torch.float32, "float32"), (torch.bfloat16, "bfloat16")):
    table = torch.randn(rows * t, dim, device="cuda").to(dtype)
    ids = torch.randint(0, rows, (n, t), device="cuda", dtype=torch.int32)
    off = (torch.arange(t, device="cuda") * rows).int()
    w = torch.randn(classes, dim, device="cuda").mul_(0.2).to(dtype)
    y = torch.randint(-1, classes, (n,), device="cuda", dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the tensors' stream by default: torch's current one
        wide = torch.full((n, 2 * dim), float("nan"), device="cuda", dtype=dtype)
        h = wide[:, :dim]
        hb.leaf_embedding(table, ids, h, offset=off)
        loss = torch.empty(n, device="cuda")
        dh, dw = torch.empty(n, dim, device="cuda", dtype=dtype), torch.empty_like(w)
        ws = torch.empty(hb.softmax_head_workspace(n, classes, dim, dtype), dtype=torch.uint8, device="cuda")
        hb.softmax_head(h, w, labels=y, loss=loss, dh=dh, dw=dw, grad_scale=0.5, workspace=ws)
        dt = torch.empty_like(table)
        ws = torch.empty(hb.leaf_embedding_grad_workspace(n, t, rows * t, dim, dtype), dtype=torch.uint8, device="cuda")
        hb.leaf_embedding_grad(dh, ids, dt, offset=off, workspace=ws)
        norm = torch.empty(1, device="cuda")
        ws = torch.empty(hb.clip_gradients_workspace(2), dtype=torch.uint8, device="cuda")
        clipped = [torch.empty_like(dt), torch.empty_like(dw)]
        hb.clip_gradients([dt, dw], 1.0, norm=norm, out=clipped, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    v = lambda x: x.detach().cpu().double().numpy()
    assert torch.isnan(wide[:, dim:]).all()

    def close(got, want):
        assert np.all(np.abs(v(got) - want[0]) <= want[1])
    close(h, R.embedding(v(table), ids.cpu().numpy(), off.cpu().numpy(), None, name))
    want = R.head(v(h), v(w), None, y.cpu().numpy(), None, 0.5, name)
    close(loss, want["loss"]); close(dh, want["dh"]); close(dw, want["dw"])
    close(dt, R.embedding_grad(v(dh), ids.cpu().numpy(), off.cpu().numpy(), None, rows * t, name))
    true = np.sqrt(np.sum(v(dt) ** 2) + np.sum(v(dw) ** 2))
    assert abs(v(norm)[0] - true) <= 2 * R.EPS32 * true and true > 1
    for a, b in zip(clipped, (dt, dw)):
        close(a, (v(b) / (true + 1e-6), (R.HALF[name] + 4 * R.EPS32) * np.abs(v(b)) / true))
for bad in (lambda: hb.leaf_embedding(table.cpu(), ids, h, offset=off),
            lambda: hb.leaf_embedding(table.half(), ids, h, offset=off),
            lambda: hb.leaf_embedding(table, ids.long(), h, offset=off),
            lambda: hb.leaf_embedding(table.t(), ids, h, offset=off)):
    try:
        bad()
    except ValueError:
        continue
    raise AssertionError("not refused")
print("torch ok", flush=True)
"""


CAPTURED = """
import sys, threading
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import hessboost_amd as hb


class Step:
    def __init__(self, seed, dtype, n, t, rows, dim, classes):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g, device="cuda")
        self.table, self.w, self.b = r(rows * t, dim).to(dtype), r(classes, dim).mul_(0.2).to(dtype), r(classes)
        self.ids = torch.randint(0, rows, (n, t), generator=g, device="cuda", dtype=torch.int32)
        self.y = torch.randint(-1, classes, (n,), generator=g, device="cuda", dtype=torch.int32)
        self.off = (torch.arange(t, device="cuda") * rows).int() if t > 1 else None
        self.h, self.dh, self.dt, self.dw = (torch.empty_like(x) for x in (r(n, dim).to(dtype), r(n, dim).to(dtype), self.table, self.w))
        self.db, self.loss, self.norm = torch.empty(classes, device="cuda"), torch.empty(n, device="cuda"), torch.empty(1, device="cuda")
        self.best = torch.empty(n, dtype=torch.int32, device="cuda")
        self.ws = [torch.empty(max(16, b), dtype=torch.uint8, device="cuda") for b in (
            hb.softmax_head_workspace(n, classes, dim, dtype), hb.leaf_embedding_grad_workspace(n, t, rows * t, dim, dtype),
            hb.clip_gradients_workspace(3))]

    def run(self):
        hb.leaf_embedding(self.table, self.ids, self.h, offset=self.off)
        hb.softmax_head(self.h, self.w, bias=self.b, labels=self.y, loss=self.loss, dh=self.dh, dw=self.dw, db=self.db,
                        grad_scale=0.5, workspace=self.ws[0])
        hb.leaf_embedding_grad(self.dh, self.ids, self.dt, offset=self.off, workspace=self.ws[1])
        hb.clip_gradients([self.dt, self.dw, self.db], 1.0, norm=self.norm, workspace=self.ws[2])
        hb.softmax_head(self.h, self.w, bias=self.b, best=self.best, workspace=self.ws[0])

    def outputs(self):
        torch.cuda.synchronize()
        return [x.clone() for x in (self.h, self.loss, self.dh, self.dt, self.dw, self.db, self.norm, self.best)]


SIZES = [(torch.float32, 300, 5, 15, 24, 9), (torch.bfloat16, 500, 7, 31, 40, 60), (torch.float32, 900, 3, 63, 48, 300),
         (torch.bfloat16, 700, 4, 31, 136, 200), (torch.float32, 400, 1, 3000, 200, 90), (torch.bfloat16, 1500, 1, 50000, 64, 2000)]
# a first call of any operator; the steps' own kernels are met first in their captures
one = torch.zeros(1, 4, device="cuda")
hb.leaf_embedding(one, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.empty(1, 4, device="cuda"))
graphs = []
for k, size in enumerate(SIZES):
    s = Step(k, *size)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    graphs.append((s, graph))
for turn in range(3):
    for k, ((s, graph), size) in enumerate(zip(graphs, SIZES)):
        t = Step(100 * turn + k, *size)
        for mine, its in ((s.table, t.table), (s.w, t.w), (s.b, t.b), (s.ids, t.ids), (s.y, t.y)):
            mine.copy_(its)
        graph.replay()
        got = s.outputs()
        t.run()
        assert all(torch.equal(a, b) for a, b in zip(got, t.outputs())), (turn, k)
    print("replayed", turn, flush=True)
# several threads at once, each on a stream of its own
steps = [Step(k, *size) for k, size in enumerate(SIZES)]
again = [Step(k, *size) for k, size in enumerate(SIZES)]
for s in steps:
    s.run()
want = [s.outputs() for s in steps]
streams, failed = [torch.cuda.Stream() for _ in again], []


def work(s, stream):
    try:
        with torch.cuda.stream(stream):
            for _ in range(20):
                s.run()
    except Exception as e:
        failed.append(e)


threads = [threading.Thread(target=work, args=a) for a in zip(again, streams)]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert not failed, failed
for s, w in zip(again, want):
    assert all(torch.equal(a, b) for a, b in zip(s.outputs(), w))
print("captured ok", flush=True)
"""


def test_torch_graphs_and_threads_give_the_eager_bits():
    """Steps of several sizes captured by torch, the first of their kernels'
    calls, and several threads on streams of their own."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = CAPTURED.replace("{root!r}", repr(os.path.dirname(here))).replace("{tests!r}", repr(here))
    r = subprocess.run([sys.executable, "-u", "-c", code], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "captured ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_torch_tensors_are_taken_on_their_stream():
    """In a process of its own: torch brings its own HIP runtime."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = TORCH.format(root=os.path.dirname(here), tests=here)
    r = subprocess.run([sys.executable, "-u", "-c", code], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "torch ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
