"""The operators over leaves and many classes refuse what they cannot run,
before they touch a device."""
import ctypes as C

import numpy as np
import pytest

import hessboost_amd as hb
from hessboost_amd import _capi as A
from hessboost_amd.leafops import DeviceArray


class Memory:
    """Stands for a DeviceBuffer: an address that nothing reads."""

    def __init__(self, nbytes=1 << 20, ptr=1 << 20, ordinal=0):
        self.ptr, self.nbytes, self.ordinal = ptr, nbytes, ordinal


def arr(dtype, *shape, **kw):
    mem = {k: kw.pop(k) for k in ("ptr", "ordinal") if k in kw}
    return DeviceArray(Memory(**mem), dtype, shape, **kw)


def lookup(**kw):
    p = dict(dtype=A.F32, dim=4, n_rows=3, n_columns=2, pad=0, table_rows=5, table_stride=4, ids_stride=2, out_stride=4,
             ids=1 << 20, offset=None, scale=None)
    p.update(kw)
    return A.Lookup(**p)


@pytest.mark.parametrize("bad, said", [
    (dict(dtype=7), "type"), (dict(dim=0), "no elements"), (dict(ids=None), "null ids"),
    (dict(ids_stride=1), "overlap"), (dict(table_stride=3), "overlap"), (dict(out_stride=3), "overlap"),
    (dict(ids=(1 << 20) + 2), "aligned"), (dict(scale=(1 << 20) + 1), "aligned")])
def test_lookups_with_malformed_records_are_invalid(bad, said):
    p, n = lookup(**bad), C.c_uint64()
    ok = 1 << 20
    assert A.lib().hbr_leaf_embedding(0, C.byref(p), ok, ok, None) == A.INVALID and said in A.last_error()
    assert A.lib().hbr_leaf_embedding_grad(0, C.byref(p), ok, ok, ok, ok, None) == A.INVALID and said in A.last_error()
    # the workspace's size is one of the sizes alone
    arrays = set(bad) <= {"ids", "offset", "scale"}
    assert A.lib().hbr_leaf_embedding_grad_workspace(C.byref(p), C.byref(n)) == (A.OK if arrays else A.INVALID)


def test_lookups_of_null_and_misaligned_arrays_are_invalid():
    p, ok = lookup(), 1 << 20
    L = A.lib()
    assert L.hbr_leaf_embedding(0, None, ok, ok, None) == A.INVALID
    for t, o in ((None, ok), (ok, None), (ok + 1, ok), (ok, ok + 2)):
        assert L.hbr_leaf_embedding(0, C.byref(p), t, o, None) == A.INVALID
        assert L.hbr_leaf_embedding_grad(0, C.byref(p), t, o, ok, 1 << 30, None) == A.INVALID


def test_lookups_past_the_index_range_are_refused():
    n = C.c_uint64()
    for big in (dict(table_rows=1 << 31), dict(n_rows=1 << 31), dict(n_rows=1 << 24, n_columns=1 << 7, ids_stride=1 << 7)):
        p = lookup(**big)
        assert A.lib().hbr_leaf_embedding_grad_workspace(C.byref(p), C.byref(n)) == A.REFUSED
    p = lookup(n_rows=(1 << 24) - 1, n_columns=1 << 7, ids_stride=1 << 7)
    assert A.lib().hbr_leaf_embedding_grad_workspace(C.byref(p), C.byref(n)) == A.OK and n.value > 1 << 31


def test_more_columns_than_the_kernels_count_are_refused():
    """One row of 2^32 - 1 ids fits a device's memory, and no loop over them
    in 32 bits would end."""
    n, ok = C.c_uint64(), 1 << 20
    for columns in (1 << 31, (1 << 32) - 1):
        p = lookup(n_rows=1, n_columns=columns, ids_stride=columns, ids=1 << 50)
        assert A.lib().hbr_leaf_embedding(99, C.byref(p), ok, 2 * ok, None) == A.REFUSED and "columns" in A.last_error()
        assert A.lib().hbr_leaf_embedding_grad(99, C.byref(p), ok, 2 * ok, 3 * ok, 1 << 60, None) == A.REFUSED
        assert A.lib().hbr_leaf_embedding_grad_workspace(C.byref(p), C.byref(n)) == A.REFUSED
    p = lookup(n_rows=1, n_columns=(1 << 31) - 1, ids_stride=1 << 31, ids=1 << 50)
    assert A.lib().hbr_leaf_embedding(99, C.byref(p), ok, 2 * ok, None) not in (A.OK, A.REFUSED)  # no such device


def softmax(**kw):
    ok = 1 << 20
    p = dict(dtype=A.BF16, dim=8, n_rows=3, n_classes=5, grad_scale=1.0, h_stride=8, w_stride=8, dh_stride=8,
             dw_stride=8, h=ok, w=ok, bias=None, labels=ok, weight=None, loss=ok, lse=None, best=None, dh=ok, dw=ok,
             db=ok)
    p.update(kw)
    return A.Softmax(**p)


@pytest.mark.parametrize("bad, said", [
    (dict(dtype=2), "type"), (dict(dim=0), "no classes"), (dict(n_classes=0), "no classes"), (dict(h=None), "null"),
    (dict(w=None), "null"), (dict(labels=None), "labels"), (dict(h_stride=7), "overlap"), (dict(w_stride=7), "overlap"),
    (dict(dh_stride=7), "overlap"), (dict(dw_stride=7), "overlap"), (dict(h=(1 << 20) + 1), "aligned"),
    (dict(dw=(1 << 20) + 1), "aligned"), (dict(bias=(1 << 20) + 2), "aligned"), (dict(best=(1 << 20) + 1), "aligned")])
def test_heads_with_malformed_records_are_invalid(bad, said):
    p = softmax(**bad)
    assert A.lib().hbr_softmax_head(0, C.byref(p), 1 << 20, 1 << 40, None) == A.INVALID and said in A.last_error()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_workspaces_of_all_sizes_are_named(dtype):
    """From no rows to the largest, with every count of classes on either
    side of a tile."""
    for n in (0, 1, 31, 1023, 1024, 70_000, (1 << 31) - 1):
        for classes in (1, 2, 64, 65, 128, 129, 131_072):
            for dim in (1, 7, 64, 1024, 70_000):
                for gradient in (False, True):
                    need = hb.softmax_head_workspace(n, classes, dim, dtype, gradient=gradient)
                    assert need >= 0 and need % 256 == 0
    for n in (0, 1, 16_383, 1 << 20):
        for columns in (0, 1, 3, 1000):
            for rows in (0, 1, 512, 1 << 20):
                assert hb.leaf_embedding_grad_workspace(n, columns, rows, 33, dtype) >= 0
    for n in (0, 1, 96, 97, 1 << 20):
        assert hb.clip_gradients_workspace(n) >= 8 * n // 96


def test_a_workspace_that_is_missing_short_or_misaligned_is_invalid():
    L, ok = A.lib(), 1 << 20
    need = hb.softmax_head_workspace(3, 5, 8, "bfloat16")
    p, q = softmax(), lookup()
    for w, size in ((None, need), (ok, need - 1), (ok + 8, need)):
        assert L.hbr_softmax_head(0, C.byref(p), w, size, None) == A.INVALID and "workspace" in A.last_error()
    need = hb.leaf_embedding_grad_workspace(3, 2, 5, 4, "float32")
    for w, size in ((None, need), (ok, need - 1), (ok + 4, need)):
        assert L.hbr_leaf_embedding_grad(0, C.byref(q), ok, ok, w, size, None) == A.INVALID
    need = hb.clip_gradients_workspace(1)
    t = A.Tensor(ok, ok, 4, A.F32, 0)
    for w, size in ((None, need), (ok, need - 1), (ok + 4, need)):
        assert L.hbr_clip_gradients(0, C.byref(t), 1, 1.0, None, w, size, None) == A.INVALID


def test_clipping_refuses_malformed_sets():
    L, ok, big = A.lib(), 1 << 20, 1 << 40
    t = A.Tensor(ok, ok, 4, A.F32, 0)
    for norm in (-1.0, float("nan")):
        assert L.hbr_clip_gradients(0, C.byref(t), 1, norm, None, ok, big, None) == A.INVALID
    assert L.hbr_clip_gradients(0, None, 1, 1.0, None, ok, big, None) == A.INVALID
    for bad in (A.Tensor(None, ok, 4, A.F32, 0), A.Tensor(ok, None, 4, A.F32, 0), A.Tensor(ok, ok, 4, 5, 0),
                A.Tensor(ok + 2, ok, 4, A.F32, 0), A.Tensor(ok, ok + 1, 4, A.BF16, 0)):
        assert L.hbr_clip_gradients(0, C.byref(bad), 1, 1.0, None, ok, big, None) == A.INVALID
    huge = A.Tensor(ok, ok, (1 << 42) + 1, A.BF16, 0)
    assert L.hbr_clip_gradients(0, C.byref(huge), 1, 1.0, None, ok, big, None) == A.REFUSED
    many = (A.Tensor * 9)(*[A.Tensor(ok, ok, 1 << 42, A.BF16, 0)] * 9)
    assert L.hbr_clip_gradients(0, many, 9, 1.0, None, ok, big, None) == A.REFUSED
    n = C.c_uint64()
    assert L.hbr_clip_gradients_workspace((1 << 20) + 1, C.byref(n)) == A.REFUSED


def test_clipping_refuses_sets_whose_outputs_overlap():
    L, ok, big, n = A.lib(), 1 << 20, 1 << 40, 64
    for pairs in ([(ok, ok), (ok, ok)], [(ok, ok), (ok + 4, ok + 4)], [(ok, ok + 4)], [(ok + 4, ok)],
                  [(ok, 2 * ok), (3 * ok, 2 * ok + 252)], [(ok, 2 * ok), (2 * ok, 3 * ok)],
                  [(5 * ok, 5 * ok), (ok, 3 * ok), (ok, 5 * ok - 4)]):
        t = (A.Tensor * len(pairs))(*[A.Tensor(a, b, n, A.F32, 0) for a, b in pairs])
        assert L.hbr_clip_gradients(0, t, len(pairs), 1.0, None, ok, big, None) == A.INVALID
        assert "overlaps" in A.last_error(), pairs
    # side by side, one tensor to two outputs, and empty ones anywhere, are not
    for pairs, last in (([(ok, ok), (ok + 4 * n, ok + 4 * n)], n), ([(ok, 2 * ok), (ok, 3 * ok)], n), ([(ok, ok), (ok + 4, ok + 4)], 0)):
        t = (A.Tensor * len(pairs))(*[A.Tensor(a, b, n, A.F32, 0) for a, b in pairs])
        t[len(pairs) - 1].len = last
        assert L.hbr_clip_gradients(99, t, len(pairs), 1.0, None, ok, big, None) != A.OK
        assert "overlaps" not in A.last_error(), pairs


def test_outputs_over_inputs_or_each_other_are_invalid():
    L, big = A.lib(), 1 << 40
    at = [(i + 1) << 20 for i in range(12)]  # arrays well apart

    def said(call):  # past the arguments' checks the device is what there is not
        assert call() != A.OK
        return "overlap" in A.last_error()

    def look(table=at[0], out=at[1], **kw):
        p = lookup(n_rows=300, table_rows=500, dim=8, table_stride=8, out_stride=8, n_columns=3, ids_stride=3, offset=at[3], scale=at[4], **{"ids": at[2], **kw})
        return [said(lambda: L.hbr_leaf_embedding(99, C.byref(p), table, out, None)),
                said(lambda: L.hbr_leaf_embedding_grad(99, C.byref(p), out, table, at[5], big, None))]

    assert look() == [False, False]
    assert look(table=at[1]) == [True, True]
    assert look(out=at[0] + 499 * 32) == [True, True] and look(out=at[0] + 500 * 32) == [False, False]
    assert look(out=at[2] + 8) == [True, False] and look(table=at[2] + 8) == [False, True]
    assert look(out=at[3] + 8) == [True, False] and look(table=at[4] - 8) == [False, True]
    assert look(ids=at[1] - 300 * 12) == [False, False] and look(ids=at[1] - 300 * 12 + 4) == [True, False]

    def head(**kw):
        p = softmax(**{**dict(n_rows=40, n_classes=70, dim=16, h_stride=16, w_stride=16, dh_stride=16, dw_stride=16, h=at[0],
                              w=at[1], bias=at[2], labels=at[3], weight=at[4], loss=at[5], lse=at[6], best=at[7], dh=at[8],
                              dw=at[9], db=at[10]), **kw})
        return said(lambda: L.hbr_softmax_head(99, C.byref(p), at[11], big, None))

    assert not head()
    assert head(dh=at[0]) and head(dw=at[1] + 69 * 32) and head(loss=at[3]) and head(lse=at[5] + 156) and head(best=at[4] - 4)
    assert not head(lse=at[5] + 160) and not head(dh=at[0] + 40 * 32)
    # rows beside each other in one buffer, and not quite beside
    assert not head(h_stride=32, dh=at[0] + 32, dh_stride=32) and not head(dh=at[0] - 32, h_stride=32, dh_stride=32)
    assert head(h_stride=32, dh=at[0] + 30, dh_stride=32) and head(h_stride=31, dh=at[0] + 32, dh_stride=31)
    assert head(h_stride=32, dh=at[0] + 39 * 64 + 16, dh_stride=32) and not head(h_stride=32, dh=at[0] + 39 * 64 + 32, dh_stride=32)
    # a vector within a row, and between two
    assert head(h_stride=1024, db=at[0] + 5 * 2048 + 28) and not head(h_stride=1024, db=at[0] + 5 * 2048 + 32)
    assert head(h_stride=1024, db=at[0] + 5 * 2048 - 276) and not head(h_stride=1024, db=at[0] + 5 * 2048 - 280)
    # what takes no room overlaps nothing
    assert not head(n_rows=0, dh=at[0], loss=at[3])

    def clip(norm, *spans):
        t = (A.Tensor * len(spans))(*[A.Tensor(a, b, 64, A.F32, 0) for a, b in spans])
        return said(lambda: L.hbr_clip_gradients(99, t, len(spans), 1.0, norm, at[11], big, None))

    assert not clip(at[2], (at[0], at[0]), (at[1], at[3]))
    assert clip(at[0] + 252, (at[0], at[0])) and clip(at[1], (at[0], at[0]), (at[1], at[3])) and clip(at[3] + 4, (at[1], at[3]))
    assert not clip(at[0] + 256, (at[0], at[0])) and not clip(at[0] - 4, (at[0], at[0]))


def test_a_workspace_over_an_array_is_invalid():
    L, big = A.lib(), 1 << 40
    at = [(i + 1) << 24 for i in range(12)]

    def lies_over(call):
        assert call() != A.OK
        return "the call's own use" in A.last_error()

    need = hb.leaf_embedding_grad_workspace(300, 3, 500, 8, "float32")
    p = lookup(n_rows=300, table_rows=500, dim=8, table_stride=8, out_stride=8, n_columns=3, ids_stride=3, ids=at[2], scale=at[4])
    for w, over in ((at[8], False), (at[2] - 16, True), (at[0] + 256, True), (at[1] + 500 * 32, False), (at[4], True)):
        assert lies_over(lambda: L.hbr_leaf_embedding_grad(99, C.byref(p), at[0], at[1], w, max(need, big), None)) == over, w
    q = softmax(n_rows=40, n_classes=70, dim=16, h_stride=16, w_stride=16, dh_stride=16, dw_stride=16, h=at[0], w=at[1], bias=at[2],
                labels=at[3], weight=at[4], loss=at[5], lse=at[6], best=at[7], dh=at[8], dw=at[9], db=at[10])
    for w, over in ((at[11], False), (at[0], True), (at[9] - 256, True), (at[10] + 512, False), (at[3] - 64, True)):
        assert lies_over(lambda: L.hbr_softmax_head(99, C.byref(q), w, big, None)) == over, w
    t = A.Tensor(at[0], at[1], 64, A.F32, 0)
    for w, over in ((at[3], False), (at[0] - 16, True), (at[1] + 240, True), (at[1] + 256, False), (at[2] - 16, True)):
        assert lies_over(lambda: L.hbr_clip_gradients(99, C.byref(t), 1, 1.0, at[2], w, big, None)) == over, w


def test_sizes_past_a_launch_are_refused():
    L, ok, big, n = A.lib(), 1 << 20, 1 << 62, C.c_uint64()
    p = lookup(dim=1 << 20, table_stride=1 << 20, out_stride=1 << 20)
    assert L.hbr_leaf_embedding(0, C.byref(p), ok, ok, None) == A.REFUSED
    assert L.hbr_leaf_embedding_grad(0, C.byref(p), ok, ok, ok, big, None) == A.REFUSED
    assert L.hbr_softmax_head_workspace(3, 5, 1 << 20, A.F32, 1, C.byref(n)) == A.REFUSED
    for rows, classes, dim in ((1 << 20, 1 << 18, 256), (1 << 20, 1 << 18, 8), ((1 << 31) - 1, 100, 8)):
        p = softmax(n_rows=rows, n_classes=classes, dim=dim, h_stride=dim, w_stride=dim, dh_stride=dim, dw_stride=dim)
        assert L.hbr_softmax_head(0, C.byref(p), ok, big, None) == A.REFUSED and "tiles" in A.last_error()
    # many columns of long vectors are not summed a column at a time
    for columns in (1 << 15, 1 << 15 | 1):
        p = lookup(n_rows=1 << 12, n_columns=columns, ids_stride=columns, table_rows=1 << 15 | 1, dim=1024, table_stride=1024, out_stride=1024)
        assert L.hbr_leaf_embedding_grad_workspace(C.byref(p), C.byref(n)) == A.OK and n.value > 1 << 30


def test_a_named_workspace_serves_every_stride_and_offset():
    """A gradient's way, and so its need, depends on them too."""
    L, ok, n = A.lib(), 1 << 20, C.c_uint64()
    for rows, columns, table_rows, dim in ((9, 1, 8, 37), (500, 1, 8, 37), (500, 20, 300, 16), (200_003, 100, 12_700, 64), (20_000, 1, 500, 256), (50_000, 3, 90, 1000)):
        p = lookup(n_rows=rows, n_columns=columns, ids_stride=columns, table_rows=table_rows, dim=dim, table_stride=dim, out_stride=dim)
        assert L.hbr_leaf_embedding_grad_workspace(C.byref(p), C.byref(n)) == A.OK
        for stride in (dim, 1 << 20):
            for offset in (None, ok):
                p.out_stride, p.offset = stride, C.cast(offset, C.POINTER(C.c_int32)) if isinstance(p.offset, C.POINTER(C.c_int32)) else offset
                # past the arguments' checks: the device is what there is not
                assert L.hbr_leaf_embedding_grad(99, C.byref(p), ok, ok, ok, n.value, None) != A.OK
                assert "workspace" not in A.last_error()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_workspace_serves_fewer_rows_and_calls_without_gradients(dtype):
    """A loop's last batch, and its evaluation, run on what its largest batch
    was given."""
    rng = np.random.default_rng(3)
    counts = np.unique(np.r_[0:70, 4000:4200:7, 599_990:600_010, np.exp(rng.uniform(0, 13.5, 700)).astype(int)])
    for classes, dim in ((10, 50), (64, 300), (65, 8), (200, 96), (5003, 64), (5003, 256), (30_000, 100), (8192, 1024),
                         (131_072, 16), (131_072, 1024), (1_000_003, 200)):
        held = 0
        for n in counts.tolist():
            need = hb.softmax_head_workspace(n, classes, dim, dtype)
            assert need >= held, (n, classes, dim)
            assert need >= hb.softmax_head_workspace(n, classes, dim, dtype, gradient=False), (n, classes, dim)
            held = need
        held = 0
        for n in counts.tolist():
            need = hb.softmax_head_workspace(n, classes, dim, dtype, gradient=False)
            assert need >= held, (n, classes, dim)
            held = need
    for columns, rows, dim in ((1, 500, 64), (1, 131_072, 1024), (20, 10_220, 256), (100, 12_700, 64), (6, 594, 388), (3, 90, 5000)):
        held = 0
        for n in counts.tolist():
            need = hb.leaf_embedding_grad_workspace(n, columns, rows, dim, dtype)
            assert need >= held, (n, columns, rows, dim)
            held = need
    # 200,000 rows over all classes: scores alone do not hold a part of each tile of them
    assert hb.softmax_head_workspace(200_000, 131_072, 16, dtype, gradient=False) < 200 << 20
    held = [hb.clip_gradients_workspace(n) for n in range(400)]
    assert held == sorted(held)


def test_a_call_needs_no_more_than_was_named_for_more_rows():
    """Past the arguments' checks on a workspace named for a larger batch: the
    device is what there is not."""
    L, ok, rng = A.lib(), 1 << 20, np.random.default_rng(4)
    for dtype, code in (("float32", A.F32), ("bfloat16", A.BF16)):
        for _ in range(300):
            classes, dim = (int(v) for v in np.exp(rng.uniform(np.log([2, 4]), np.log([131_072, 1_024]))))
            most = int(np.exp(rng.uniform(0, 12)))
            need = hb.softmax_head_workspace(most, classes, dim, dtype)
            for n in rng.integers(1, most + 1, 8).tolist():
                p = softmax(dtype=code, dim=dim, n_rows=n, n_classes=classes, h_stride=dim, w_stride=dim, dh_stride=dim, dw_stride=dim)
                assert L.hbr_softmax_head(99, C.byref(p), ok, need, None) != A.OK and "workspace" not in A.last_error()
                p.labels = p.dh = p.dw = p.db = None
                assert L.hbr_softmax_head(99, C.byref(p), ok, need, None) != A.OK and "workspace" not in A.last_error()
            columns = int(rng.choice([1, 3, 40]))
            rows = columns * int(np.exp(rng.uniform(0, 8)))
            need = hb.leaf_embedding_grad_workspace(most, columns, rows, dim, dtype)
            for n in rng.integers(1, most + 1, 8).tolist():
                q = lookup(dtype=code, dim=dim, n_rows=n, n_columns=columns, ids_stride=columns, table_rows=rows,
                           table_stride=dim, out_stride=dim, offset=ok if rng.random() < 0.7 else None)
                assert L.hbr_leaf_embedding_grad(99, C.byref(q), ok, ok, ok, need, None) != A.OK
                assert "workspace" not in A.last_error()


def test_python_arrays_are_checked():
    f, i = "float32", "int32"
    table, ids, out = arr(f, 10, 4), arr(i, 6, 3), arr(f, 6, 4)
    bad = [
        dict(table=arr(i, 10, 4)), dict(table=arr(f, 40)), dict(out=arr(f, 6, 5)), dict(out=arr("bfloat16", 6, 4)),
        dict(out=arr(f, 5, 4)), dict(ids=arr(f, 6, 3)), dict(ids=arr(i, 6)), dict(offset=arr(i, 4)),
        dict(scale=arr(i, 3)), dict(out=arr(f, 6, 4, ordinal=1)), dict(table=arr(f, 10, 4, stride=3)),
    ]
    for kw in bad:
        a = dict(table=table, ids=ids, out=out)
        a.update(kw)
        with pytest.raises(ValueError):
            hb.leaf_embedding(a.pop("table"), a.pop("ids"), a.pop("out"), **a)
    h, w = arr(f, 6, 4), arr(f, 7, 4)
    for kw in (dict(bias=arr(f, 6)), dict(labels=arr(f, 6)), dict(labels=arr(i, 7)), dict(weight=arr(f, 7)),
               dict(dh=arr(f, 7, 4)), dict(dw=arr(f, 6, 4)), dict(db=arr(f, 6)), dict(best=arr(f, 6)),
               dict(loss=arr("bfloat16", 6))):
        with pytest.raises(ValueError):
            hb.softmax_head(h, w, **kw)
    with pytest.raises(ValueError):
        hb.softmax_head(h, arr(f, 7, 5))
    with pytest.raises(ValueError):
        hb.softmax_head(h, arr("bfloat16", 7, 4))
    with pytest.raises(hb.HbrError, match="labels"):
        hb.softmax_head(h, w, db=arr(f, 7))
    with pytest.raises(ValueError):
        hb.clip_gradients([h], 1.0, out=[arr(f, 23)])
    with pytest.raises(ValueError):
        hb.clip_gradients([h], 1.0, out=[])
    with pytest.raises(ValueError):
        hb.clip_gradients([arr(f, 6, 4, stride=5)], 1.0)
    with pytest.raises(ValueError):
        hb.clip_gradients([arr(i, 6)], 1.0)
    with pytest.raises(ValueError):
        hb.softmax_head_workspace(3, 5, 8, "float16")


def test_sizes_past_a_record_s_fields_are_refused_and_not_cut_off():
    far = dict(nbytes=1 << 60)
    f, i = "float32", "int32"

    def big(dtype, *shape):
        return DeviceArray(Memory(**far), dtype, shape)

    for bad in (dict(n=-1), dict(classes=(1 << 32) + 5), dict(dim=(1 << 32) + 8), dict(dim=-8), dict(n=1 << 64), dict(dtype="int32")):
        with pytest.raises(ValueError):
            hb.softmax_head_workspace(**{**dict(n=3, classes=70, dim=8, dtype=f), **bad})
    for bad in (dict(n=-1), dict(columns=(1 << 32) + 1), dict(dim=(1 << 32) + 8), dict(table_rows=-5), dict(dtype="int32")):
        with pytest.raises(ValueError):
            hb.leaf_embedding_grad_workspace(**{**dict(n=3, columns=2, table_rows=8, dim=8, dtype=f), **bad})
    with pytest.raises(ValueError):
        hb.clip_gradients_workspace(-1)
    wide = (1 << 32) + 8
    with pytest.raises(ValueError, match="dim"):
        hb.leaf_embedding(big(f, 1, wide), arr(i, 1, 1), big(f, 1, wide))
    with pytest.raises(ValueError, match="columns"):
        hb.leaf_embedding(arr(f, 5, 4), big(i, 1, wide), arr(f, 1, 4))
    with pytest.raises(ValueError, match="dim"):
        hb.leaf_embedding_grad(big(f, 1, wide), arr(i, 1, 1), big(f, 1, wide))
    with pytest.raises(ValueError, match="dim"):
        hb.softmax_head(big(f, 1, wide), big(f, 3, wide), loss=arr(f, 1))
    with pytest.raises(ValueError, match="classes"):
        hb.softmax_head(arr(f, 1, 4), big(f, wide, 4), loss=arr(f, 1))


def test_types_are_named_or_given_as_type_objects():
    for d in ("float32", np.float32, np.dtype(np.float32), "torch.float32"):
        assert hb.softmax_head_workspace(3, 70, 8, d) == hb.softmax_head_workspace(3, 70, 8, "float32")
    assert DeviceArray(Memory(), np.int32, 5).dtype == "int32"
    for d in (np.float64, "float16", float):
        with pytest.raises(ValueError):
            hb.softmax_head_workspace(3, 70, 8, d)


def test_a_device_array_fits_its_buffer():
    m = Memory(nbytes=100)
    DeviceArray(m, "float32", (5, 5))
    DeviceArray(m, "bfloat16", (5, 4), stride=11)
    DeviceArray(m, "uint8", 100)
    for bad in (dict(dtype="float32", shape=(5, 5), byte_offset=4), dict(dtype="float32", shape=26),
                dict(dtype="bfloat16", shape=(5, 5), stride=12), dict(dtype="float32", shape=4, byte_offset=-4),
                dict(dtype="float32", shape=(2, 2, 2)), dict(dtype="float64", shape=2)):
        with pytest.raises(ValueError):
            DeviceArray(m, **bad)


def test_the_reference_rounds_to_bf16_as_numpy_can_check():
    from leaf_reference import from_bf16, to_bf16
    x = np.array([1.0, 1.00390625, 1.01171875, -3.4e38, 1e-40, np.inf], np.float32)
    assert to_bf16(x).tolist() == [0x3F80, 0x3F80, 0x3F82, 0xFF80, 0x0001, 0x7F80]
    assert np.isnan(from_bf16(to_bf16(np.array([np.nan], np.float32))))[0]
