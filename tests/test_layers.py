"""The operators of the layers between leaf vectors and classes refuse what
they cannot run, before they touch a device."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import hessboost_amd as hb
import layer_reference as L
from hessboost_amd import _capi as A
from test_leafops import Memory, arr  # noqa: F401

OK = 1 << 20
AT = [(i + 1) << 24 for i in range(20)]  # arrays well apart
BIG = 1 << 60


def norm(**kw):
    p = dict(dtype=A.BF16, dim=40, n_rows=6, x_stride=40, residual_stride=40, out_stride=40, total_stride=40, codes_stride=40,
             scales_stride=2, x=AT[0], residual=AT[1], weight=AT[2], out=AT[3], total=AT[4], inv=AT[5], codes=AT[6], scales=AT[7],
             eps=1e-6, normed=0)
    p.update(kw)
    return A.lib().hbr_rms_norm(99, C.byref(A.Norm(**p)), None)


def norm_grad(workspace=(AT[12], BIG), **kw):
    p = dict(dtype=A.F32, dim=40, n_rows=6, dout_stride=40, x_stride=40, codes_stride=40, scales_stride=2, dtotal_stride=40, dx_stride=40,
             dout=AT[0], x=AT[1], codes=None, scales=None, inv=AT[4], weight=AT[5], dtotal=AT[6], dx=AT[7], dweight=AT[8], eps=1e-6, pad=0)
    p.update(kw)
    return A.lib().hbr_rms_norm_grad(99, C.byref(A.NormGrad(**p)), *workspace, None)


def packed(unpack, x=AT[0], codes=AT[1], scales=AT[2], weight=None, **kw):
    p = dict(dtype=A.F32, dim=40, n_rows=6, x_stride=40, codes_stride=40, scales_stride=2)
    p.update(kw)
    p = A.Packed(**p)
    if unpack:
        return A.lib().hbr_unpack_rows(99, C.byref(p), codes, scales, weight, x, None)
    return A.lib().hbr_pack_rows(99, C.byref(p), x, codes, scales, None)


def linear(workspace=(AT[12], BIG), **kw):
    p = dict(dtype=A.BF16, dim=40, n_rows=70, n_outs=30, rank=4, n_adapters=3, pad=0, x_stride=40, w_stride=40, out_stride=30,
             down_stride=40, up_stride=4, x=AT[0], w=AT[1], bias=AT[2], down=AT[3], up=AT[4], ids=AT[5], scale=AT[6], out=AT[7])
    p.update(kw)
    return A.lib().hbr_linear(99, C.byref(A.Linear(**p)), *workspace, None)


def linear_grad(workspace=(AT[12], BIG), **kw):
    p = dict(dtype=A.F32, dim=40, n_rows=70, n_outs=30, pad=0, dout_stride=30, w_stride=40, x_stride=40, codes_stride=40, scales_stride=2,
             dx_stride=40, dw_stride=40, dout=AT[0], w=AT[1], x=AT[2], codes=None, scales=None, weight=AT[5], dx=AT[6], dw=AT[7], db=AT[8])
    p.update(kw)
    return A.lib().hbr_linear_grad(99, C.byref(A.LinearGrad(**p)), *workspace, None)


def checked(status):
    """Past the arguments' checks: the device is what there is not."""
    return status != A.OK and "device" in A.last_error()


def test_whole_records_pass_the_checks():
    for call in (norm, norm_grad, lambda: packed(False), lambda: packed(True), linear, linear_grad):
        assert checked(call()), A.last_error()
    L_ = A.lib()
    for f in (lambda: L_.hbr_rms_norm(0, None, None), lambda: L_.hbr_rms_norm_grad(0, None, OK, 1, None),
              lambda: L_.hbr_pack_rows(0, None, OK, OK, OK, None), lambda: L_.hbr_unpack_rows(0, None, OK, OK, None, OK, None),
              lambda: L_.hbr_linear(0, None, OK, 1, None), lambda: L_.hbr_linear_grad(0, None, OK, 1, None),
              lambda: L_.hbr_rms_norm_grad_workspace(1, 1, 0, None), lambda: L_.hbr_linear_workspace(1, 1, 1, 1, 0, None),
              lambda: L_.hbr_linear_grad_workspace(1, 1, 1, 0, None)):
        assert f() == A.INVALID and "null" in A.last_error()


@pytest.mark.parametrize("bad, said", [
    (dict(dtype=2), "type"), (dict(dim=0), "no elements"), (dict(x=None), "null"), (dict(x_stride=39), "overlap"),
    (dict(residual_stride=39), "overlap"), (dict(out_stride=39), "overlap"), (dict(total_stride=1), "overlap"),
    (dict(codes_stride=39), "overlap"), (dict(scales_stride=1), "overlap"), (dict(codes=None), "together"), (dict(scales=None), "together"),
    (dict(x=AT[0] + 1), "aligned"), (dict(weight=AT[2] + 2), "aligned"), (dict(inv=AT[5] + 1), "aligned"), (dict(eps=-1e-6), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(out=AT[4]), "two outputs"), (dict(out=AT[0] + 2 * 40), "overlaps an input"),
    (dict(out=AT[0], out_stride=41), "overlaps an input"), (dict(total=AT[2]), "overlaps an input"), (dict(inv=AT[1] + 8), "overlaps an input"),
    (dict(codes=AT[0] + 479), "overlaps an input"), (dict(scales=AT[6] + 239), "two outputs")])
def test_malformed_norms_are_invalid(bad, said):
    assert norm(**bad) == A.INVALID and said in A.last_error()


def test_norms_over_their_inputs_are_not_refused():
    for kw in (dict(out=AT[0]), dict(total=AT[1]), dict(out=AT[0], total=AT[1]), dict(out=AT[1], total=AT[0]), dict(codes=AT[0] + 480),
               dict(n_rows=1, x_stride=0, out_stride=7), dict(residual=None, weight=None), dict(out=None, total=None, inv=None)):
        assert checked(norm(**kw)), (kw, A.last_error())
    # the same array, but in another place of it
    assert norm(out=AT[0], total=AT[0]) == A.INVALID
    assert norm(n_rows=0, x=None) == A.OK


@pytest.mark.parametrize("bad, said", [
    (dict(dtype=9), "type"), (dict(dim=0), "no elements"), (dict(dout=None), "null"), (dict(x=None), "are needed"),
    (dict(codes=AT[2], scales=AT[3]), "are needed"), (dict(codes=AT[2]), "together"), (dict(x=None, codes=AT[2], scales=AT[3], inv=None), "inv"),
    (dict(inv=None, eps=-1.0), "eps"), (dict(dout_stride=39), "overlap"), (dict(dx_stride=39), "overlap"), (dict(dtotal_stride=39), "overlap"),
    (dict(dx=AT[7] + 2), "aligned"), (dict(dweight=AT[8] + 1), "aligned"), (dict(dx=AT[1]), "overlaps an input"),
    (dict(dx=AT[0] + 4), "overlaps an input"), (dict(dweight=AT[5]), "overlaps an input"), (dict(dweight=AT[7] + 8), "two outputs")])
def test_malformed_norm_gradients_are_invalid(bad, said):
    assert norm_grad(**bad) == A.INVALID and said in A.last_error()


def test_norm_gradients_over_their_inputs_are_not_refused():
    for kw in (dict(dx=AT[0]), dict(dx=AT[6]), dict(dx=None), dict(dweight=None), dict(dtotal=None, weight=None, inv=None),
               dict(x=None, codes=AT[2], scales=AT[3])):
        assert checked(norm_grad(**kw)), (kw, A.last_error())
    # without dweight no workspace
    assert checked(norm_grad(workspace=(None, 0), dweight=None))
    assert norm_grad(dx=None, dweight=None) == A.OK


@pytest.mark.parametrize("bad, said", [
    (dict(dtype=3), "type"), (dict(dim=0), "no elements"), (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"),
    (dict(x_stride=39), "overlap"), (dict(codes_stride=39), "overlap"), (dict(scales_stride=1), "overlap"), (dict(x=AT[0] + 2), "aligned"),
    (dict(codes=AT[0] + 959), "overlap"), (dict(scales=AT[0]), "overlap")])
@pytest.mark.parametrize("unpack", [False, True])
def test_malformed_packs_are_invalid(unpack, bad, said):
    assert packed(unpack, **bad) == A.INVALID and said in A.last_error()
    assert packed(unpack, n_rows=0, x=None) == A.OK
    assert packed(True, weight=AT[3] + 2) == A.INVALID and packed(True, weight=AT[0] + 8) == A.INVALID


@pytest.mark.parametrize("bad, said", [
    (dict(dtype=5), "type"), (dict(dim=0), "no elements"), (dict(n_outs=0), "no outputs"), (dict(x=None), "null"), (dict(w=None), "null"),
    (dict(out=None), "null"), (dict(down=None), "adapters need"), (dict(up=None), "adapters need"), (dict(ids=None), "adapters need"),
    (dict(x_stride=39), "overlap"), (dict(w_stride=39), "overlap"), (dict(out_stride=29), "overlap"), (dict(down_stride=39), "overlap"),
    (dict(up_stride=3), "overlap"), (dict(x=AT[0] + 1), "aligned"), (dict(bias=AT[2] + 1), "aligned"), (dict(ids=AT[5] + 2), "aligned"),
    (dict(out=AT[0]), "overlaps an input"), (dict(out=AT[1] + 8), "overlaps an input"), (dict(out=AT[4]), "overlaps an input"),
    (dict(out=AT[5] + 276), "overlaps an input"), (dict(x=AT[12] + 64), "own use")])
def test_malformed_projections_are_invalid(bad, said):
    assert linear(**bad) == A.INVALID and said in A.last_error()


def test_projections_without_adapters_need_none_of_their_arrays():
    for kw in (dict(rank=0), dict(n_adapters=0)):
        assert checked(linear(down=None, up=None, ids=None, scale=None, **kw)), A.last_error()
        assert checked(linear(out=AT[5], **kw))  # what is not read may be written
    assert checked(linear(bias=None, scale=None)) and linear(n_rows=0, x=None) == A.OK


@pytest.mark.parametrize("bad, said", [
    (dict(dtype=5), "type"), (dict(dim=0), "no elements"), (dict(n_outs=0), "no outputs"), (dict(dout=None), "null"), (dict(w=None), "needs w"),
    (dict(x=None), "needs the rows"), (dict(codes=AT[3], scales=AT[4]), "needs the rows"), (dict(codes=AT[3]), "together"),
    (dict(dout_stride=29), "overlap"), (dict(w_stride=39), "overlap"), (dict(x_stride=39), "overlap"), (dict(dx_stride=39), "overlap"),
    (dict(dw_stride=39), "overlap"), (dict(dout=AT[0] + 2), "aligned"), (dict(weight=AT[5] + 2), "aligned"), (dict(db=AT[8] + 2), "aligned"),
    (dict(dx=AT[0]), "overlaps an input"), (dict(dw=AT[1]), "overlaps an input"), (dict(db=AT[6] + 16), "two outputs"),
    (dict(dw=AT[12] + 1024), "own use")])
def test_malformed_projection_gradients_are_invalid(bad, said):
    assert linear_grad(**bad) == A.INVALID and said in A.last_error()


def test_projection_gradients_need_only_what_they_read():
    for kw in (dict(w=None, dx=None), dict(x=None, dw=None), dict(x=None, codes=AT[3], scales=AT[4]), dict(dx=None, dw=None, w=None, x=None),
               dict(db=None, weight=None)):
        assert checked(linear_grad(**kw)), (kw, A.last_error())
    assert linear_grad(dx=None, dw=None, db=None) == A.OK


def test_workspaces_that_are_missing_short_or_misaligned_are_invalid():
    for call, need in ((norm_grad, hb.rms_norm_grad_workspace(6, 40, "float32")), (linear, hb.linear_workspace(70, 30, 40, "bfloat16", rank=4)),
                       (linear_grad, hb.linear_grad_workspace(70, 30, 40, "float32"))):
        assert checked(call(workspace=(AT[12], need)))
        for ws in ((None, need), (AT[12], need - 1), (AT[12] + 8, need)):
            assert call(workspace=ws) == A.INVALID and "workspace" in A.last_error()


def test_sizes_past_the_limits_are_refused():
    n = C.c_uint64()
    L_ = A.lib()
    big = 1 << 20
    for f in (lambda: norm(dim=big, x_stride=big), lambda: norm(n_rows=1 << 31), lambda: norm_grad(dim=big), lambda: packed(False, dim=big),
              lambda: packed(True, n_rows=1 << 31), lambda: linear(dim=big), lambda: linear(n_outs=big), lambda: linear(rank=big),
              lambda: linear(n_rows=1 << 31), lambda: linear(n_adapters=1 << 31), lambda: linear(n_rows=1 << 28),
              lambda: linear(n_rows=1 << 25, n_outs=1 << 18), lambda: linear_grad(dim=big),
              lambda: linear_grad(n_outs=big), lambda: linear_grad(n_rows=1 << 25, dim=1 << 18),
              lambda: L_.hbr_rms_norm_grad_workspace(1 << 31, 8, A.F32, C.byref(n)), lambda: L_.hbr_linear_workspace(5, big, 8, 0, A.F32, C.byref(n)),
              lambda: L_.hbr_linear_workspace(5, 8, 8, big, A.F32, C.byref(n)), lambda: L_.hbr_linear_grad_workspace(5, 8, big, A.F32, C.byref(n))):
        assert f() == A.REFUSED, A.last_error()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_workspace_serves_fewer_rows(dtype):
    """Named for more rows it is no smaller, and a call on fewer needs no more."""
    rng = np.random.default_rng(7)
    code = A.F32 if dtype == "float32" else A.BF16
    counts = np.unique(np.r_[0:300:7, 1:9, 4090:4100, np.exp(rng.uniform(0, 13, 300)).astype(int)]).tolist()
    for dim, outs, rank in ((1, 1, 1), (8, 300, 4), (250, 333, 9), (1024, 4096, 16), (4096, 64, 64), (64, 8192, 0), (5000, 130, 3)):
        held = [0, 0, 0]
        for n in counts:
            need = [hb.rms_norm_grad_workspace(n, dim, dtype), hb.linear_workspace(n, outs, dim, dtype, rank=rank),
                    hb.linear_grad_workspace(n, outs, dim, dtype)]
            assert all(a >= b for a, b in zip(need, held)), (n, dim, outs)
            held = need
            assert need[1] >= hb.linear_workspace(n, outs, dim, dtype)
    for _ in range(300):
        dim, outs, most = (int(v) for v in np.exp(rng.uniform(0, np.log([8192, 8192, 100_000]))))
        rank = int(rng.integers(0, 65))
        named = hb.linear_workspace(most, outs, dim, dtype, rank=rank), hb.linear_grad_workspace(most, outs, dim, dtype)
        for n in rng.integers(1, most + 1, 6).tolist():
            kw = dict(dtype=code, dim=dim, n_rows=n, n_outs=outs, x_stride=dim, w_stride=dim)
            # arrays far enough apart for any of these sizes
            far = [(i + 1) << 40 for i in range(12)]
            assert checked(linear(workspace=(far[11], named[0]), rank=rank, down_stride=dim, up_stride=max(1, rank), out_stride=outs,
                                  x=far[0], w=far[1], bias=far[2], down=far[3], up=far[4], ids=far[5], scale=far[6], out=far[7], **kw)), A.last_error()
            for held in (False, True):
                rows = dict(x=None, codes=far[2], scales=far[3]) if held else dict(x=far[2])
                assert checked(linear_grad(workspace=(far[11], named[1]), dout_stride=outs, codes_stride=dim, scales_stride=dim, dx_stride=dim,
                                           dw_stride=dim, dout=far[0], w=far[1], weight=far[4], dx=far[5], dw=far[6], db=far[7], **rows, **kw)), A.last_error()


def test_python_arrays_of_layers_are_checked():
    f, b, u = "float32", "bfloat16", "uint8"
    x, codes, scales = arr(f, 6, 40), arr(u, 6, 40), arr(u, 6, 2)
    bad = [
        lambda: hb.pack_rows(arr(u, 6, 40), codes, scales), lambda: hb.pack_rows(x, arr(u, 6, 41), scales), lambda: hb.pack_rows(x, codes, arr(u, 6, 3)),
        lambda: hb.pack_rows(x, arr(f, 6, 40), scales), lambda: hb.unpack_rows(codes, scales, arr(f, 6, 39)),
        lambda: hb.unpack_rows(codes, scales, x, weight=arr(f, 41)), lambda: hb.rms_norm(x, arr(b, 6, 40)), lambda: hb.rms_norm(x, arr(f, 5, 40)),
        lambda: hb.rms_norm(x, weight=arr(b, 40)), lambda: hb.rms_norm(x, residual=arr(f, 6, 41)), lambda: hb.rms_norm(x, inv=arr(f, 7)),
        lambda: hb.rms_norm(x, codes=codes), lambda: hb.rms_norm(x, scales=scales), lambda: hb.rms_norm(arr(f, 240)),
        lambda: hb.rms_norm(x, total=arr(f, 6, 40, ordinal=1)), lambda: hb.rms_norm_grad(x, arr(f, 6, 41), x=x),
        lambda: hb.rms_norm_grad(x, x=x, dweight=arr(f, 41)), lambda: hb.rms_norm_grad(x, x=arr(b, 6, 40)),
        lambda: hb.linear(x, arr(f, 7, 41), arr(f, 6, 7)), lambda: hb.linear(x, arr(f, 7, 40), arr(f, 6, 8)), lambda: hb.linear(x, arr(b, 7, 40), arr(f, 6, 7)),
        lambda: hb.linear(x, arr(f, 7, 40), arr(f, 6, 7), down=arr(f, 6, 40)), lambda: hb.linear(x, arr(f, 7, 40), arr(f, 6, 7), scale=arr(f, 3)),
        lambda: hb.linear(x, arr(f, 7, 40), arr(f, 6, 7), down=arr(f, 6, 40), up=arr(f, 22, 2), ids=arr("int32", 6)),
        lambda: hb.linear(x, arr(f, 7, 40), arr(f, 6, 7), down=arr(f, 6, 40), up=arr(f, 14, 2), ids=arr("int32", 6)),
        lambda: hb.linear(x, arr(f, 7, 40), arr(f, 6, 7), down=arr(f, 7, 40), up=arr(f, 21, 2), ids=arr("int32", 6)),
        lambda: hb.linear(x, arr(f, 7, 40), arr(f, 6, 7), down=arr(f, 6, 40), up=arr(f, 21, 2), ids=arr("int32", 7)),
        lambda: hb.linear_grad(arr(f, 6, 7), arr(f, 8, 40), dx=x), lambda: hb.linear_grad(arr(f, 6, 7), x=x, dw=arr(f, 7, 41)),
        lambda: hb.linear_grad(arr(f, 6, 7), codes=codes, dw=arr(f, 7, 40)), lambda: hb.linear_grad(arr(f, 6, 7), db=arr(f, 6)),
        lambda: hb.packed_scales(-1), lambda: hb.linear_workspace(5, 7, 1 << 32, f), lambda: hb.rms_norm_grad_workspace(5, 8, "int32"),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k}")
    assert [hb.packed_scales(d) for d in (1, 32, 33, 64, 65)] == [1, 1, 2, 2, 3]


def test_records_are_filled_as_the_header_lays_them_out():
    for record in (A.Packed, A.Norm, A.NormGrad, A.Linear, A.LinearGrad):
        values = [float(k) if t is C.c_float else k + 1 for k, (_, t) in enumerate(record._fields_)]
        p = record.from_buffer_copy(A.packer(record)(*values))
        assert [getattr(p, name) for name, _ in record._fields_] == values


def test_the_codes_of_the_plain_form_are_the_nearest():
    """The reference's own codes, by another way: every code tried."""
    rng = np.random.default_rng(1)
    v = (rng.standard_normal((5, 70)) * 10.0 ** rng.integers(-8, 8, (5, 70))).astype(np.float32).astype(np.float64)
    v[1, 3], v[2, 0], v[3, :32] = np.inf, np.nan, 0.0
    codes, scales = L.codes_of(v)
    held = L.values_of(codes, scales)
    power = np.repeat(2.0 ** (scales.astype(np.float64) - 127), 32, 1)[:, :70]
    grid = L.code_values()
    for r in range(5):
        for c in range(70):
            if np.isfinite(v[r, c]):
                best = np.nanmin(np.abs(grid * power[r, c] - v[r, c]))
                assert np.abs(held[r, c] - v[r, c]) == best
            else:
                assert np.isnan(held[r, c])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_few_rows_need_room_for_their_low_values_alone(dtype):
    """Up to 64 rows (in bfloat16 16, and more where w is small) read x and w in
    place: without adapters no workspace is needed, with them f32 values."""
    code = A.F32 if dtype == "float32" else A.BF16
    far = [(i + 1) << 40 for i in range(12)]
    for n, outs, dim in ((1, 8192, 8192), (16, 14_336, 4096), (64, 512, 256), (3, 7, 5)):
        assert hb.linear_workspace(n, outs, dim, dtype) == 0
        assert 4 * n * 16 <= hb.linear_workspace(n, outs, dim, dtype, rank=16) <= 4 * n * 16 + 255
        kw = dict(dtype=code, dim=dim, n_rows=n, n_outs=outs, x_stride=dim, w_stride=dim, out_stride=outs, x=far[0], w=far[1], bias=far[2], out=far[7])
        assert checked(linear(workspace=(None, 0), rank=0, down=None, up=None, ids=None, scale=None, **kw)), A.last_error()
        kw.update(rank=16, down_stride=dim, up_stride=16, down=far[3], up=far[4], ids=far[5], scale=far[6])
        assert checked(linear(workspace=(far[11], hb.linear_workspace(n, outs, dim, dtype, rank=16)), **kw)), A.last_error()
        assert linear(workspace=(far[11], 4 * n * 16 - 1), **kw) == A.INVALID


def test_the_layers_kernels_keep_their_registers(tmp_path):
    """Rows and tiles that are held in registers are not put away in scratch
    memory: by the built code object's own counts."""
    readelf = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-readelf")
    if not os.path.exists(readelf):
        pytest.skip("no llvm-readelf")
    with open(os.path.join(os.path.dirname(hb.__file__), "lib", "hbrocm_gfx950.hsaco"), "rb") as f:
        bundle = f.read()
    code = tmp_path / "code"
    code.write_bytes(bundle[bundle.index(b"\x7fELF"):])
    notes = subprocess.run([readelf, "--notes", str(code)], capture_output=True, text=True, check=True).stdout
    spilled = dict(re.findall(r"\.name: +(hbr_\w+)\n(?:.*\n)*?.*\.vgpr_spill_count: +(\d+)", notes))
    held = {k: int(v) for k, v in spilled.items() if re.match(r"hbr_(rms_norm|pack|unpack|linear_(y|ya|dx|dw|pair))_", k)}
    assert len(held) > 60 and not any(held.values()), {k: v for k, v in held.items() if v}
