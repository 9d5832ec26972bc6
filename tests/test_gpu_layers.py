"""The operators of the layers between leaf vectors and classes against their
plain forms in 64 bits, at the sizes, masks and layouts where they can go wrong."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import hessboost_amd as hb
import layer_reference as L
import leaf_reference as R
from hessboost_amd.leafops import DeviceArray
from test_gpu_leafops import back, close, dev, far, far_back, hip, like, ok, work

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16")


def bytes_(values, pad=0, lead=0):
    """Bytes on the device, rows `pad` apart beyond their own; the gaps hold 0xEE."""
    v = np.asarray(values, np.uint8)
    stride = v.shape[1] + pad
    whole = np.full(lead + v.shape[0] * stride, 0xEE, np.uint8)
    for r in range(v.shape[0]):
        whole[lead + r * stride: lead + r * stride + v.shape[1]] = v[r]
    buf = hb.DeviceBuffer(max(16, whole.nbytes))
    if whole.nbytes:
        buf.upload(whole)
    a = DeviceArray(buf, "uint8", v.shape, stride=stride, byte_offset=lead)
    a.lead, a.pad = lead, pad
    return a


def bytes_back(a):
    whole = a.buffer.download(np.uint8, a.buffer.nbytes)
    stride = a.shape[1] + a.pad
    body = whole[a.lead: a.lead + a.shape[0] * stride].reshape(a.shape[0], stride)
    assert np.all(whole[:a.lead] == 0xEE) and np.all(body[:, a.shape[1]:] == 0xEE), "written outside the array"
    return np.ascontiguousarray(body[:, :a.shape[1]])


def packed_like(n, dim, pad=0, lead=0):
    return (bytes_(np.full((n, dim), 0xAA), pad, lead), bytes_(np.full((n, hb.packed_scales(dim)), 0xAA), pad % 3, lead % 5))


def rows(rng, n, dim, dtype, by=1.0):
    v = rng.standard_normal((n, dim)) * np.exp(0.7 * rng.standard_normal((n, 1))) * by
    return R.rounded(np.where(rng.random((n, dim)) < 0.02, 20.0 * v, v), dtype)


def f32(rng, shape, by=1.0, to=0.0):
    return (to + by * rng.standard_normal(shape)).astype(np.float32).astype(np.float64)


# ---- rows in 8 bits -------------------------------------------------------------------

# rows, dim, stride gap, lead
PACKS = [(1, 1, 0, 0), (3, 31, 0, 0), (5, 32, 0, 0), (4, 33, 3, 1), (7, 50, 0, 0), (2, 64, 16, 16), (9, 127, 1, 0), (300, 8, 0, 0),
         (3, 1000, 8, 8), (2, 4100, 4, 4), (1, 70_001, 0, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim, pad, lead", PACKS)
def test_rows_are_packed_to_the_nearest_codes(n, dim, pad, lead, dtype):
    """Bit for bit, and unpacked to just what the codes stand for."""
    rng = np.random.default_rng(dim)
    v = rows(rng, n, dim, dtype, 10.0 ** rng.integers(-30, 30))
    v[rng.random(v.shape) < 0.1] = 0.0
    codes, scales = packed_like(n, dim, pad, lead)
    hb.pack_rows(dev(v, dtype, pad, lead), codes, scales)
    want = L.codes_of(v)
    assert np.array_equal(bytes_back(scales), want[1])
    assert np.array_equal(bytes_back(codes), want[0])
    held = L.values_of(*want)
    for to in DTYPES:
        out = like((n, dim), to, pad, lead)
        hb.unpack_rows(codes, scales, out)
        assert np.array_equal(back(out), held)
    weight = f32(rng, dim)
    out = like((n, dim), dtype, pad, lead)
    hb.unpack_rows(codes, scales, out, weight=dev(weight, "float32"))
    close(back(out), (held * weight, (R.EPS32 + R.HALF[dtype]) * np.abs(held * weight) + 1e-40), "weighted")


def test_packed_borders_and_values_that_are_no_numbers():
    """Every code's value and every tie between two, powers' borders, the
    least power, zeros of both signs, infinities and NaN beside numbers."""
    grid = L.code_values()[:127]
    ties = (grid[1:] + grid[:-1]) / 2
    some = np.concatenate([grid, ties, [np.nextafter(np.float32(448), np.float32(0)), 464.0, 479.0, 480.0, 0.0]])
    some = np.concatenate([some, -some])
    lines = []
    for e in (0, -3, 60, -60, -100, -109, -112, -126, 118):
        for first in (448.0, 1.0, 449.0, 0.0):
            line = np.zeros((-(-len(some) // 31), 32))
            line[:, 0] = first
            line[:, 1:].flat[:len(some)] = some
            lines.append(line * 2.0 ** e)
    v = np.concatenate(lines).astype(np.float32).astype(np.float64)
    v[5, 3], v[5, 4], v[6, 0], v[7] = np.inf, -np.inf, np.nan, np.nan
    v[8] = np.where(np.arange(32) % 2, -0.0, 0.0)
    v = v.reshape(-1, 64) if len(v) % 2 == 0 else v[:-1].reshape(-1, 64)
    codes, scales = packed_like(*v.shape)
    hb.pack_rows(dev(v, "float32"), codes, scales)
    want = L.codes_of(v)
    assert np.array_equal(bytes_back(scales), want[1])
    got = bytes_back(codes)
    nan = ~np.isfinite(v)
    assert np.all((got & 0x7F)[nan] == 0x7F) and np.array_equal(got[~nan], want[0][~nan])


# ---- the norm ----------------------------------------------------------------------------

# rows, dim, residual, weight, stride gap, lead
NORMS = [(1, 1, False, False, 0, 0), (3, 5, True, True, 0, 0), (65, 32, True, False, 0, 0), (1000, 50, False, True, 0, 0),
         (33, 64, True, True, 8, 8), (7, 129, True, True, 1, 1), (5, 512, False, True, 0, 0), (9, 1000, True, True, 2, 2),
         (130, 1024, True, True, 0, 0), (4, 1500, True, False, 4, 0), (3, 2049, False, True, 0, 0), (3, 4096, True, True, 0, 0),
         (2, 5001, True, True, 0, 3), (2, 8200, False, True, 0, 0), (2, 17_000, True, True, 0, 0), (1, 40_000, True, True, 8, 8),
         (2, 33_333, True, True, 1, 0), (40, 310, True, True, 1, 1), (6, 10, True, True, 1, 1), (4, 1022, True, True, 1, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim, residual, weight, pad, lead", NORMS)
def test_norms(n, dim, residual, weight, pad, lead, dtype):
    rng = np.random.default_rng(n * 7 + dim)
    x, eps = rows(rng, n, dim, dtype), np.float32(1e-5)
    r = rows(rng, n, dim, dtype) if residual else None
    w = f32(rng, dim, 0.3, 1.0) if weight else None
    x[-1] = 0.0  # a padded row
    if residual:
        r[-1] = 0.0
    want = L.norm(x, r, w, float(eps), dtype)
    args = dict(weight=None if w is None else dev(w, "float32"), eps=float(eps),
                residual=None if r is None else dev(r, dtype, pad, lead))
    for normed in (False, True):
        out, total, inv = like((n, dim), dtype, pad, lead), like((n, dim), dtype, pad, lead), like(n, "float32")
        codes, scales = packed_like(n, dim, pad, lead)
        hb.rms_norm(dev(x, dtype, pad, lead), out, total=total, inv=inv, codes=codes, scales=scales, normed=normed, **args)
        close(back(out), want["out"], "out")
        close(back(total), want["total"], "total")
        close(back(inv), want["inv"], "inv")
        c, s = bytes_back(codes), bytes_back(scales)
        value, off = want["normed"] if normed else (want["out"][0], want["out"][1] - R.HALF[dtype] * np.abs(want["out"][0]))
        power = np.repeat(2.0 ** (s.astype(np.float64) - 127), 32, 1)[:, :dim]
        close(L.values_of(c, s), (value, 2.0 ** -4 * (np.abs(value) + off) + 2.0 ** -10 * power + off), "held")
        # the power is the least, but for what the values are off by
        top = np.stack([np.max(np.abs(value[:, b:b + 32]), 1) for b in range(0, dim, 32)], 1)
        p = 2.0 ** (s.astype(np.float64) - 127)
        assert np.all(top <= 448 * p * (1 + 1e-3)) and np.all((top > 224 * p * (1 - 1e-3)) | (s == 18))
    # each output by itself, and without codes (another number of lanes)
    out, total, inv = like((n, dim), dtype, pad, lead), like((n, dim), dtype), like(n, "float32")
    hb.rms_norm(dev(x, dtype), out, **args)
    hb.rms_norm(dev(x, dtype), total=total, **args)
    hb.rms_norm(dev(x, dtype), inv=inv, **args)
    close(back(out), want["out"], "out alone")
    close(back(total), want["total"], "total alone")
    close(back(inv), want["inv"], "inv alone")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [50, 1003, 1024, 9001, 40_000, 40_003])
def test_norms_in_place(dim, dtype):
    rng = np.random.default_rng(dim)
    n = 5
    x, r, w = rows(rng, n, dim, dtype), rows(rng, n, dim, dtype), f32(rng, dim)
    want = L.norm(x, r, w, 1e-6, dtype)
    dx, dr = dev(x, dtype), dev(r, dtype)
    hb.rms_norm(dx, dx, weight=dev(w, "float32"), residual=dr, total=dr)
    close(back(dx), want["out"], "out over x")
    close(back(dr), want["total"], "total over the residual")
    dx, dr = dev(x, dtype), dev(r, dtype)
    hb.rms_norm(dx, dr, weight=dev(w, "float32"), residual=dr, total=dx)
    close(back(dr), want["out"], "out over the residual")
    close(back(dx), want["total"], "total over x")


@pytest.mark.parametrize("dim", [3, 300, 20_000])
def test_norms_of_rows_beyond_the_range_of_f32_squares(dim):
    """Squares past f32's range or below it, alone and beside ordinary rows."""
    rng = np.random.default_rng(dim)
    x = f32(rng, (8, dim))
    x[0] *= 1e25
    x[1] *= 1e-30
    x[2] *= 3e36 / np.max(np.abs(x[2]))
    x[4, 0] = 1e22
    x = x.astype(np.float32).astype(np.float64)
    for eps in (0.0, 1e-6):
        want = L.norm(x, None, None, eps, "float32")
        out, inv = like(x.shape, "float32"), like(8, "float32")
        hb.rms_norm(dev(x, "float32"), out, eps=eps, inv=inv)
        # (below 2^-126 inv has steps of 2^-149)
        value, off = want["inv"]
        close(back(inv), (value, off + 2.0 ** -149), "inv")
        value, off = want["out"]
        close(back(out), (value, off + np.abs(x) * 2.0 ** -149), "out")


def test_norms_of_values_that_are_no_numbers_stay_in_their_rows():
    rng = np.random.default_rng(5)
    x = f32(rng, (9, 70))
    clean = L.norm(x, None, None, 1e-6, "float32")["out"]
    x[2, 3], x[5, 69], x[7, 0] = np.inf, np.nan, -np.inf
    out = like(x.shape, "float32")
    codes, scales = packed_like(*x.shape)
    hb.rms_norm(dev(x, "float32"), out, codes=codes, scales=scales)
    got, held = back(out), L.values_of(bytes_back(codes), bytes_back(scales))
    others = [r for r in range(9) if r not in (2, 5, 7)]
    close(got[others], (clean[0][others], clean[1][others]), "the other rows")
    assert np.all(np.isnan(got[5])) and np.all(np.isnan(held[5]))
    for r, c in ((2, 3), (7, 0)):  # 1 / infinity, and infinity times that
        assert np.isnan(got[r, c]) and np.isnan(held[r, c])
        rest = np.arange(70) != c
        assert np.all(got[r, rest] == 0) and np.all(held[r, rest] == 0)


GRADS = [(1, 1, False, False, 0, 0), (3, 5, True, True, 0, 0), (65, 32, True, False, 0, 0), (2000, 50, False, True, 0, 0),
         (33, 64, True, True, 8, 8), (7, 129, True, True, 1, 1), (9, 1000, True, True, 2, 2), (700, 1024, True, True, 0, 0),
         (4, 1500, True, False, 4, 0), (3, 2049, False, True, 0, 0), (3, 4096, True, True, 0, 0), (2, 9000, False, True, 0, 0),
         (3, 40_000, True, True, 8, 8), (1030, 33_333 // 8, True, True, 1, 0),
         (5, 10, True, True, 1, 1), (40, 310, True, True, 1, 1), (2, 8193, True, True, 1, 0), (3, 20_003, True, True, 3, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim, dtotal, weight, pad, lead", GRADS)
def test_norm_gradients(n, dim, dtotal, weight, pad, lead, dtype):
    rng = np.random.default_rng(n + dim)
    x, dout = rows(rng, n, dim, dtype), rows(rng, n, dim, dtype, 1.0 / n)
    t = rows(rng, n, dim, dtype, 1.0 / n) if dtotal else None
    w = f32(rng, dim, 0.3, 1.0) if weight else None
    eps = float(np.float32(1e-5))
    inv = (1.0 / np.sqrt(np.mean(x * x, 1) + eps)).astype(np.float32).astype(np.float64)
    held = L.codes_of(np.asarray(x * inv[:, None], np.float32).astype(np.float64))
    args = dict(weight=None if w is None else dev(w, "float32"), dtotal=None if t is None else dev(t, dtype, pad, lead), eps=eps)
    ways = [("rows", dict(x=dev(x, dtype, pad, lead), inv=dev(inv, "float32")), (x, inv, False)),
            ("rows alone", dict(x=dev(x, dtype, pad, lead)), (x, None, False)),
            ("held", dict(codes=bytes_(held[0], pad, lead), scales=bytes_(held[1]), inv=dev(inv, "float32")),
             (L.values_of(*held), inv, True))]
    ws = work(hb.rms_norm_grad_workspace(n, dim, dtype))
    for name, of, (v, by, is_held) in ways:
        want = L.norm_grad(dout, v, by, w, t, eps, is_held, dtype)
        dx, dweight = like((n, dim), dtype, pad, lead), like(dim, "float32")
        hb.rms_norm_grad(dev(dout, dtype, pad, lead), dx, dweight=dweight, workspace=ws, **of, **args)
        close(back(dx), want["dx"], f"{name}: dx")
        close(back(dweight), want["dweight"], f"{name}: dweight")
        dx = like((n, dim), dtype)
        hb.rms_norm_grad(dev(dout, dtype), dx, **of, **args)
        close(back(dx), want["dx"], f"{name}: dx alone")
    alone = like(dim, "float32")
    hb.rms_norm_grad(dev(dout, dtype), dweight=alone, workspace=ws, **of, **args)
    assert np.array_equal(back(alone), back(dweight))
    # over its inputs
    for over in ("dout", "dtotal"):
        if over == "dtotal" and t is None:
            continue
        g, d = dev(dout, dtype), None if t is None else dev(t, dtype)
        to = g if over == "dout" else d
        hb.rms_norm_grad(g, to, **of, **{**args, "dtotal": d})
        close(back(to), want["dx"], f"dx over {over}")


def test_norm_gradients_agree_with_differences():
    """d/dt of <dout, rms_norm(x + t e)> by central differences in 64 bits."""
    rng = np.random.default_rng(8)
    n, dim, eps = 4, 37, 1e-5
    x, dout, w = f32(rng, (n, dim)), f32(rng, (n, dim)), f32(rng, dim, 0.3, 1.0)
    dx, dweight = like((n, dim), "float32"), like(dim, "float32")
    hb.rms_norm_grad(dev(dout, "float32"), dx, x=dev(x, "float32"), weight=dev(w, "float32"), eps=eps, dweight=dweight,
                     workspace=work(hb.rms_norm_grad_workspace(n, dim, "float32")))

    def loss(x, w):
        return np.sum(dout * x / np.sqrt(np.mean(x * x, 1, keepdims=True) + eps) * w)

    for got, of in ((back(dx), "x"), (back(dweight), "w")):
        for _ in range(10):
            e = rng.standard_normal(got.shape)
            h = 1e-4
            up, down = ((x + h * e, w), (x - h * e, w)) if of == "x" else ((x, w + h * e), (x, w - h * e))
            slope = (loss(*up) - loss(*down)) / (2 * h)
            # differences are off by h^2 (1e-8 of third derivatives below 1e3), the gradient by f32's roundings
            assert abs(np.sum(got * e) - slope) <= 1e-5 * np.sum(np.abs(got * e)) + 1e-5


# ---- projections -----------------------------------------------------------------------------

# rows, dim, outs, rank, adapters, order of ids, bias, scale, stride gap, lead
LINEARS = [
    (1, 1, 1, 0, 0, None, False, False, 0, 0),
    (1, 8, 16, 1, 1, "one", True, True, 0, 0),
    (3, 33, 17, 2, 3, "each", True, False, 0, 0),
    (7, 256, 300, 16, 9, "each", True, True, 0, 0),
    (16, 64, 64, 8, 4, "runs", False, True, 8, 8),
    (17, 70, 130, 5, 3, "mixed", True, True, 1, 1),
    (64, 128, 256, 64, 2, "runs", True, True, 0, 0),
    (65, 40, 129, 7, 70, "each", True, True, 0, 0),
    (130, 96, 257, 16, 200, "each", True, True, 0, 0),
    (200, 512, 96, 33, 5, "mixed", False, True, 8, 0),
    (300, 250, 515, 9, 5, "runs", True, True, 0, 0),
    (257, 1024, 264, 16, 6, "runs", True, True, 0, 0),
    (600, 31, 40, 3, 2, "none", True, True, 0, 0),
    (129, 2048, 128, 0, 0, None, True, False, 0, 0),
    (1100, 64, 1030, 24, 30, "mixed", True, True, 2, 0),
]


def ids_of(rng, n, adapters, order):
    if order == "one":
        return np.zeros(n, np.int32)
    if order == "none":
        return np.where(rng.random(n) < 0.5, -1, adapters + rng.integers(0, 5, n)).astype(np.int32)
    if order == "each":
        return (np.arange(n) * 7 % adapters).astype(np.int32)
    if order == "mixed":
        return rng.integers(-1, adapters + 1, n).astype(np.int32)
    return np.sort(rng.integers(-1, adapters, n)).astype(np.int32)[::-1].copy()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim, outs, rank, adapters, order, bias, scale, pad, lead", LINEARS)
def test_projections(n, dim, outs, rank, adapters, order, bias, scale, pad, lead, dtype):
    rng = np.random.default_rng(n + dim + outs)
    x, w = rows(rng, n, dim, dtype), R.rounded(rng.standard_normal((outs, dim)) / np.sqrt(dim), dtype)
    b = f32(rng, outs) if bias else None
    down = up = ids = s = None
    args = {}
    if rank:
        down = R.rounded(rng.standard_normal((adapters, rank, dim)) / np.sqrt(dim), dtype)
        up = R.rounded(rng.standard_normal((adapters, outs, rank)), dtype)
        ids = ids_of(rng, n, adapters, order)
        s = f32(rng, adapters, 0.5, 1.0) if scale else None
        args = dict(down=dev(down.reshape(-1, dim), dtype, pad, lead), up=dev(up.reshape(-1, rank), dtype, pad, lead),
                    ids=dev(ids, "int32"), scale=None if s is None else dev(s, "float32"))
    out = like((n, outs), dtype, pad, lead)
    hb.linear(dev(x, dtype, pad, lead), dev(w, dtype, pad, lead), out, bias=None if b is None else dev(b, "float32"),
              workspace=work(hb.linear_workspace(n, outs, dim, dtype, rank=rank)), **args)
    close(back(out), L.linear(x, w, b, down, up, ids, s, dtype), "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim, outs, rank", [(12, 64, 80, 8), (200, 40, 300, 16), (200, 40, 300, 5), (1500, 64, 1100, 8), (2100, 64, 2100, 3), (2100, 512, 4100, 8)])
def test_an_adapter_that_is_no_number_is_its_own_rows_alone(n, dim, outs, rank, dtype):
    """Elements of adapters that are infinite or NaN, its rows among others'."""
    rng = np.random.default_rng(rank + n)
    adapters = 5
    x, w = rows(rng, n, dim, dtype), R.rounded(rng.standard_normal((outs, dim)) / np.sqrt(dim), dtype)
    down = R.rounded(rng.standard_normal((adapters, rank, dim)) / np.sqrt(dim), dtype)
    up = R.rounded(rng.standard_normal((adapters, outs, rank)), dtype)
    ids = rng.integers(-1, adapters, n).astype(np.int32)
    value, off = L.linear(x, w, None, down, up, ids, None, dtype)
    for array, of in (("up", 1), ("up", 3), ("down", 2)):
        d, u = down.copy(), up.copy()
        bad = np.zeros((n, outs), bool)
        if array == "up":
            cells = rng.choice(outs, 9, replace=False)
            u[of, cells, rng.integers(0, rank, 9)] = np.array([np.inf, -np.inf, np.nan])[np.arange(9) % 3]
            bad[np.ix_(ids == of, cells)] = True
        else:
            d[of, rank - 1, dim // 2] = np.nan
            bad[ids == of] = True
        out = like((n, outs), dtype)
        hb.linear(dev(x, dtype), dev(w, dtype), out, down=dev(d.reshape(-1, dim), dtype), up=dev(u.reshape(-1, rank), dtype),
                  ids=dev(ids, "int32"), workspace=work(hb.linear_workspace(n, outs, dim, dtype, rank=rank)))
        got = back(out)
        assert not np.any(np.isfinite(got[bad])), array
        close(got[~bad], (value[~bad], off[~bad]), array)


def test_a_row_without_an_adapter_reads_none():
    """NaN adapters that no row has, and NaN rows beside others."""
    rng = np.random.default_rng(3)
    for n in (5, 140):
        x, w = f32(rng, (n, 48)), f32(rng, (70, 48))
        down, up = f32(rng, (3, 4, 48)), f32(rng, (3, 70, 4))
        down[1], up[1] = np.nan, np.nan
        ids = np.where(np.arange(n) % 3 == 0, 0, np.where(np.arange(n) % 3 == 1, -1, 2)).astype(np.int32)
        x[1] = np.nan
        for dtype in DTYPES:
            xs, ws, d, u = (R.rounded(v, dtype) for v in (x, w, down, up))
            out = like((n, 70), dtype)
            hb.linear(dev(xs, dtype), dev(ws, dtype), out, down=dev(d.reshape(-1, 48), dtype), up=dev(u.reshape(-1, 4), dtype),
                      ids=dev(ids, "int32"), workspace=work(hb.linear_workspace(n, 70, 48, dtype, rank=4)))
            got = back(out)
            assert np.all(np.isnan(got[1]))
            xs[1], d[1], u[1] = 0.0, 0.0, 0.0
            value, off = L.linear(xs, ws, None, d, u, ids, None, dtype)
            keep = np.arange(n) != 1
            close(got[keep], (value[keep], off[keep]), dtype)


def test_infinite_inputs_of_a_projection():
    """An infinity reaches its row's outputs as f32 arithmetic says."""
    rng = np.random.default_rng(4)
    for n in (3, 150):
        x, w = f32(rng, (n, 40)), f32(rng, (66, 40))
        x[2, 7] = np.inf
        w[5, 7] = 0.0
        for dtype in DTYPES:
            xs, ws = R.rounded(x, dtype), R.rounded(w, dtype)
            out = like((n, 66), dtype)
            hb.linear(dev(xs, dtype), dev(ws, dtype), out, workspace=work(hb.linear_workspace(n, 66, 40, dtype)))
            got = back(out)
            assert np.isnan(got[2, 5])
            rest = np.arange(66) != 5
            assert np.array_equal(got[2, rest], np.where(ws[rest, 7] > 0, np.inf, -np.inf))
            xs[2] = 0.0
            value, off = L.linear(xs, ws, None, None, None, None, None, dtype)
            keep = np.arange(n) != 2
            close(got[keep], (value[keep], off[keep]), dtype)


# rows, dim, outs, weight, stride gap, lead
LINEAR_GRADS = [(1, 1, 1, False, 0, 0), (1, 64, 40, True, 0, 0), (5, 33, 17, True, 0, 0), (64, 32, 8, False, 0, 0), (100, 50, 70, True, 1, 1),
                (130, 256, 136, True, 8, 8), (1000, 64, 64, True, 0, 0), (515, 250, 333, False, 0, 0), (2000, 96, 300, True, 0, 0),
                (300, 1032, 520, True, 8, 0), (3001, 40, 24, True, 0, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim, outs, weight, pad, lead", LINEAR_GRADS)
def test_projection_gradients(n, dim, outs, weight, pad, lead, dtype):
    rng = np.random.default_rng(n + dim + outs)
    x, dout, w = rows(rng, n, dim, dtype), rows(rng, n, outs, dtype, 1.0 / n), rows(rng, outs, dim, dtype)
    by = f32(rng, dim, 0.3, 1.0) if weight else None
    held = L.codes_of(x)
    ws = work(hb.linear_grad_workspace(n, outs, dim, dtype))
    weights = None if by is None else dev(by, "float32")
    for name, of, v in (("rows", dict(x=dev(x, dtype, pad, lead)), x),
                        ("held", dict(codes=bytes_(held[0], pad, lead), scales=bytes_(held[1], pad % 3)), L.values_of(*held))):
        want = L.linear_grad(dout, w, v, by, dtype)
        got = dict(dx=like((n, dim), dtype, pad, lead), dw=like((outs, dim), dtype, pad, lead), db=like(outs, "float32"))
        hb.linear_grad(dev(dout, dtype, pad, lead), dev(w, dtype, pad, lead), weight=weights, workspace=ws, **of, **got)
        whole = {k: back(a) for k, a in got.items()}
        for k in got:
            close(whole[k], want[k], f"{name}: {k}")
    # each by itself
    g = dev(dout, dtype)
    dx, dw, db = like((n, dim), dtype), like((outs, dim), dtype), like(outs, "float32")
    hb.linear_grad(g, dev(w, dtype), dx=dx, workspace=ws)
    hb.linear_grad(g, weight=weights, dw=dw, workspace=ws, **of)
    hb.linear_grad(g, dev(w, dtype), db=db, workspace=ws)
    close(back(dx), want["dx"], "dx alone")
    close(back(dw), want["dw"], "dw alone")
    close(back(db), want["db"], "db alone")


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dtype):
    """Nothing is written but the gradients' sums, which are zeros."""
    none, dim, outs = np.zeros((0, 40)), 40, 24
    codes, scales = packed_like(0, dim)
    hb.pack_rows(dev(none, dtype), codes, scales)
    hb.unpack_rows(codes, scales, dev(none, dtype))
    hb.rms_norm(dev(none, dtype), dev(none, dtype))
    dweight, dw, db = like(dim, "float32"), like((outs, dim), dtype), like(outs, "float32")
    hb.rms_norm_grad(dev(none, dtype), dev(none, dtype), x=dev(none, dtype), dweight=dweight,
                     workspace=work(hb.rms_norm_grad_workspace(0, dim, dtype)))
    w, out = dev(np.ones((outs, dim)), dtype), dev(np.zeros((0, outs)), dtype)
    hb.linear(dev(none, dtype), w, out, workspace=work(hb.linear_workspace(0, outs, dim, dtype)))
    hb.linear_grad(out, w, x=dev(none, dtype), dx=dev(none, dtype), dw=dw, db=db,
                   workspace=work(hb.linear_grad_workspace(0, outs, dim, dtype)))
    for a in (dweight, dw, db):
        assert np.all(back(a) == 0)


# ---- arrays of more than 4 GiB, and other places ------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_over_more_than_4_gib(dtype):
    """Rows far apart: 8 of them 2 GiB or so, and 70 of them 128 MiB."""
    rng = np.random.default_rng(9)
    size = 2 if dtype == "bfloat16" else 4
    for n, dim, gap in ((8, 40, (1 << 30) // size + 16), (70, 200, (1 << 27) // size + 8)):
        x, r, w = rows(rng, n, dim, dtype), rows(rng, n, dim, dtype), rows(rng, 24, dim, dtype)
        want = L.norm(x, r, None, 1e-6, dtype)
        held = far(n, dim, dtype, gap, x)
        out = like((n, dim), dtype)
        hb.rms_norm(held, out, residual=dev(r, dtype))
        close(back(out), want["out"], "x far")
        codes, scales = packed_like(n, dim)
        hb.pack_rows(held, codes, scales)
        assert np.array_equal(bytes_back(codes), L.codes_of(x)[0])
        dout = rows(rng, n, dim, dtype)
        dx = like((n, dim), dtype)
        hb.rms_norm_grad(dev(dout, dtype), dx, x=held)
        close(back(dx), L.norm_grad(dout, x, None, None, None, 1e-6, False, dtype)["dx"], "x of the gradient far")
        g = rows(rng, n, 24, dtype)
        y = like((n, 24), dtype)
        hb.linear(held, dev(w, dtype), y, workspace=work(hb.linear_workspace(n, 24, dim, dtype)))
        close(back(y), L.linear(x, w, None, None, None, None, None, dtype), "x of a projection far")
        dw = like((24, dim), dtype)
        hb.linear_grad(dev(g, dtype), x=held, dw=dw, workspace=work(hb.linear_grad_workspace(n, 24, dim, dtype)))
        close(back(dw), L.linear_grad(g, None, x, None, dtype)["dw"], "x of dw far")
        del held
        for call, value in ((lambda a: hb.rms_norm(dev(x, dtype), a, residual=dev(r, dtype)), want["out"]),
                            (lambda a: hb.unpack_rows(codes, scales, a), (L.values_of(*L.codes_of(x)), 1e-40 + 0 * x)),
                            (lambda a: hb.linear_grad(dev(g, dtype), dev(w, dtype), dx=a, workspace=work(hb.linear_grad_workspace(n, 24, dim, dtype))),
                             L.linear_grad(g, w, None, None, dtype)["dx"])):
            a = far(n, dim, dtype, gap)
            call(a)
            close(far_back(a), value, "an output far")
            del a


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(dtype):
    """More rows than a launch has workgroups, tiles of several rounds, shares
    of long sums: against sums in 64 bits of what the operators were given."""
    rng = np.random.default_rng(12)
    n, dim, outs = 70_001, 40, 72
    x, w = rows(rng, n, dim, dtype), rows(rng, outs, dim, dtype, 0.2)
    out, codes, scales = like((n, dim), dtype), *packed_like(n, dim)
    inv = like(n, "float32")
    hb.rms_norm(dev(x, dtype), out, inv=inv, codes=codes, scales=scales, normed=True)
    want = L.norm(x, None, None, 1e-6, dtype)
    close(back(out), want["out"], "out")
    dout = rows(rng, n, dim, dtype, 1.0 / n)
    v = L.values_of(bytes_back(codes), bytes_back(scales))
    by = back(inv)
    dx, dweight = like((n, dim), dtype), like(dim, "float32")
    hb.rms_norm_grad(dev(dout, dtype), dx, codes=codes, scales=scales, inv=inv, dweight=dweight,
                     workspace=work(hb.rms_norm_grad_workspace(n, dim, dtype)))
    want = L.norm_grad(dout, v, by, None, None, 0.0, True, dtype)
    close(back(dx), want["dx"], "dx")
    close(back(dweight), want["dweight"], "dweight")
    ids = ids_of(rng, n, 5, "runs")
    down, up = rows(rng, 5 * 8, dim, dtype, 0.2), rows(rng, 5 * outs, 8, dtype)
    y = like((n, outs), dtype)
    hb.linear(dev(x, dtype), dev(w, dtype), y, down=dev(down, dtype), up=dev(up, dtype), ids=dev(ids, "int32"),
              workspace=work(hb.linear_workspace(n, outs, dim, dtype, rank=8)))
    got = back(y)
    some = np.unique(np.r_[0:300, n - 300:n, rng.integers(0, n, 500)])
    value, off = L.linear(x[some], w, None, down.reshape(5, 8, dim), up.reshape(5, outs, 8), ids[some], None, dtype)
    close(got[some], (value, off), "y")
    g = rows(rng, n, outs, dtype, 1.0 / n)
    dw, db, dx = like((outs, dim), dtype), like(outs, "float32"), like((n, dim), dtype)
    hb.linear_grad(dev(g, dtype), dev(w, dtype), codes=codes, scales=scales, dw=dw, db=db, dx=dx,
                   workspace=work(hb.linear_grad_workspace(n, outs, dim, dtype)))
    want = L.linear_grad(g, w, v, None, dtype)
    for name, a in (("dw", dw), ("db", db), ("dx", dx)):
        close(back(a), want[name], name)


@pytest.mark.parametrize("n, dim, outs", [(600, 256, 2560), (1500, 2000, 300), (5000, 520, 1030), (130, 70, 9000), (16_500, 64, 1024),
                                          (8191, 1000, 4096), (8191, 4096, 1000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_projections_of_large_and_small_tiles(n, dim, outs, dtype):
    """Sizes at which a product has tiles of either size, several a workgroup,
    or shares of its steps: a sample of the cells, in 64 bits."""
    rng = np.random.default_rng(n + outs)
    x, w, g = rows(rng, n, dim, dtype), rows(rng, outs, dim, dtype, 0.1), rows(rng, n, outs, dtype, 1.0 / n)
    b = f32(rng, outs)
    y, dx, dw, db = like((n, outs), dtype), like((n, dim), dtype), like((outs, dim), dtype), like(outs, "float32")
    hb.linear(dev(x, dtype), dev(w, dtype), y, bias=dev(b, "float32"), workspace=work(hb.linear_workspace(n, outs, dim, dtype)))
    hb.linear_grad(dev(g, dtype), dev(w, dtype), x=dev(x, dtype), dx=dx, dw=dw, db=db, workspace=work(hb.linear_grad_workspace(n, outs, dim, dtype)))
    some = np.unique(np.r_[0, n - 1, rng.integers(0, n, 40)])
    value, off = L.linear(x[some], w, b, None, None, None, None, dtype)
    close(back(y)[some], (value, off), "y")
    value, off = L.linear_grad(g[some], w, None, None, dtype)["dx"]
    close(back(dx)[some], (value, off), "dx")
    few = np.unique(np.r_[0, outs - 1, rng.integers(0, outs, 40)])
    want = L.linear_grad(np.ascontiguousarray(g[:, few]), None, x, None, dtype)
    close(back(dw)[few], want["dw"], "dw")
    close(back(db), L.linear_grad(g, None, None, None, dtype)["db"], "db")


# ---- a training step of all of them ----------------------------------------------------------


class Layers:
    """One step of a model on leaves with a layer in its middle: look-up, norm
    with its checkpoint, projection, head, and all gradients back to the table."""

    def __init__(self, dtype, seed, n=500, columns=6, table=31, dim=40, outs=72, classes=130):
        rng = np.random.default_rng(seed)
        self.dtype, self.n = dtype, n
        self.v = dict(ids=rng.integers(0, table, (n, columns)).astype(np.int32), off=(np.arange(columns) * table).astype(np.int32),
                      table=rows(rng, table * columns, dim, dtype, 0.3), residual=rows(rng, n, dim, dtype), weight=f32(rng, dim, 0.2, 1.0),
                      w=rows(rng, outs, dim, dtype, 0.15), bias=f32(rng, outs, 0.1), head=rows(rng, classes, outs, dtype, 0.2),
                      y=rng.integers(-1, classes, n).astype(np.int32))
        kinds = dict(ids="int32", off="int32", y="int32", weight="float32", bias="float32")
        self.inputs = {k: dev(a, kinds.get(k, dtype)) for k, a in self.v.items()}
        new = lambda *s: like(s, dtype)
        self.h, self.total, self.out, self.z = new(n, dim), new(n, dim), new(n, dim), new(n, outs)
        self.inv, self.loss = like(n, "float32"), like(n, "float32")
        self.codes, self.scales = packed_like(n, dim)
        self.dz, self.dhead, self.dout, self.dw, self.dh, self.dtable = new(n, outs), new(classes, outs), new(n, dim), new(outs, dim), new(n, dim), new(table * columns, dim)
        self.db, self.dweight, self.norm = like(outs, "float32"), like(dim, "float32"), like(1, "float32")
        self.ws = [work(b) for b in (hb.linear_workspace(n, outs, dim, dtype), hb.softmax_head_workspace(n, classes, outs, dtype),
                                     hb.linear_grad_workspace(n, outs, dim, dtype), hb.rms_norm_grad_workspace(n, dim, dtype),
                                     hb.leaf_embedding_grad_workspace(n, columns, table * columns, dim, dtype), hb.clip_gradients_workspace(5))]

    def run(self, stream=None):
        i, kw = self.inputs, dict(stream=stream)
        hb.leaf_embedding(i["table"], i["ids"], self.h, offset=i["off"], **kw)
        hb.rms_norm(self.h, self.out, weight=i["weight"], residual=i["residual"], total=self.total, inv=self.inv, codes=self.codes,
                    scales=self.scales, normed=True, **kw)
        hb.linear(self.out, i["w"], self.z, bias=i["bias"], workspace=self.ws[0], **kw)
        hb.softmax_head(self.z, i["head"], labels=i["y"], loss=self.loss, dh=self.dz, dw=self.dhead, grad_scale=1.0 / self.n,
                        workspace=self.ws[1], **kw)
        hb.linear_grad(self.dz, i["w"], codes=self.codes, scales=self.scales, weight=i["weight"], dx=self.dout, dw=self.dw, db=self.db,
                       workspace=self.ws[2], **kw)
        hb.rms_norm_grad(self.dout, self.dh, codes=self.codes, scales=self.scales, inv=self.inv, weight=i["weight"], dweight=self.dweight,
                         workspace=self.ws[3], **kw)
        hb.leaf_embedding_grad(self.dh, i["ids"], self.dtable, offset=i["off"], workspace=self.ws[4], **kw)
        hb.clip_gradients([self.dtable, self.dw, self.db, self.dweight, self.dhead], 0.01, norm=self.norm, workspace=self.ws[5], **kw)

    def outputs(self):
        return [back(a) for a in (self.total, self.z, self.loss, self.dw, self.db, self.dweight, self.dhead, self.dtable, self.norm)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_of_layers_runs_through_all_of_them(dtype):
    """Every call against its plain form on what the call before it gave."""
    s = Layers(dtype, 3)
    s.run()
    v = s.v
    h = back(s.h)
    close(h, R.embedding(v["table"], v["ids"], v["off"], None, dtype), "h")
    want = L.norm(h, v["residual"], v["weight"], float(np.float32(1e-6)), dtype)
    for name, a in (("out", s.out), ("total", s.total), ("inv", s.inv)):
        close(back(a), want[name], name)
    close(back(s.z), L.linear(back(s.out), v["w"], v["bias"], None, None, None, None, dtype), "z")
    want = R.head(back(s.z), v["head"], None, v["y"], None, float(np.float32(1 / s.n)), dtype)
    close(back(s.loss), want["loss"], "loss")
    close(back(s.dz), want["dh"], "dz")
    held = L.values_of(bytes_back(s.codes), bytes_back(s.scales))
    want = L.linear_grad(back(s.dz), v["w"], held, v["weight"], dtype)
    close(back(s.dout), want["dx"], "dout")
    last = L.norm_grad(back(s.dout), held, back(s.inv), v["weight"], None, 0.0, True, dtype)
    close(back(s.dh), last["dx"], "dh")
    table = R.embedding_grad(back(s.dh), v["ids"], v["off"], None, len(v["table"]), dtype)
    full = [table, want["dw"], want["db"], last["dweight"], R.head(back(s.z), v["head"], None, v["y"], None, float(np.float32(1 / s.n)), dtype)["dw"]]
    true = np.sqrt(sum(np.sum(a * a) for a, _ in full))
    slack = np.sqrt(sum(np.sum(e * e) for _, e in full))
    assert true > 0.01 and abs(back(s.norm)[0] - true) <= slack + 2 * R.EPS32 * true
    by = 0.01 / (true + 1e-6)
    for a, (x, e), t in zip((s.dtable, s.dw, s.db, s.dweight, s.dhead), full, (dtype, dtype, "float32", "float32", dtype)):
        close(back(a), (x * by, (e + np.abs(x) * (slack / true + 6 * R.EPS32)) * by * 1.01 + R.HALF[t] * 1.01 * (np.abs(x) + e) * by + 1e-38))


def test_layers_on_several_streams_give_the_same_bits():
    H = hip()
    sizes = [("bfloat16", 21, {}), ("bfloat16", 22, dict(n=900, dim=264, outs=300)), ("float32", 23, {}), ("float32", 24, dict(n=30, dim=33, outs=17))]
    want = []
    for dtype, seed, kw in sizes:
        s = Layers(dtype, seed, **kw)
        s.run()
        want.append(s.outputs())
    again, streams = [Layers(dtype, seed, **kw) for dtype, seed, kw in sizes], []
    for _ in again:
        st = C.c_void_p()
        ok(H.hipStreamCreateWithFlags(C.byref(st), 1))
        streams.append(st)
    for _ in range(3):
        for s, st in zip(again, streams):
            s.run(st.value)
    ok(H.hipDeviceSynchronize())
    for s, w in zip(again, want):
        for a, b in zip(s.outputs(), w):
            assert np.array_equal(a, b)
    for st in streams:
        ok(H.hipStreamDestroy(st))


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_layers_replay_with_the_eager_bits(dtype):
    """Captured once; replayed on other inputs with eager work between."""
    H = hip()
    st = C.c_void_p()
    ok(H.hipStreamCreateWithFlags(C.byref(st), 1))
    s, other = Layers(dtype, 31), Layers(dtype, 32)
    other.run()
    ok(H.hipStreamBeginCapture(st, 2))
    s.run(st.value)
    graph, run = C.c_void_p(), C.c_void_p()
    ok(H.hipStreamEndCapture(st, C.byref(graph)))
    ok(H.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
    for seed in (31, 41, 42, 31):
        t = Layers(dtype, seed)
        for k, a in s.inputs.items():
            a.buffer.copy_from(t.inputs[k].buffer)
        ok(H.hipDeviceSynchronize())
        ok(H.hipGraphLaunch(run, st))
        ok(H.hipStreamSynchronize(st))
        got = s.outputs()
        t.run()
        for a, b in zip(got, t.outputs()):
            assert np.array_equal(a, b)
        other.run()
    ok(H.hipGraphExecDestroy(run))
    ok(H.hipGraphDestroy(graph))
    ok(H.hipStreamDestroy(st))


TORCH = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import hessboost_amd as hb

torch.manual_seed(0)
n, dim, outs, rank, adapters = 300, 96, 200, 8, 5
for dtype in (torch.float32, torch.bfloat16):
    r = lambda *s: torch.randn(*s, device="cuda").to(dtype)
    x, res, w, dout = r(n, dim), r(n, dim), r(outs, dim), r(n, outs)
    weight, bias, scale = torch.rand(dim, device="cuda") + 0.5, torch.randn(outs, device="cuda"), torch.rand(adapters, device="cuda")
    down, up = r(adapters, rank, dim), r(adapters, outs, rank)
    ids = torch.randint(-1, adapters, (n,), device="cuda", dtype=torch.int32)
    names = ("out", "total", "y", "dx", "dw", "db", "dres", "dweight", "held")

    def step():
        got = dict(out=torch.empty_like(x), total=torch.empty_like(x), y=torch.empty(n, outs, device="cuda", dtype=dtype), dx=torch.empty_like(x),
                   dw=torch.empty_like(w), db=torch.empty(outs, device="cuda"), dres=torch.empty_like(x), dweight=torch.empty_like(weight),
                   held=torch.empty(n, dim, device="cuda", dtype=torch.bfloat16))
        inv = torch.empty(n, device="cuda")
        codes = torch.empty(n, dim, device="cuda", dtype=torch.float8_e4m3fn)
        scales = torch.empty(n, hb.packed_scales(dim), device="cuda", dtype=torch.uint8)
        ws = lambda b: torch.empty(max(16, b), dtype=torch.uint8, device="cuda")
        hb.rms_norm(x, got["out"], weight=weight, residual=res, total=got["total"], inv=inv, codes=codes, scales=scales, normed=True)
        hb.unpack_rows(codes, scales, got["held"])
        hb.linear(got["out"], w, got["y"], bias=bias, down=down, up=up, ids=ids, scale=scale, workspace=ws(hb.linear_workspace(n, outs, dim, dtype, rank=rank)))
        hb.linear_grad(dout, w, codes=codes.view(torch.uint8), scales=scales, weight=weight, dx=got["dx"], dw=got["dw"], db=got["db"],
                       workspace=ws(hb.linear_grad_workspace(n, outs, dim, dtype)))
        hb.rms_norm_grad(got["dx"], got["dres"], codes=codes, scales=scales, inv=inv, weight=weight, dtotal=res, dweight=got["dweight"],
                         workspace=ws(hb.rms_norm_grad_workspace(n, dim, dtype)))
        return got

    eager = step()
    torch.cuda.synchronize()
    t = (x.double() + res.double())
    nn = t * (t.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    assert (eager["out"].double() - nn * weight.double()).abs().max() < 0.05
    assert ((eager["held"].double() - nn).abs() <= nn.abs() / 16 + 0.01).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the tensors' stream by default: torch's current one
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(there[k], eager[k]) for k in names)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for seed in range(3):
        for a in (x, res, dout, down):
            a.copy_(r(*a.shape))
        graph.replay()
        torch.cuda.synchronize()
        mine = step()
        torch.cuda.synchronize()
        assert all(torch.equal(kept[k], mine[k]) for k in names), seed
    # rows of views, and adapters whose rows lie apart
    wide = torch.full((n, 2 * outs), float("nan"), device="cuda", dtype=dtype)
    spread = torch.zeros(adapters, rank, 2 * dim, device="cuda", dtype=dtype)
    spread[:, :, :dim] = down
    hb.linear(kept["out"], w, wide[:, :outs], bias=bias, down=spread[:, :, :dim], up=up, ids=ids, scale=scale,
              workspace=torch.empty(hb.linear_workspace(n, outs, dim, dtype, rank=rank), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(wide[:, :outs], kept["y"]) and torch.isnan(wide[:, outs:]).all()
    try:
        hb.linear(x, w, kept["y"], down=down.transpose(0, 1).contiguous().transpose(0, 1), up=up, ids=ids)
        raise SystemExit("adapters of two strides were taken")
    except ValueError:
        pass
print("torch layers ok", flush=True)
"""


def test_torch_tensors_of_layers_are_taken_on_their_stream():
    """In a process of its own: torch brings its own HIP runtime."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = TORCH.replace("{root!r}", repr(os.path.dirname(here))).replace("{tests!r}", repr(here))
    r = subprocess.run([sys.executable, "-u", "-c", code], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "torch layers ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("n, dim, outs, rank", [(1, 64, 80, 8), (12, 64, 80, 8), (40, 200, 96, 4), (200, 64, 300, 16), (200, 40, 300, 6), (300, 2048, 130, 8),
                                                (1500, 64, 1100, 8), (2100, 64, 2100, 32), (2100, 512, 4100, 8)])
def test_the_low_values_of_adapters_are_f32_sums_for_any_number_of_rows(n, dim, outs, rank):
    """Ranks in pairs that take each other off but for their last bits: in
    bfloat16 the outputs are those of float32 low values, rounded once."""
    rng = np.random.default_rng(n + rank)
    adapters = 3
    x = rows(rng, n, dim, "bfloat16")
    down = R.rounded(rng.standard_normal((adapters, rank, dim)) / np.sqrt(dim), "bfloat16")
    down[:, 1::2] = R.rounded(down[:, ::2] * (1 + 2.0 ** -7 * rng.integers(-1, 2, down[:, ::2].shape)), "bfloat16")
    up = R.rounded(rng.standard_normal((adapters, outs, rank)), "bfloat16")
    up[:, :, 1::2] = -up[:, :, ::2]
    ids, scale = rng.integers(-1, adapters, n).astype(np.int32), f32(rng, adapters, 0.5, 1.0)
    ids[0] = 1
    out = like((n, outs), "bfloat16")
    hb.linear(dev(x, "bfloat16"), dev(np.zeros((outs, dim)), "bfloat16"), out, down=dev(down.reshape(-1, dim), "bfloat16"),
              up=dev(up.reshape(-1, rank), "bfloat16"), ids=dev(ids, "int32"), scale=dev(scale, "float32"),
              workspace=work(hb.linear_workspace(n, outs, dim, "bfloat16", rank=rank)))
    value, off = L.linear(x, np.zeros((outs, dim)), None, down, up, ids, scale, "float32")
    close(back(out), (value, off + R.HALF["bfloat16"] * (np.abs(value) + off)), "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim, outs, rank", [(12, 64, 80, 8), (200, 40, 300, 16), (200, 40, 300, 5), (300, 2048, 130, 8), (1500, 64, 1100, 8),
                                                (2100, 64, 2100, 3), (2100, 512, 4100, 8)])
def test_infinite_adapters_give_what_their_formula_does(n, dim, outs, rank, dtype):
    """Infinities of either sign and NaN in either factor and in the scales, for
    low values of either sign, zeros and infinities among them: the same outputs
    for any number of rows, infinite with their sign or no numbers. All is whole
    numbers, so that no low value's sign is a matter of roundings."""
    rng = np.random.default_rng(rank + n)
    adapters = 4
    x, w = rng.integers(-2, 3, (n, dim)).astype(float), rng.integers(-1, 2, (outs, dim)).astype(float)
    x[::7] = 0.0
    down, up = rng.integers(-1, 2, (adapters, rank, dim)).astype(float), rng.integers(-2, 3, (adapters, outs, rank)).astype(float)
    ids, scale = rng.integers(-1, adapters, n).astype(np.int32), np.array([1.0, -2.0, 0.5, 1.0])
    ids[:4] = 0, 1, 2, 3
    off = L.linear(x, w, None, down, up, ids, scale, dtype)[1]
    cells = rng.permutation(outs)[:18].reshape(2, 9)
    for a in (0, 1):
        up[a, cells[a], rng.integers(0, rank, 9)] = np.array([np.inf, -np.inf, np.inf, -np.inf, np.nan, np.inf, -np.inf, np.inf, -np.inf])
        up[a, cells[a][:3], rng.integers(0, rank, 3)] = np.inf  # two of a sum, of one sign or of both
    down[1, 0, dim // 2], scale[3] = -np.inf, np.inf
    out = like((n, outs), dtype)
    hb.linear(dev(x, dtype), dev(w, dtype), out, down=dev(down.reshape(-1, dim), dtype), up=dev(up.reshape(-1, rank), dtype), ids=dev(ids, "int32"),
              scale=dev(scale, "float32"), workspace=work(hb.linear_workspace(n, outs, dim, dtype, rank=rank)))
    got, want = back(out), x @ w.T
    with np.errstate(invalid="ignore"):
        for r in np.flatnonzero(ids >= 0):
            low = np.sum(x[r] * down[ids[r]], 1) * scale[ids[r]]
            want[r] += np.sum(low * up[ids[r]], 1)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    some = np.isinf(want)
    assert np.array_equal(got[some], want[some]) and np.any(want[some] > 0) and np.any(want[some] < 0)
    rest = np.isfinite(want)
    close(got[rest], (want[rest], off[rest]), "finite outputs")


@pytest.mark.parametrize("n", [10, 130, 2000])
def test_low_values_past_bfloat16_stay_finite(n):
    """A low value of more than bfloat16's largest, and less than float32's."""
    outs, dim = 1100, 64
    x, down, up = np.ones((n, dim)), np.zeros((1, 1, dim)), np.full((1, outs, 1), 2.0 ** -20)
    down[0, 0, 0] = 1.0
    out = like((n, outs), "bfloat16")
    scale = float(np.float32(3.4e38))
    hb.linear(dev(x, "bfloat16"), dev(np.zeros((outs, dim)), "bfloat16"), out, down=dev(down[0], "bfloat16"), up=dev(up[0], "bfloat16"),
              ids=dev(np.zeros(n), "int32"), scale=dev(np.array([scale]), "float32"), workspace=work(hb.linear_workspace(n, outs, dim, "bfloat16", rank=1)))
    value = np.full((n, outs), scale * 2.0 ** -20)
    close(back(out), (value, (R.HALF["bfloat16"] + 10 * R.EPS32) * value), "out")


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_without_adapters_need_no_workspace(dtype):
    rng = np.random.default_rng(6)
    for n, dim, outs in ((1, 1024, 700), (16, 96, 33), (64, 72, 64)):
        x, w = rows(rng, n, dim, dtype), rows(rng, outs, dim, dtype, 0.2)
        out = like((n, outs), dtype)
        hb.linear(dev(x, dtype), dev(w, dtype), out)
        close(back(out), L.linear(x, w, None, None, None, None, None, dtype), "out")


# rows, dim: either side of what rows of 8 bytes are taken by, and of what a
# workgroup's registers hold, by vectors of 8 bytes and of 16
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, dim", [(5, 2), (70, 126), (33, 130), (9, 258), (7, 510), (5, 514), (300, 514), (5, 600), (3, 1018), (3, 1026), (5, 2046),
                                    (5, 2050), (3, 4094), (3, 4098), (300, 4098), (4, 6002), (3, 8190), (3, 8194), (2, 16_382), (2, 16_386)])
def test_norms_of_every_width(n, dim, dtype):
    """And their gradients, from the rows and from 8 bits, in views too."""
    rng = np.random.default_rng(n + dim)
    x, r, dout, w = rows(rng, n, dim, dtype), rows(rng, n, dim, dtype), rows(rng, n, dim, dtype, 1.0 / n), f32(rng, dim, 0.3, 1.0)
    eps, weight = float(np.float32(1e-5)), dev(w, "float32")
    for pad, lead in ((0, 0), (3, 1)):
        want = L.norm(x, r, w, eps, dtype)
        out, total, inv, (codes, scales) = like((n, dim), dtype, pad, lead), like((n, dim), dtype, pad, lead), like(n, "float32"), packed_like(n, dim, pad, lead)
        hb.rms_norm(dev(x, dtype, pad, lead), out, weight=weight, eps=eps, residual=dev(r, dtype, pad, lead), total=total, inv=inv, codes=codes,
                    scales=scales, normed=True)
        close(back(out), want["out"], "out")
        close(back(total), want["total"], "total")
        close(back(inv), want["inv"], "inv")
        held, by = L.values_of(bytes_back(codes), bytes_back(scales)), back(inv)
        value, off = want["normed"]
        power = np.repeat(2.0 ** (bytes_back(scales).astype(np.float64) - 127), 32, 1)[:, :dim]
        close(held, (value, 2.0 ** -4 * (np.abs(value) + off) + 2.0 ** -10 * power + off), "held")
        ws = work(hb.rms_norm_grad_workspace(n, dim, dtype))
        for of, args in (((x, None, False), dict(x=dev(x, dtype, pad, lead))), ((held, by, True), dict(codes=codes, scales=scales, inv=inv))):
            want = L.norm_grad(dout, of[0], of[1], w, r, eps, of[2], dtype)
            dx, dweight = like((n, dim), dtype, pad, lead), like(dim, "float32")
            hb.rms_norm_grad(dev(dout, dtype, pad, lead), dx, weight=weight, eps=eps, dtotal=dev(r, dtype, pad, lead), dweight=dweight, workspace=ws, **args)
            close(back(dx), want["dx"], "dx")
            close(back(dweight), want["dweight"], "dweight")
