"""Plain 64-bit forms of the operators of the layers between leaf vectors and
classes, and the bounds of what a right f32 computation may be off by."""
import numpy as np

from leaf_reference import EPS32, HALF

BLOCK = 32


def codes_of(v):
    """Rows (f64 holding f32 or bf16 values) in 8 bits: (codes, scales), by the
    definition: every code's value, the nearest one, ties to the even code."""
    n, dim = v.shape
    grid = code_values()[:127]  # 0 .. 448, ascending
    codes = np.zeros((n, dim), np.uint8)
    scales = np.zeros((n, -(-dim // BLOCK)), np.uint8)
    for r in range(n):
        for b in range(scales.shape[1]):
            x = v[r, b * BLOCK:(b + 1) * BLOCK]
            fine = np.isfinite(x)
            top = np.max(np.abs(x[fine]), initial=0.0)
            e = -109
            while 448.0 * 2.0 ** e < top:
                e += 1
            scales[r, b] = e + 127
            u = np.abs(np.where(fine, x, 0.0)) / 2.0 ** e
            hi = np.searchsorted(grid, u).clip(0, 126)
            lo = np.maximum(hi - 1, 0)
            up = (u - grid[lo] > grid[hi] - u) | ((u - grid[lo] == grid[hi] - u) & (hi % 2 == 0)) | (grid[lo] == grid[hi])
            at = np.where(up, hi, lo).astype(np.uint8)
            codes[r, b * BLOCK:(b + 1) * BLOCK] = np.where(fine, at | (np.signbit(x).astype(np.uint8) << 7), 0x7F)
    return codes, scales


def code_values():
    """What the 256 codes stand for."""
    c = np.arange(256)
    e, m = c >> 3 & 15, (c & 7).astype(np.float64)
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >> 7, -v, v)


def values_of(codes, scales):
    by = np.repeat(2.0 ** (scales.astype(np.float64) - 127), BLOCK, 1)[:, :codes.shape[1]]
    return code_values()[codes] * by


def roundings(dim):
    """Of a row's sum: a lane's own, and the joins over lanes and waves."""
    return dim // 1024 + 40


def norm(x, residual, weight, eps, dtype):
    """name -> (value, bound): out, total, inv, normed (f32, before 8 bits).
    inv: half the roundings of the squares' sum and of the s in it, and two
    steps of the square root; normed: that, s's own and a product's; out: one
    product and the type's rounding."""
    s = x + (0.0 if residual is None else residual)
    w = np.ones(s.shape[1]) if weight is None else weight
    dim = s.shape[1]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        inv = 1.0 / np.sqrt(np.mean(s * s, 1) + eps)
        rel = (roundings(dim) / 2 + 6) * EPS32
        normed = s * inv[:, None]
        out = normed * w
        tiny = 2.0 ** -149
        return {"total": (s, (EPS32 + HALF[dtype]) * np.abs(s) + tiny), "inv": (inv, rel * inv + tiny),
                "normed": (normed, (rel + 3 * EPS32) * np.abs(normed) + tiny),
                "out": (out, (rel + 4 * EPS32 + HALF[dtype]) * np.abs(out) + 1e-40)}


def norm_grad(dout, rows, inv, weight, dtotal, eps, held, dtype):
    """name -> (value, bound): dx, dweight. rows: as the norm saw them, or
    the normed ones (held)."""
    n, dim = dout.shape
    w = np.ones(dim) if weight is None else weight
    rel = 0.0
    if inv is None:
        inv = 1.0 / np.sqrt(np.mean(rows * rows, 1) + eps)
        rel = (roundings(dim) / 2 + 6) * EPS32
    inv = inv[:, None]
    normed = rows if held else rows * inv
    off = (0.0 if held else rel + EPS32) * np.abs(normed)      # of the normed values
    g = dout * w
    along = np.mean(g * normed, 1, keepdims=True)
    size = np.mean(np.abs(g * normed), 1, keepdims=True)
    along_off = (roundings(dim) + 4) * EPS32 * size + np.mean(np.abs(g) * off, 1, keepdims=True)
    dx = inv * (g - normed * along)
    dx_off = np.abs(inv) * (3 * EPS32 * (np.abs(g) + np.abs(normed * along)) + np.abs(normed) * along_off + off * np.abs(along))
    dx_off += (rel + EPS32) * np.abs(dx)
    if dtotal is not None:
        dx = dx + dtotal
        dx_off += EPS32 * np.abs(dx)
    dx_off += HALF[dtype] * np.abs(dx) + 1e-40
    dweight = np.sum(dout * normed, 0)
    dw_off = (n + 40) * EPS32 * np.sum(np.abs(dout * normed), 0) + np.sum(np.abs(dout) * off, 0) + 1e-40
    return {"dx": (dx, dx_off), "dweight": (dweight, dw_off)}


def product(a, b, dtype):
    """a b with the bound of an f32 sum: a rounding a term (f32 terms, of three
    parts each, eight more), none of the result's type."""
    size = np.abs(a) @ np.abs(b)
    return a @ b, (a.shape[1] + 8) * EPS32 * size


def linear(x, w, bias, down, up, ids, scale, dtype):
    """(out, bound). The adapter's `rank` values have the bound of their sum,
    one more for the scale and in bf16 half a step of bf16; their product with
    `up` a rounding a term and eight more."""
    out, off = product(x, w.T, dtype)
    if bias is not None:
        out = out + bias
        off = off + EPS32 * np.abs(out)
    if down is not None:
        for r, a in enumerate(ids):
            if not 0 <= a < len(down):
                continue
            low, low_off = product(x[r:r + 1], down[a].T, dtype)
            s = 1.0 if scale is None else scale[a]
            low, low_off = low * s, low_off * abs(s) + np.abs(low * s) * (EPS32 + (HALF[dtype] if dtype == "bfloat16" else 0.0))
            more = (low @ up[a].T)[0]
            size = (np.abs(low) @ np.abs(up[a]).T)[0]
            out[r] += more
            off[r] += (low_off @ np.abs(up[a]).T)[0] + (low.shape[1] + 8) * EPS32 * (size + np.abs(out[r]) + np.abs(more))
    return out, off + HALF[dtype] * np.abs(out) + 1e-40


def linear_grad(dout, w, x, weight, dtype):
    """name -> (value, bound): dx, dw, db."""
    got = {}
    if w is not None:
        dx, off = product(dout, w, dtype)
        got["dx"] = (dx, off + HALF[dtype] * np.abs(dx) + 1e-40)
    if x is not None:
        dw, off = product(dout.T, x, dtype)
        by = 1.0 if weight is None else weight
        dw, off = dw * by, off * np.abs(by)
        got["dw"] = (dw, off + (EPS32 + HALF[dtype]) * np.abs(dw) + 1e-40)
    got["db"] = (dout.sum(0), (len(dout) + 8) * EPS32 * np.abs(dout).sum(0) + 1e-40)
    return got
