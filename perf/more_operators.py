"""Operators of the layers between leaf vectors and classes, as measurable cases.

A row's leaf vectors are summed (`leaf_embedding`) and scored against every
class (`softmax_head`). Between the two a model normalises the sums and
projects them, keeps what its backward pass reads in 8 bits, and serves many
customers by low-rank adapters beside one projection. Kinds (`case["kind"]`):

- "norm": root-mean-square norm of rows, the residual added first, its result
  in the rows' type and, for the backward pass, the normalised rows in 8 bits;
- "norm_grad": its gradient, from the rows or from the normalised rows in 8 bits;
- "pack": rows to 8 bits and back;
- "linear": a projection of rows, each with its request's low-rank adapter;
- "linear_grad": the projection's gradients, its inputs held in 8 bits or not.

Rows in 8 bits are e4m3 codes, 32 columns of a row sharing a power of two: the
smallest (and at least 2^-109) under which none of the 32 is above 448. The
powers' exponents lie in bytes, 127 more than they are.
"""
import math

import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5
_BLOCK = 32


def _norm(name, n, dim, dtype, residual, held=False):
    """held: the normalised rows in 8 bits too, and the rows' factors."""
    return dict(name=name, kind="norm", n=n, dim=dim, dtype=dtype, residual=residual, held=held)


def _norm_grad(name, n, dim, dtype, held, residual):
    return dict(name=name, kind="norm_grad", n=n, dim=dim, dtype=dtype, held=held, residual=residual)


def _pack(name, n, dim, dtype):
    return dict(name=name, kind="pack", n=n, dim=dim, dtype=dtype)


def _linear(name, n, dim, out, rank, adapters, requests, dtype):
    """requests: runs of rows that share an adapter (some have none)."""
    return dict(name=name, kind="linear", n=n, dim=dim, out=out, rank=rank, adapters=adapters, requests=requests, dtype=dtype)


def _linear_grad(name, n, dim, out, dtype, held):
    return dict(name=name, kind="linear_grad", n=n, dim=dim, out=out, dtype=dtype, held=held)


def listed():
    return [
        # a service's single row, added to what its layer before gave
        _norm("norm_row", 1, 1_024, "bf16", True),
        # a training step's forward pass: the sums, the norm and its checkpoint
        _norm("norm_step", 65_537, 1_024, "bf16", True, held=True),
        # a scoring batch of short odd rows in full precision
        _norm("norm_odd", 200_003, 50, "f32", False),
        # the step's backward pass out of its checkpoint
        _norm_grad("norm_grad_step", 65_537, 1_024, "bf16", True, True),
        # the same for short odd rows that were kept as they are
        _norm_grad("norm_grad_odd", 200_003, 50, "f32", False, False),
        # a small batch's activations put away and taken back
        _pack("pack_small", 1_000, 64, "f32"),
        # a large batch's
        _pack("pack_large", 262_144, 1_024, "bf16"),
        # a handful of requests for one row each, every one its own adapter
        _linear("linear_requests", 7, 1_024, 4_096, 16, 64, 7, "bf16"),
        # a scoring job over many customers' rows
        _linear("linear_batch", 8_191, 1_024, 4_096, 16, 64, 50, "bf16"),
        # odd sizes in full precision
        _linear("linear_odd", 1_003, 250, 515, 9, 5, 12, "f32"),
        # the largest step: both gradients of a wide layer out of its checkpoint
        _linear_grad("linear_grad_step", 65_536, 1_024, 4_096, "bf16", True),
        # an odd one in full precision, the inputs kept as they are
        _linear_grad("linear_grad_odd", 4_001, 250, 333, "f32", False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm_grad", "pack", "linear", "linear", "linear_grad", "linear_grad"))
    dtype = rng.choice(("f32", "bf16"))
    dim = _log(rng, 8, 8_192)
    if rng.random() < 0.5:
        dim = max(8, dim // 64 * 64)
    if kind in ("norm", "norm_grad", "pack"):
        n = max(1, min(_log(rng, 1, 262_144), 67_000_000 // dim))
        if kind == "pack":
            return dict(kind=kind, n=n, dim=dim, dtype=dtype)
        return dict(kind=kind, n=n, dim=dim, dtype=dtype, residual=rng.random() < 0.5, held=rng.random() < 0.5)
    dim, out = min(dim, 4_096), _log(rng, 8, 8_192)
    if rng.random() < 0.5:
        out = max(8, out // 64 * 64)
    if kind == "linear_grad":
        n = max(1, min(_log(rng, 1, 65_536), 60_000_000_000 // (dim * out)))
        return dict(kind=kind, n=n, dim=dim, out=out, dtype=dtype, held=rng.random() < 0.5)
    n = max(1, min(_log(rng, 1, 16_384), 60_000_000_000 // (dim * out), 100_000_000 // out))
    requests = min(n, _log(rng, 1, 64))
    return dict(kind=kind, n=n, dim=dim, out=out, rank=_log(rng, 1, 64), adapters=_log(rng, 1, 64), requests=requests, dtype=dtype)


# ---- inputs --------------------------------------------------------------------------

def _held(v):
    """Rows as codes and exponents."""
    n, dim = v.shape
    blocks = torch.nn.functional.pad(v.float(), (0, -dim % _BLOCK)).reshape(n, -1, _BLOCK)
    m, e = torch.frexp(blocks.abs().amax(2, keepdim=True))
    e = (e - 9 + (m > 0.875)).clamp_min(-109)
    codes = torch.ldexp(blocks, -e).to(torch.float8_e4m3fn).reshape(n, -1)[:, :dim].contiguous().view(torch.uint8)
    return codes, (e[:, :, 0] + 127).to(torch.uint8)


def _values(codes, scales):
    """What codes and exponents stand for."""
    n, dim = codes.shape
    by = torch.exp2(scales.float() - 127.0).repeat_interleave(_BLOCK, 1)[:, :dim]
    return codes.view(torch.float8_e4m3fn).float() * by


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    dtype, kind, n, dim = _TYPES[case["dtype"]], case["kind"], case["n"], case["dim"]

    def normal(shape, by=1.0):
        return torch.randn(shape, generator=gen, device=_DEV).mul_(by)

    def rows(shape):
        # rows of different sizes, a few columns far larger than the others
        v = normal(shape) * torch.exp(normal((shape[0], 1), 0.5))
        return v.mul_(torch.where(torch.rand(shape[1], generator=gen, device=_DEV) < 0.02, 20.0, 1.0))

    state = dict(kind=kind, dtype=dtype)
    if kind in ("norm", "norm_grad"):
        state["weight"] = 1.0 + normal((dim,), 0.2)
        state["hold"] = case["held"]
        x = rows((n, dim))
        if kind == "norm":
            state["x"] = x.to(dtype)
            state["residual"] = rows((n, dim)).to(dtype) if case["residual"] else None
        else:
            state["dout"] = normal((n, dim), 1.0 / n).to(dtype)
            state["dtotal"] = normal((n, dim), 1.0 / n).to(dtype) if case["residual"] else None
            inv = torch.rsqrt(x.to(dtype).float().square().mean(1) + _EPS)
            state["inv"] = inv
            if case["held"]:
                state["codes"], state["scales"] = _held(x.to(dtype).float() * inv[:, None])
            else:
                state["x"] = x.to(dtype)
            if own:
                import hessboost_amd as hb
                state["workspace"] = _bytes(hb.rms_norm_grad_workspace(n, dim, dtype))
    elif kind == "pack":
        state["x"] = rows((n, dim)).to(dtype)
    else:
        out = case["out"]
        state["w"] = normal((out, dim), 1.0 / math.sqrt(dim)).to(dtype)
        if kind == "linear":
            state["x"] = normal((n, dim)).to(dtype)
            state["bias"] = normal((out,), 0.1)
            # a trained pair's product is small beside the projection
            state["down"] = normal((case["adapters"], case["rank"], dim), 1.0 / math.sqrt(dim)).to(dtype)
            state["up"] = normal((case["adapters"], out, case["rank"]), 0.1).to(dtype)
            state["scale"] = 2.0 * torch.rand(case["adapters"], generator=gen, device=_DEV)
            # requests of uneven lengths, one in twenty without an adapter
            cut = torch.randperm(n - 1, generator=gen, device=_DEV)[:case["requests"] - 1] + 1 if n > 1 else torch.zeros(0, device=_DEV)
            start = torch.zeros(n, dtype=torch.int64, device=_DEV)
            start[cut.long()] = 1
            of = torch.randint(0, case["adapters"], (case["requests"],), generator=gen, device=_DEV)
            of[torch.rand(case["requests"], generator=gen, device=_DEV) < 0.05] = -1
            state["ids"] = of[start.cumsum(0)].to(torch.int32)
        else:
            state["dout"] = normal((n, out), 1.0 / n).to(dtype)
            state["weight"] = None
            if case["held"]:
                # normalised rows, whose norm's weight is applied to the columns
                state["codes"], state["scales"] = _held(normal((n, dim)))
                state["weight"] = 1.0 + normal((dim,), 0.2)
            else:
                state["x"] = normal((n, dim)).to(dtype)
        if own:
            import hessboost_amd as hb
            state["workspace"] = _bytes(hb.linear_workspace(n, out, dim, dtype, rank=case["rank"]) if kind == "linear" else
                                        hb.linear_grad_workspace(n, out, dim, dtype))
    torch.cuda.synchronize()
    return state


def _bytes(n):
    return torch.empty(max(1, n), dtype=torch.uint8, device=_DEV)


# ---- one pass ----------------------------------------------------------------------------

def _plain(state):
    kind, dtype = state["kind"], state["dtype"]
    if kind == "pack":
        return {"values": _values(*_held(state["x"])).to(torch.bfloat16)}
    if kind == "norm":
        total = state["x"].float()
        if state["residual"] is not None:
            total = total + state["residual"].float()
        inv = 1.0 / torch.sqrt(total.square().mean(1) + _EPS)
        normed = total * inv[:, None]
        got = {"out": (normed * state["weight"]).to(dtype)}
        if state["residual"] is not None:
            got["total"] = total.to(dtype)
        if state["hold"]:
            got["inv"] = inv
            got["held"] = _values(*_held(normed)).to(torch.bfloat16)
        return got
    if kind == "norm_grad":
        inv = state["inv"][:, None]
        normed = _values(state["codes"], state["scales"]) if state["hold"] else state["x"].float() * inv
        dout = state["dout"].float()
        g = dout * state["weight"]
        dx = inv * (g - normed * (g * normed).mean(1, keepdim=True))
        if state["dtotal"] is not None:
            dx = dx + state["dtotal"].float()
        return {"dx": dx.to(dtype), "dweight": (dout * normed).sum(0)}
    if kind == "linear":
        x, ids = state["x"].float(), state["ids"].long()
        out = x @ state["w"].float().T + state["bias"]
        some = (ids >= 0).float()
        at = ids.clamp_min(0)
        by = (state["scale"][at] * some)[:, None]
        count, rank, dim = state["down"].shape
        if x.shape[0] <= 64:
            low = (state["down"][at].float() * x[:, None, :]).sum(2) * by
            more = (state["up"][at].float() * low[:, None, :]).sum(2)
        else:
            # every adapter at once, the others' places zeros
            low = (x @ state["down"].float().reshape(count * rank, dim).T).reshape(-1, count, rank)
            low = low * (torch.arange(count, device=x.device) == ids[:, None])[:, :, None] * by[:, :, None]
            more = low.reshape(-1, count * rank) @ state["up"].float().transpose(1, 2).reshape(count * rank, -1)
        return {"out": (out + more).to(dtype)}
    dout = state["dout"].float()
    x = state["x"].float() if state["weight"] is None else _values(state["codes"], state["scales"])
    dw = dout.T @ x
    if state["weight"] is not None:
        dw = dw * state["weight"]
    return {"dx": (dout @ state["w"].float()).to(dtype), "dw": dw.to(dtype), "db": dout.sum(0)}


def _codes(n, dim):
    return torch.empty((n, dim), dtype=torch.uint8, device=_DEV), torch.empty((n, -(-dim // _BLOCK)), dtype=torch.uint8, device=_DEV)


def _own(state):
    import hessboost_amd as hb
    kind = state["kind"]
    if kind == "pack":
        x = state["x"]
        codes, scales = _codes(*x.shape)
        values = torch.empty(x.shape, dtype=torch.bfloat16, device=_DEV)
        hb.pack_rows(x, codes, scales)
        hb.unpack_rows(codes, scales, values)
        return {"values": values}
    if kind == "norm":
        x = state["x"]
        got = {"out": torch.empty_like(x)}
        if state["residual"] is not None:
            got["total"] = torch.empty_like(x)
        if not state["hold"]:
            hb.rms_norm(x, got["out"], weight=state["weight"], eps=_EPS, residual=state["residual"], total=got.get("total"))
            return got
        codes, scales = _codes(*x.shape)
        got["inv"] = torch.empty(x.shape[0], device=_DEV)
        got["held"] = torch.empty(x.shape, dtype=torch.bfloat16, device=_DEV)
        hb.rms_norm(x, got["out"], weight=state["weight"], eps=_EPS, residual=state["residual"], total=got.get("total"),
                    inv=got["inv"], codes=codes, scales=scales, normed=True)
        hb.unpack_rows(codes, scales, got["held"])
        return got
    if kind == "norm_grad":
        dx, dweight = torch.empty_like(state["dout"]), torch.empty_like(state["weight"])
        of = dict(codes=state["codes"], scales=state["scales"]) if state["hold"] else dict(x=state["x"])
        hb.rms_norm_grad(state["dout"], dx, **of, inv=state["inv"], weight=state["weight"], dtotal=state["dtotal"],
                         dweight=dweight, workspace=state["workspace"])
        return {"dx": dx, "dweight": dweight}
    if kind == "linear":
        out = torch.empty((state["x"].shape[0], state["w"].shape[0]), dtype=state["dtype"], device=_DEV)
        hb.linear(state["x"], state["w"], out, bias=state["bias"], down=state["down"], up=state["up"], ids=state["ids"],
                  scale=state["scale"], workspace=state["workspace"])
        return {"out": out}
    dout, w = state["dout"], state["w"]
    dx = torch.empty((dout.shape[0], w.shape[1]), dtype=state["dtype"], device=_DEV)
    dw, db = torch.empty_like(w), torch.empty(w.shape[0], device=_DEV)
    of = dict(x=state["x"]) if state["weight"] is None else dict(codes=state["codes"], scales=state["scales"], weight=state["weight"])
    hb.linear_grad(dout, w, **of, dx=dx, dw=dw, db=db, workspace=state["workspace"])
    return {"dx": dx, "dw": dw, "db": db}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    size = 4.0 if case["dtype"] == "f32" else 2.0
    kind, n, dim = case["kind"], case["n"], case["dim"]
    codes = n * dim + n * -(-dim // _BLOCK)
    if kind == "pack":  # to codes, and from codes to 16 bits
        return {"bytes": size * n * dim + 2 * codes + 2.0 * n * dim, "flops": 4.0 * n * dim}
    if kind == "norm":
        arrays = 4 if case["residual"] else 2
        more = 2 * codes + 2.0 * n * dim + 4.0 * n if case["held"] else 0.0
        return {"bytes": arrays * size * n * dim + 4.0 * dim + more, "flops": 6.0 * n * dim}
    if kind == "norm_grad":
        arrays = 3 if case["residual"] else 2
        return {"bytes": arrays * size * n * dim + (codes if case["held"] else size * n * dim) + 4.0 * n + 8.0 * dim,
                "flops": 10.0 * n * dim}
    out = case["out"]
    if kind == "linear":
        rank, used = case["rank"], min(case["adapters"], case["requests"])
        return {"bytes": size * (n * (dim + out) + dim * out + used * rank * (dim + out)) + 4.0 * (out + n),
                "flops": 2.0 * n * (dim * out + rank * (dim + out))}
    held = codes if case["held"] else size * n * dim
    return {"bytes": size * (n * (out + dim) + 2.0 * dim * out) + held + 4.0 * out, "flops": 4.0 * n * dim * out + n * out}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _in_8_bits(v):
    """The values that rows in 8 bits hold, by their grid: three bits behind
    the leading one, steps of 2^-9 below 2^-6."""
    n, dim = v.shape
    v = torch.nn.functional.pad(v, (0, -dim % _BLOCK)).reshape(n, -1, _BLOCK)
    top = v.abs().amax(2, keepdim=True)
    by = torch.where(top > 0, torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0)), -109.0)
    # the logarithm's own rounding, at a power of two's border
    by = torch.where(torch.exp2(by - 1) * 448.0 >= top, by - 1, by)
    by = torch.where(torch.exp2(by) * 448.0 < top, by + 1, by).clamp_min(-109.0)
    u = v / torch.exp2(by)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3.0)
    return (torch.round(u / step) * step * torch.exp2(by)).reshape(n, -1)[:, :dim]


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "pack":
        return {"values": _in_8_bits(s["x"].double())}
    if kind == "norm":
        total = s["x"].double()
        got = {"out": None}
        if s["residual"] is not None:
            total = total + s["residual"].double()
            got["total"] = total
        inv = (total.pow(2).sum(1) / case["dim"] + _EPS).pow(-0.5)
        got["out"] = total * inv[:, None] * s["weight"].double()
        if s["hold"]:
            got["inv"] = inv
            got["held"] = _in_8_bits(total * inv[:, None])
        return got
    if kind == "linear":
        x, w = s["x"].double(), s["w"].double()
        out = torch.addmm(s["bias"].double(), x, w.t())
        for i in range(case["adapters"]):
            r = torch.nonzero(s["ids"] == i).squeeze(1)
            if len(r):
                out[r] += float(s["scale"][i]) * ((x[r] @ s["down"][i].double().t()) @ s["up"][i].double().t())
        return {"out": out}
    if s["hold"] if kind == "norm_grad" else s["weight"] is not None:
        # e4m3 by its bits: a sign, four of exponent, three behind the leading one
        c = s["codes"].long()
        e, m = c >> 3 & 15, (c & 7).double()
        v = torch.where(e > 0, (8 + m) * torch.exp2(e.double() - 10), m * 2.0 ** -9) * (1.0 - 2.0 * (c >> 7).double())
        v *= torch.exp2(s["scales"].double() - 127).repeat_interleave(_BLOCK, 1)[:, :case["dim"]]
    else:
        v = s["x"].double()
    dout = s["dout"].double()
    if kind == "norm_grad":
        inv = s["inv"].double()[:, None]
        normed = v if s["hold"] else v * inv
        along = (dout * s["weight"].double() * normed).sum(1, keepdim=True) / case["dim"]
        dx = (dout * s["weight"].double() - along * normed) * inv
        if s["dtotal"] is not None:
            dx = dx + s["dtotal"].double()
        return {"dx": dx, "dweight": (dout * normed).sum(0)}
    dw = dout.t().contiguous() @ v
    if s["weight"] is not None:
        dw = dw * s["weight"].double()
    return {"dx": dout @ s["w"].double(), "dw": dw, "db": dout.sum(0)}
