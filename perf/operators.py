"""Operators over a forest's leaves and over many classes, as measurable cases.

A forest answers with one leaf a tree (`Forest.predict_leaf`,
`predict_margin_device`). A model on those leaves looks each one up in a table
of vectors, scores the sum against every class, and steps by clipped
gradients. Kinds (`case["kind"]`):

- "embed": rows' leaf vectors, scaled by tree and summed (one column of ids is
  a plain table lookup);
- "embed_grad": the table's gradient;
- "answer": each row's best class and minus its log probability, the scores
  not kept;
- "head": the softmax cross entropy of a linear layer over the classes with
  the gradients of its inputs, weights and intercepts;
- "clip": the norm of a set of gradients, and the set scaled to a largest norm.
"""
import math

import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _embed(name, n, columns, rows, dim, dtype, kind="embed", padded=0.0):
    """`rows`: table rows a column (a tree's nodes, or the whole vocabulary)."""
    return dict(name=name, kind=kind, n=n, columns=columns, rows=rows, dim=dim, dtype=dtype, padded=padded)


def _head(name, n, classes, dim, dtype, kind="head", ignored=0.0, weighted=False):
    return dict(name=name, kind=kind, n=n, classes=classes, dim=dim, dtype=dtype, ignored=ignored, weighted=weighted)


def _clip(name, tensors, total, dtype):
    return dict(name=name, kind="clip", tensors=tensors, total=total, dtype=dtype)


def listed():
    return [
        # a service's request: a handful of rows through 100 trees of depth 6
        _embed("embed_request", 32, 100, 127, 32, "f32"),
        # a batch scoring job over the same forest, an odd row count
        _embed("embed_batch", 200_003, 100, 127, 64, "bf16"),
        # a step of a small model: 20 shallow trees, short vectors
        _embed("embed_grad_small", 4_000, 20, 31, 16, "f32", "embed_grad"),
        # a step over a large batch, the table much smaller than the batch
        _embed("embed_grad_batch", 200_003, 100, 127, 64, "bf16", "embed_grad"),
        # one id a row into a large table, frequent ids first, some rows padding
        _embed("embed_grad_tokens", 65_536, 1, 131_072, 1_024, "bf16", "embed_grad", padded=0.02),
        # one row answered from the largest set of classes
        _head("answer_row", 1, 131_072, 1_024, "bf16", "answer"),
        # ten classes over a large weighted batch, an odd width
        _head("head_ten_classes", 200_003, 10, 50, "f32", weighted=True),
        # thousands of classes in full precision
        _head("head_full_precision", 4_096, 5_003, 256, "f32"),
        # an ordinary step over tens of thousands of classes, some rows ignored
        _head("head_ordinary", 8_191, 32_768, 512, "bf16", ignored=0.05),
        # the largest step
        _head("head_large", 16_384, 131_072, 1_024, "bf16"),
        # a small model's gradients: many little tensors of odd sizes
        _clip("clip_small", 40, 300_001, "f32"),
        # a large model's: its tables and head
        _clip("clip_large", 6, 400_000_003, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("embed", "embed", "embed_grad", "embed_grad", "answer", "head", "head", "head", "clip"))
    dtype = rng.choice(("f32", "bf16"))
    if kind in ("embed", "embed_grad"):
        if rng.random() < 0.6:
            columns, rows, dim = _log(rng, 2, 200), (2 << rng.randint(2, 8)) - 1, _log(rng, 4, 256)
            n, padded = _log(rng, 1, 200_003), 0.0
        else:
            columns, rows, dim = 1, _log(rng, 500, 131_072), _log(rng, 16, 1_024)
            n, padded = _log(rng, 1, 65_536), rng.choice((0.0, 0.02))
        n = max(1, min(n, 200_003 * 100 * 64 // (columns * dim)))
        return dict(kind=kind, n=n, columns=columns, rows=rows, dim=dim, dtype=dtype, padded=padded)
    if kind == "answer":
        return dict(kind=kind, n=_log(rng, 1, 64), classes=_log(rng, 1_000, 131_072), dim=_log(rng, 16, 1_024),
                    dtype=dtype, ignored=0.0, weighted=False)
    if kind == "head":
        classes, dim = _log(rng, 2, 131_072), _log(rng, 8, 1_024)
        n = _log(rng, 16, 500_000)
        n = max(1, min(n, 400_000_000 // classes, 60_000_000_000 // (classes * dim), 30_000_000 // dim))
        return dict(kind=kind, n=n, classes=classes, dim=dim, dtype=dtype, ignored=rng.choice((0.0, 0.05)),
                    weighted=rng.random() < 0.5)
    total = _log(rng, 10_000, 200_000_000)
    return dict(kind=kind, tensors=_log(rng, 1, 60), total=total, dtype=dtype)


# ---- inputs --------------------------------------------------------------------------

def _tensor_sizes(case):
    """A set's tensor sizes: the first half of the total in one table, the
    rest halving again and again, the last tensors a few elements each."""
    left, sizes = case["total"], []
    for i in range(case["tensors"] - 1):
        sizes.append(max(1, min(left - (case["tensors"] - 1 - i), left // 2 | 1)))
        left -= sizes[-1]
    return sizes + [left]


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    dtype, kind = _TYPES[case["dtype"]], case["kind"]

    def normal(shape, by=1.0):
        return torch.randn(shape, generator=gen, device=_DEV).mul_(by).to(dtype)

    def uniform(shape):
        return torch.rand(shape, generator=gen, device=_DEV)

    state = dict(kind=kind, dtype=dtype)
    if kind == "clip":
        # gradients of a diverging step: the set's norm is above the largest
        sizes = _tensor_sizes(case)
        state["grads"] = [normal((s,), 0.01 * (1 + i % 3)) for i, s in enumerate(sizes)]
        state["max_norm"] = 0.005 * math.sqrt(case["total"])
        if own:
            import hessboost_amd as hb
            state["workspace"] = _bytes(hb.clip_gradients_workspace(len(sizes)))
    elif kind in ("embed", "embed_grad"):
        n, t, rows, dim = case["n"], case["columns"], case["rows"], case["dim"]
        u = uniform((n, t))
        if t > 1:
            # complete trees: the leaves are the second half of the nodes,
            # some of them far fuller than others
            inner = rows // 2
            state["ids"] = (inner + (u * u * (rows - inner)).long().clamp_max(rows - inner - 1)).to(torch.int32)
            state["offset"] = (torch.arange(t, device=_DEV) * rows).to(torch.int32)
            state["scale"] = 0.5 + uniform((t,))
            state["table_rows"] = rows * t
        else:
            state["ids"] = (torch.exp(u * math.log(rows)).long() - 1).clamp_(0, rows - 1).to(torch.int32)
            state["offset"], state["table_rows"] = None, rows
            state["scale"] = torch.full((1,), math.sqrt(dim), device=_DEV)
        if case["padded"]:
            state["ids"][uniform((n, t)) < case["padded"]] = -1
        if kind == "embed":
            state["table"] = normal((state["table_rows"], dim), 0.05)
        else:
            state["dout"] = normal((n, dim), 1.0 / n)
            if own:
                import hessboost_amd as hb
                state["workspace"] = _bytes(hb.leaf_embedding_grad_workspace(n, t, state["table_rows"], dim, dtype))
    else:
        n, classes, dim = case["n"], case["classes"], case["dim"]
        state["w"] = normal((classes, dim), 2.0 / math.sqrt(dim))
        state["h"] = normal((n, dim))
        state["bias"] = torch.randn((classes,), generator=gen, device=_DEV) * 0.5
        state["labels"], state["weight"] = None, None
        if kind == "head":
            # frequent classes first; some rows lie near their class's weights
            y = (torch.exp(uniform((n,)) * math.log(classes + 1)).long() - 1).clamp_(0, classes - 1)
            near = uniform((n,)) < 0.5
            state["h"] = torch.where(near[:, None], state["h"] + state["w"][y], state["h"])
            if case["ignored"]:
                y[uniform((n,)) < case["ignored"]] = -1
            state["labels"] = y.to(torch.int32)
            if case["weighted"]:
                state["weight"] = 0.5 + uniform((n,))
            state["by"] = 1.0 / n
        if own:
            import hessboost_amd as hb
            state["workspace"] = _bytes(hb.softmax_head_workspace(n, classes, dim, dtype, gradient=kind == "head"))
    torch.cuda.synchronize()
    return state


def _bytes(n):
    return torch.empty(max(1, n), dtype=torch.uint8, device=_DEV)


# ---- one pass ----------------------------------------------------------------------------

def _places(state):
    """Each id's table row, and one past the table for an id that adds nothing."""
    ids = state["ids"].long()
    rows = ids if state["offset"] is None else ids + state["offset"].long()
    return torch.where((ids >= 0) & (rows < state["table_rows"]), rows, state["table_rows"])


def _plain(state):
    kind, dtype = state["kind"], state["dtype"]
    if kind == "embed":
        table = torch.nn.functional.pad(state["table"].float(), (0, 0, 0, 1))
        return {"out": (table[_places(state)] * state["scale"][:, None]).sum(1).to(dtype)}
    if kind == "embed_grad":
        n, dim = state["dout"].shape
        part = state["dout"].float()[:, None, :] * state["scale"][None, :, None]
        total = torch.zeros((state["table_rows"] + 1, dim), device=part.device)
        total.index_add_(0, _places(state).reshape(-1), part.reshape(-1, dim))
        return {"dtable": total[:-1].to(dtype)}
    if kind == "clip":
        norm = torch.stack([g.float().square().sum() for g in state["grads"]]).sum().sqrt()
        by = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        return {"norm": norm.reshape(1), "grads": [(g.float() * by).to(dtype) for g in state["grads"]]}
    h, w = state["h"].float(), state["w"].float()
    margin = h @ w.T
    margin += state["bias"]
    top = margin.amax(1, keepdim=True)
    e = torch.exp(margin - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    if kind == "answer":
        # the first of the largest
        best = torch.where(margin == top, torch.arange(w.shape[0], device=w.device), w.shape[0]).amin(1)
        return {"best": best.to(torch.int32), "loss": lse - top.squeeze(1), "lse": lse}
    y = state["labels"].long()
    row = (y >= 0).float() if state["weight"] is None else torch.where(y >= 0, state["weight"], 0.0)
    at = y.clamp_min(0)[:, None]
    loss = row * (lse - margin.gather(1, at).squeeze(1))
    g = e.div_(total)
    g.scatter_add_(1, at, torch.full_like(top, -1.0))
    g *= (row * state["by"])[:, None]
    return {"loss": loss, "lse": lse, "dh": (g @ w).to(dtype), "dw": (g.T @ h).to(dtype), "db": g.sum(0)}


def _own(state):
    import hessboost_amd as hb
    kind = state["kind"]
    if kind == "embed":
        out = torch.empty((state["ids"].shape[0], state["table"].shape[1]), dtype=state["dtype"], device=_DEV)
        hb.leaf_embedding(state["table"], state["ids"], out, offset=state["offset"], scale=state["scale"])
        return {"out": out}
    if kind == "embed_grad":
        dtable = torch.empty((state["table_rows"], state["dout"].shape[1]), dtype=state["dtype"], device=_DEV)
        hb.leaf_embedding_grad(state["dout"], state["ids"], dtable, offset=state["offset"], scale=state["scale"],
                               workspace=state["workspace"])
        return {"dtable": dtable}
    if kind == "clip":
        norm = torch.empty(1, device=_DEV)
        out = [torch.empty_like(g) for g in state["grads"]]
        hb.clip_gradients(state["grads"], state["max_norm"], norm=norm, out=out, workspace=state["workspace"])
        return {"norm": norm, "grads": out}
    n, classes = state["h"].shape[0], state["w"].shape[0]
    loss, lse = torch.empty(n, device=_DEV), torch.empty(n, device=_DEV)
    if kind == "answer":
        best = torch.empty(n, dtype=torch.int32, device=_DEV)
        hb.softmax_head(state["h"], state["w"], bias=state["bias"], best=best, loss=loss, lse=lse,
                        workspace=state["workspace"])
        return {"best": best, "loss": loss, "lse": lse}
    dh, dw, db = torch.empty_like(state["h"]), torch.empty_like(state["w"]), torch.empty(classes, device=_DEV)
    hb.softmax_head(state["h"], state["w"], bias=state["bias"], labels=state["labels"], weight=state["weight"],
                    loss=loss, lse=lse, dh=dh, dw=dw, db=db, grad_scale=state["by"], workspace=state["workspace"])
    return {"loss": loss, "lse": lse, "dh": dh, "dw": dw, "db": db}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    size = 4.0 if case["dtype"] == "f32" else 2.0
    if case["kind"] == "clip":
        return {"bytes": 2 * size * case["total"], "flops": 3.0 * case["total"]}
    if case["kind"] in ("embed", "embed_grad"):
        n, t, dim = case["n"], case["columns"], case["dim"]
        # a tree's leaves are half its nodes; the gradient's table is written whole
        leaves = min(n * t, case["rows"] if t == 1 else t * (case["rows"] // 2 + 1))
        rows = leaves if case["kind"] == "embed" else case["rows"] * t
        return {"bytes": 4.0 * n * t + size * dim * (n + rows), "flops": 2.0 * n * t * dim}
    n, classes, dim = case["n"], case["classes"], case["dim"]
    once = size * dim * (n + classes) + 4.0 * classes + 8.0 * n
    if case["kind"] == "answer":
        return {"bytes": once + 4.0 * n, "flops": 2.0 * n * classes * dim}
    # the scores, and each factor's gradient
    return {"bytes": 2 * once, "flops": 6.0 * n * classes * dim}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "clip":
        squares = math.fsum(float((g.double() ** 2).sum()) for g in s["grads"])
        norm = math.sqrt(squares)
        by = min(1.0, s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor([norm], dtype=torch.float64), "grads": [g.double() * by for g in s["grads"]]}
    if s["kind"] in ("embed", "embed_grad"):
        n, t = s["ids"].shape
        dim = case["dim"]
        to = torch.zeros((n if s["kind"] == "embed" else s["table_rows"], dim), dtype=torch.float64, device=_DEV)
        src = (s["table"] if s["kind"] == "embed" else s["dout"]).double()
        for c in range(t):
            ids = s["ids"][:, c].long()
            base = 0 if s["offset"] is None else int(s["offset"][c])
            r = torch.nonzero((ids >= 0) & (ids + base < s["table_rows"])).squeeze(1)
            v = ids[r] + base
            by = float(s["scale"][c])
            if s["kind"] == "embed":
                to[r] += by * src[v]
            else:
                to.index_add_(0, v, src[r], alpha=by)
        return {"out" if s["kind"] == "embed" else "dtable": to}
    h, w, b = s["h"].double(), s["w"].double(), s["bias"].double()
    n, classes = h.shape[0], w.shape[0]
    loss = torch.zeros(n, dtype=torch.float64, device=_DEV)
    lse = torch.zeros_like(loss)
    if s["kind"] == "answer":
        z = torch.addmm(b, h, w.t())
        lse = torch.logsumexp(z, 1)
        best = z.max(1).values
        return {"best": z.argmax(1).to(torch.int32), "loss": lse - best, "lse": lse}
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    db = torch.zeros(classes, dtype=torch.float64, device=_DEV)
    step = max(1, (1 << 28) // classes)
    for a in range(0, n, step):
        hh, y = h[a:a + step], s["labels"][a:a + step].long()
        z = torch.addmm(b, hh, w.t())
        lse[a:a + step] = torch.logsumexp(z, 1)
        r = torch.nonzero(y >= 0).squeeze(1)
        wt = torch.ones(len(y), dtype=torch.float64, device=_DEV)
        if s["weight"] is not None:
            wt = s["weight"][a:a + step].double()
        loss[a + r] = wt[r] * (lse[a + r] - z[r, y[r]])
        p = torch.exp(z[r] - lse[a + r][:, None])
        p[torch.arange(len(r), device=_DEV), y[r]] -= 1.0
        p *= wt[r][:, None] * s["by"]
        dh[a + r] = p @ w
        dw += p.t() @ hh[r]
        db += p.sum(0)
    return {"loss": loss, "lse": lse, "dh": dh, "dw": dw, "db": db}
