"""What is measured of the operators that a model over tokens trains with: the embedding lookup with its gradient and its
sparse row update, the softmax cross-entropy against integer labels, and the orthogonalised (Muon) update of matrices.

``run`` computes a case in its plain form (elementary torch operations, 32 bits, rounded once), or, with ``own``, by the
framework's own operators.  ``exact`` gives the same outputs from the definitions in 64 bits.

Kinds of cases:

* ``lookup``      out[t] = scale * table[ids[t]] (a row of zeros where the id is outside the table)
* ``table_grad``  the lookup and the gradient of the whole table: grad[v] = scale * sum of g[t] over the t with id v
* ``row_sgd``     the sparse update: table[v] -= lr * scale * sum of g[t], rows that do not occur stay as they are
* ``xent``        row losses and the gradient of ``grad_scale * sum(losses)`` in one call
* ``xent_rows``   row losses, then the gradient for an upstream gradient of each row (two calls, as autograd makes them)
* ``ortho``       the orthogonal factor by five Newton-Schulz steps
* ``muon``        a whole optimiser step over a list of matrices: momentum, orthogonalisation, weight update
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_NS = (3.4445, -4.7750, 2.0315)
_EPS = 1e-7


def listed():
    return [
        # one decoding step of a batch of eight sequences: latency
        {"name": "lookup_decode", "kind": "lookup", "tokens": 8, "rows": 32768, "dim": 1024, "dtype": "bfloat16", "pad": 0.0},
        # an ordinary training batch of a small model, odd vocabulary
        {"name": "table_grad_f32", "kind": "table_grad", "tokens": 16384, "rows": 50001, "dim": 768, "dtype": "float32", "pad": 0.02},
        # the largest batch: 128 Ki tokens, 128 Ki rows
        {"name": "table_grad_large", "kind": "table_grad", "tokens": 131072, "rows": 131072, "dim": 4096, "dtype": "bfloat16", "pad": 0.0},
        # a parameter server's sparse apply: few of many rows
        {"name": "row_sgd_sparse", "kind": "row_sgd", "tokens": 32768, "rows": 262144, "dim": 256, "dtype": "float32", "pad": 0.0},
        # hot rows of an odd, unaligned width (a categorical feature)
        {"name": "row_sgd_hot_odd", "kind": "row_sgd", "tokens": 3001, "rows": 1009, "dim": 101, "dtype": "float32", "pad": 0.05},
        # the framework's batch of 100 over a thousand classes: latency
        {"name": "xent_small", "kind": "xent", "tokens": 100, "classes": 1000, "dtype": "float32", "pad": 0.0},
        # an ordinary training batch in fp32
        {"name": "xent_f32", "kind": "xent", "tokens": 4096, "classes": 32768, "dtype": "float32", "pad": 0.0},
        # the largest: 16 Ki tokens over 128 Ki classes
        {"name": "xent_large", "kind": "xent", "tokens": 16384, "classes": 131072, "dtype": "bfloat16", "pad": 0.0},
        # ragged: odd classes (rows start unaligned), padded labels, weighted rows through the backward pass
        {"name": "xent_rows_odd", "kind": "xent_rows", "tokens": 2047, "classes": 50001, "dtype": "bfloat16", "pad": 0.1},
        # the three matrices of the framework's 784-512-256-10 stack in one step: latency
        {"name": "muon_stack", "kind": "muon", "shapes": "784x512,512x256,256x10", "nesterov": True},
        # a wide matrix in bf16
        {"name": "ortho_bf16", "kind": "ortho", "m": 1024, "n": 4096, "dtype": "bfloat16"},
        # a large square layer
        {"name": "muon_large", "kind": "muon", "shapes": "4096x4096", "nesterov": True},
    ]


def _log_size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["lookup", "table_grad", "row_sgd", "xent", "xent_rows", "ortho", "muon", "muon"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind in ("lookup", "table_grad", "row_sgd"):
        rows, dim = _log_size(rng, 10, 262144), _log_size(rng, 8, 8192)
        while rows * dim > 1 << 29:
            rows, dim = max(10, rows // 2), dim
        tokens = min(_log_size(rng, 1, 131072), (1 << 29) // dim)
        return {"kind": kind, "tokens": tokens, "rows": rows, "dim": dim, "dtype": dtype, "pad": rng.choice([0.0, 0.05, 0.3])}
    if kind in ("xent", "xent_rows"):
        classes = _log_size(rng, 2, 262144)
        tokens = min(_log_size(rng, 1, 16384), (1 << 30) // classes)
        return {"kind": kind, "tokens": tokens, "classes": classes, "dtype": dtype, "pad": rng.choice([0.0, 0.1])}
    if kind == "ortho":
        return {"kind": kind, "m": _log_size(rng, 8, 4096), "n": _log_size(rng, 8, 4096), "dtype": dtype}
    shapes = ["%dx%d" % (_log_size(rng, 8, 2048), _log_size(rng, 8, 2048)) for _ in range(rng.randint(1, 4))]
    return {"kind": kind, "shapes": ",".join(shapes), "nesterov": rng.random() < 0.7}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ids(count, rows, pad, g):
    """Ids as words occur: the chance of id v falls as 1 / (v + 1); a share of ``pad`` is padding (-1)."""
    u = torch.rand(count, device="cuda", generator=g, dtype=torch.float64)
    ids = (torch.exp(u * math.log(rows + 1)) - 1).long().clamp_(0, rows - 1)
    if pad:
        ids[torch.rand(count, device="cuda", generator=g) < pad] = -1
    return ids


def _gradient(m, n, g):
    """A matrix with the spectrum of a layer's gradient: a few strong directions over noise."""
    r = max(1, min(m, n) // 16)
    u = torch.randn(m, r, device="cuda", generator=g)
    v = torch.randn(r, n, device="cuda", generator=g)
    return (u @ v / math.sqrt(r) + 0.3 * torch.randn(m, n, device="cuda", generator=g)) * 1e-3


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind in ("lookup", "table_grad", "row_sgd"):
        dt = _TYPES[case["dtype"]]
        t, v, d = case["tokens"], case["rows"], case["dim"]
        s = {"kind": kind, "table": (0.02 * torch.randn(v, d, device="cuda", generator=g)).to(dt),
             "ids": _ids(t, v, case["pad"], g), "scale": math.sqrt(d)}
        if kind != "lookup":
            s["g"] = (1e-2 * torch.randn(t, d, device="cuda", generator=g)).to(dt)
        if kind == "row_sgd":
            s["lr"] = torch.full((1,), 0.01, device="cuda")
        return s
    if kind in ("xent", "xent_rows"):
        dt = _TYPES[case["dtype"]]
        t, c = case["tokens"], case["classes"]
        s = {"kind": kind, "logits": torch.empty(t, c, device="cuda", dtype=dt)}
        for a in range(0, t, 2048):
            s["logits"][a:a + 2048] = 2.5 * torch.randn(min(2048, t - a), c, device="cuda", generator=g)
        s["labels"] = _ids(t, c, case["pad"], g)
        if kind == "xent":
            s["grad_scale"] = 1.0 / t
        else:
            s["g"] = torch.rand(t, device="cuda", generator=g) / t
        return s
    if kind == "ortho":
        return {"kind": kind, "x": _gradient(case["m"], case["n"], g).to(_TYPES[case["dtype"]])}
    s = {"kind": kind, "w": [], "g": [], "buf": [], "nesterov": bool(case["nesterov"]), "momentum": 0.95,
         "lr": torch.full((1,), 0.02, device="cuda")}
    for m, n in _shapes(case):
        s["w"].append(torch.randn(m, n, device="cuda", generator=g) / math.sqrt(m))
        s["g"].append(_gradient(m, n, g))
        s["buf"].append(4.0 * _gradient(m, n, g))
    if own:
        from distributed_tensorflow_amd.ops import muon

        s["plan"] = muon.MuonPlan(s["w"], s["g"], s["buf"])
    return s


def _plain_factor(u):
    x = u.float()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = (x / (x.double().square().sum().sqrt() + _EPS)).float()
    a, b, c = _NS
    for _ in range(5):
        p = x @ x.t()
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.t() if flip else x


def _plain_rows(ids, g, rows, scale):
    keep = (ids >= 0) & (ids < rows)
    total = torch.zeros(rows, g.shape[1], device=g.device)
    total.index_add_(0, torch.where(keep, ids, 0), g.float() * (keep.float() * scale)[:, None])
    return total


def _plain_lookup(table, ids, scale):
    keep = (ids >= 0) & (ids < table.shape[0])
    rows = table[torch.where(keep, ids, 0)].float() * scale
    return torch.where(keep[:, None], rows, 0.0).to(table.dtype)


def _plain_xent(logits, labels, weight):
    keep = labels >= 0
    at = torch.where(keep, labels, 0)[:, None]
    z = logits.float()
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    loss = (torch.log(total) + top - z.gather(1, at))[:, 0] * keep
    dz = e / total
    dz.scatter_add_(1, at, torch.full_like(total, -1.0))
    return loss, (dz * (weight * keep)[:, None]).to(logits.dtype)


def _run_plain(s):
    kind = s["kind"]
    if kind == "lookup":
        return _plain_lookup(s["table"], s["ids"], s["scale"])
    if kind == "table_grad":
        out = _plain_lookup(s["table"], s["ids"], s["scale"])
        return out, _plain_rows(s["ids"], s["g"], s["table"].shape[0], s["scale"]).to(s["table"].dtype)
    if kind == "row_sgd":
        total = _plain_rows(s["ids"], s["g"], s["table"].shape[0], s["scale"])
        s["table"].copy_(s["table"].float() - s["lr"] * total)
        return s["table"]
    if kind == "xent":
        return _plain_xent(s["logits"], s["labels"], torch.full_like(s["labels"], s["grad_scale"], dtype=torch.float32))
    if kind == "xent_rows":
        return _plain_xent(s["logits"], s["labels"], s["g"])
    if kind == "ortho":
        return _plain_factor(s["x"]).to(s["x"].dtype)
    for w, g, buf in zip(s["w"], s["g"], s["buf"]):
        buf.mul_(s["momentum"]).add_(g)
        u = g + s["momentum"] * buf if s["nesterov"] else buf
        w.sub_(s["lr"] * math.sqrt(max(1.0, w.shape[1] / w.shape[0])) * _plain_factor(u))
    return s["w"], s["buf"]


def _run_own(s):
    from distributed_tensorflow_amd.ops import embedding, muon, xent

    kind = s["kind"]
    if kind == "lookup":
        return embedding.lookup(s["table"], s["ids"], s["scale"])
    if kind == "table_grad":
        out = embedding.lookup(s["table"], s["ids"], s["scale"])
        return out, embedding.lookup_grad(s["ids"], s["g"], s["table"].shape[0], s["scale"])
    if kind == "row_sgd":
        return embedding.lookup_sgd(s["table"], s["ids"], s["g"], s["lr"], s["scale"])
    if kind == "xent":
        dz = torch.empty_like(s["logits"])
        return xent.sparse_softmax_xent_step(s["logits"], s["labels"], dz=dz, grad_scale=s["grad_scale"]), dz
    if kind == "xent_rows":
        logits = s["logits"].detach().requires_grad_(True)
        loss = xent.sparse_softmax_xent(logits, s["labels"])
        return loss.detach(), torch.autograd.grad(loss, logits, s["g"])[0]
    if kind == "ortho":
        return muon.orthogonalize(s["x"])
    muon.muon_step(s["plan"], s["lr"], momentum=s["momentum"], nesterov=s["nesterov"])
    return s["w"], s["buf"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _touched(case):
    """How many rows of the table a batch of ids is expected to hold."""
    v = np.arange(case["rows"], dtype=np.float64)
    p = np.log((v + 2) / (v + 1)) / math.log(case["rows"] + 1)
    return float((1 - np.exp(case["tokens"] * (1 - case["pad"]) * np.log1p(-np.minimum(p, 1 - 1e-12)))).sum())


def work(case):
    kind = case["kind"]
    if kind in ("lookup", "table_grad", "row_sgd"):
        b = 4 if case["dtype"] == "float32" else 2
        t, v, d = case["tokens"], case["rows"], case["dim"]
        rows = _touched(case)
        if kind == "lookup":
            return {"bytes": 8 * t + b * d * (rows + t), "flops": t * d}
        if kind == "table_grad":
            return {"bytes": 8 * t + b * d * (rows + t) + b * d * (t + v), "flops": 3 * t * d}
        return {"bytes": 8 * t + b * d * (t + 2 * rows), "flops": 2 * t * d}
    if kind in ("xent", "xent_rows"):
        b = 4 if case["dtype"] == "float32" else 2
        n = case["tokens"] * case["classes"]
        return {"bytes": 2 * b * n + 12 * case["tokens"], "flops": 6 * n}
    total = {"bytes": 0, "flops": 0}
    for m, n in [(case["m"], case["n"])] if kind == "ortho" else _shapes(case):
        low, high = min(m, n), max(m, n)
        if kind == "ortho":
            total["bytes"] += 2 * m * n * (4 if case["dtype"] == "float32" else 2)
        else:
            total["bytes"] += 5 * 4 * m * n
        # two of the three products of a step have symmetric results: half of each is enough
        total["flops"] += 5 * (low * low * high + low ** 3 + 2 * low * low * high)
    return total


def _exact_factor(u):
    flip = u.shape[0] > u.shape[1]
    y = (u.t() if flip else u).contiguous()
    y = y / (torch.linalg.vector_norm(y) + _EPS)
    eye = torch.eye(y.shape[0], device=y.device, dtype=torch.float64)
    for _ in range(5):
        q = torch.mm(y, y.t().contiguous())
        y = torch.mm(_NS[0] * eye + torch.mm(q, _NS[1] * eye + _NS[2] * q), y)
    return y.t() if flip else y


def _exact_sums(ids, g, rows, scale):
    """Sums by rows through a sorted order and differences at its borders, column blocks at a time."""
    ids = torch.where((ids < 0) | (ids >= rows), rows, ids)
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=rows + 1)[:rows]
    ends = torch.cumsum(counts, 0)
    out = torch.empty(rows, g.shape[1], device=g.device, dtype=torch.float64)
    for a in range(0, g.shape[1], 512):
        run_sum = torch.cumsum(g[order, a:a + 512].double(), 0)
        run_sum = torch.cat([torch.zeros_like(run_sum[:1]), run_sum])
        out[:, a:a + 512] = scale * (run_sum[ends] - run_sum[ends - counts])
    return out


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("lookup", "table_grad", "row_sgd"):
        table, ids = s["table"], s["ids"]
        valid = torch.logical_and(ids >= 0, ids < table.shape[0])
        if kind != "row_sgd":
            out = s["scale"] * table.index_select(0, ids.clamp(0, table.shape[0] - 1)).double()
            out[~valid] = 0
            return out if kind == "lookup" else (out, _exact_sums(ids, s["g"], table.shape[0], s["scale"]))
        return table.double() - float(s["lr"]) * _exact_sums(ids, s["g"], table.shape[0], s["scale"])
    if kind in ("xent", "xent_rows"):
        if s["logits"].numel() > 1 << 32:  # several copies in 64 bits have to fit the card
            return None
        z, labels = s["logits"].double(), s["labels"]
        weight = s["g"].double() if kind == "xent_rows" else torch.full(labels.shape, s["grad_scale"], device="cuda", dtype=torch.float64)
        lse = torch.logsumexp(z, 1)
        rows = torch.arange(z.shape[0], device="cuda")
        loss = lse - z[rows, labels.clamp(min=0)]
        z = z.sub_(lse[:, None]).exp_()
        z[rows, labels.clamp(min=0)] -= 1
        z *= weight[:, None]
        z[labels < 0] = 0
        loss[labels < 0] = 0
        return loss, z
    if kind == "ortho":
        return _exact_factor(s["x"].double())
    ws, bufs = [], []
    for w, g, buf in zip(s["w"], s["g"], s["buf"]):
        new = s["momentum"] * buf.double() + g.double()
        u = g.double() + s["momentum"] * new if s["nesterov"] else new
        ws.append(w.double() - float(s["lr"]) * max(1.0, w.shape[1] / w.shape[0]) ** 0.5 * _exact_factor(u))
        bufs.append(new)
    return ws, bufs
