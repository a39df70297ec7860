"""Cases of the input-layer operators: embedding lookup with scaling, its gradient
(dense, and as the distinct rows), layer norm and its gradient.

``run`` computes a case with elementary torch operations, or, where ``own`` is
true, with the calls a user makes of ``GIDS.layers``. ``exact`` is the same
value from the definition in 64 bits, by other means than the plain form.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


@functools.cache
def _layers():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "gids-study_b200")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    from GIDS import layers

    return layers


# ---------------------------------------------------------------------- cases
def _emb(n, rows, dim, distinct, table, out, skew, scale):
    return {"op": "embedding", "n": n, "rows": rows, "dim": dim, "distinct": distinct, "table": table, "out": out,
            "skew": skew, "scale": scale, "pad": 0}


def _grad(op, n, rows, dim, distinct, grad, out, skew, scale, pad):
    """``pad`` of the n ids are the padding row 0; the others are ``distinct`` rows."""
    return {"op": op, "n": n, "rows": rows, "dim": dim, "distinct": distinct, "grad": grad, "out": out, "skew": skew,
            "scale": scale, "pad": pad}


def _ln(op, n, dim, x, param, affine=True):
    return {"op": op, "n": n, "dim": dim, "x": x, "param": param, "affine": affine}


def listed():
    return [
        # the rows of a handful of nodes or tokens (a serving step): latency
        dict(_emb(8, 50000, 1024, 8, "bf16", "bf16", 3.0, 32.0), name="embedding_few"),
        # a training minibatch from a float32 master table into a 16-bit model, an odd count
        dict(_emb(65521, 1000000, 1024, 59999, "f32", "bf16", 2.0, 1.0), name="embedding_master"),
        # a sampled neighbourhood's rows of a node type without stored features
        dict(_emb(1000003, 4000000, 768, 790001, "f16", "f16", 1.5, 0.5), name="embedding_neighbourhood"),
        # a small vocabulary (types, positions) with a short batch: latency
        dict(_grad("embedding_grad", 64, 5000, 128, 57, "f32", "f32", 2.0, 1.0, 0), name="grad_dense_few"),
        # a language model's vocabulary, skewed tokens, a quarter of the batch padding
        dict(_grad("embedding_grad", 16384, 100003, 1024, 5003, "bf16", "bf16", 4.0, 32.0, 4096), name="grad_dense_tokens"),
        # a minibatch of 512-byte rows out of a table too large for a dense gradient
        dict(_grad("embedding_grad_rows", 500009, 10000000, 128, 450001, "f32", "f32", 2.0, 1.0, 0), name="grad_rows_nodes"),
        # long segments: few hot rows take most of the batch; 16-bit gradients of a float32 table
        dict(_grad("embedding_grad_rows", 131072, 200000, 1024, 15013, "bf16", "f32", 6.0, 1.0, 13107), name="grad_rows_hot"),
        # the norm of a handful of rows: latency
        dict(_ln("layer_norm", 4, 1024, "bf16", "bf16"), name="norm_few"),
        # a minibatch's 16-bit features with float32 weights, an odd count
        dict(_ln("layer_norm", 262139, 768, "f16", "f32"), name="norm_features"),
        # a sampled neighbourhood's float32 features
        dict(_ln("layer_norm", 1000003, 1024, "f32", "f32"), name="norm_neighbourhood"),
        # a small batch's backward pass: latency and the reduction over few rows
        dict(_ln("layer_norm_grad", 129, 768, "f16", "f32"), name="norm_grad_few"),
        # the backward pass of a large minibatch
        dict(_ln("layer_norm_grad", 262144, 1024, "bf16", "bf16"), name="norm_grad_large"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _dim(rng, hi=8192):
    d = _log_int(rng, 8, hi)
    kind = rng.random()
    if kind < 0.6:  # rows of whole 128-byte lines
        d = max(64, d // 64 * 64)
    elif kind < 0.8:  # rows of whole 16-byte vectors
        d = max(8, d // 8 * 8)
    return d


def draw(rng):
    budget = max(_bytes(c) for c in listed())
    while True:
        op = rng.choice(["embedding", "embedding_grad", "embedding_grad_rows", "layer_norm", "layer_norm_grad"])
        n = _log_int(rng, 1, 1000000)
        dim = _dim(rng)
        dt = rng.choice(["f32", "f16", "bf16"])
        mixed = rng.random() < 0.4
        skew = round(rng.uniform(1.0, 6.0), 2)
        scale = rng.choice([1.0, 1.0, 0.125, round(math.sqrt(dim), 3)])
        if op == "embedding":
            rows = _log_int(rng, 1000, 10000000)
            case = _emb(n, rows, dim, _log_int(rng, max(1, min(n, rows) // 50), min(n, rows)),
                        "f32" if mixed else dt, dt, skew, scale)
        elif op in ("embedding_grad", "embedding_grad_rows"):
            rows = _log_int(rng, 1000, 300000 if op == "embedding_grad" else 100000000)
            pad = int(n * rng.choice([0.0, 0.0, 0.1, 0.5]))
            most = min(n - pad, rows - 1)
            case = _grad(op, n, rows, dim, _log_int(rng, max(1, most // 50), most), dt, "f32" if mixed else dt, skew,
                         scale, pad)
        else:
            case = _ln(op, n, dim, dt, "f32" if mixed else dt, rng.random() < 0.85)
        held = case["rows"] * dim * _BYTES[case["table"]] if op == "embedding" else 0
        if _bytes(case) <= budget and held <= 16 << 30:
            return case


# ---------------------------------------------------------------------- work
def _bytes(case):
    n, d, op = case["n"], case["dim"], case["op"]
    if op == "embedding":
        return 8 * n + case["distinct"] * d * _BYTES[case["table"]] + n * d * _BYTES[case["out"]]
    if op in ("embedding_grad", "embedding_grad_rows"):
        read = 8 * n + (n - case["pad"]) * d * _BYTES[case["grad"]]
        if op == "embedding_grad":
            return read + case["rows"] * d * _BYTES[case["out"]]
        return read + case["distinct"] * (8 + d * _BYTES[case["out"]])
    e, p = _BYTES[case["x"]], _BYTES[case["param"]] if case["affine"] else 0
    if op == "layer_norm":
        return 2 * n * d * e + 2 * d * p
    return 3 * n * d * e + 8 * n + 3 * d * p


def work(case):
    n, d = case["n"], case["dim"]
    per = {"embedding": 1, "embedding_grad": 1, "embedding_grad_rows": 1, "layer_norm": 8, "layer_norm_grad": 14}
    return {"bytes": int(_bytes(case)), "flops": per[case["op"]] * n * d}


# -------------------------------------------------------------------- inputs
def _ids(case, gen, dev):
    """``distinct`` rows spread over the table by an odd multiplier: each once, the
    rest of the batch by a power law (the larger ``skew``, the hotter the
    head), in random order; ``pad`` ids are row 0, which no other id is then."""
    n, distinct, pad = case["n"] - case["pad"], case["distinct"], case["pad"]
    rows, first = (case["rows"] - 1, 1) if pad else (case["rows"], 0)
    mult = 2654435761
    while math.gcd(mult, rows) != 1:
        mult += 2
    start = torch.randint(rows, (1,), generator=gen, device=dev)
    u = torch.rand(n - distinct, generator=gen, device=dev, dtype=torch.float64)
    rank = torch.cat([torch.arange(distinct, device=dev),
                      (u.pow(case["skew"]) * distinct).long().clamp_(max=distinct - 1)])
    ids = torch.cat([first + (rank * mult + start) % rows, torch.zeros(pad, dtype=torch.int64, device=dev)])
    return ids[torch.randperm(case["n"], generator=gen, device=dev)]


def _normal(shape, dtype, gen, dev):
    return torch.randn(shape, generator=gen, device=dev, dtype=dtype)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op, n, d = case["op"], case["n"], case["dim"]
    st = {"case": case}
    if op == "embedding":
        st["ids"] = _ids(case, gen, dev)
        st["weight"] = _normal((case["rows"], d), _DT[case["table"]], gen, dev).mul_(0.05)
        return st
    if op in ("embedding_grad", "embedding_grad_rows"):
        st["ids"] = _ids(case, gen, dev)
        st["grad"] = _normal((n, d), _DT[case["grad"]], gen, dev)
        return st
    x = _normal((n, d), _DT[case["x"]], gen, dev)
    # features have a mean and a spread of their own in every column
    x.mul_(torch.rand(d, generator=gen, device=dev).add_(0.5).to(x.dtype))
    x.add_(torch.rand(d, generator=gen, device=dev).to(x.dtype))
    st["x"] = x
    st["weight"] = st["bias"] = None
    if case["affine"]:
        st["weight"] = _normal((d,), torch.float32, gen, dev).mul_(0.1).add_(1.0).to(_DT[case["param"]])
        st["bias"] = _normal((d,), torch.float32, gen, dev).mul_(0.1).to(_DT[case["param"]])
    if op == "layer_norm_grad":
        st["grad"] = _normal((n, d), _DT[case["x"]], gen, dev)
        # the statistics that the forward pass has kept
        st["mean"] = torch.empty(n, dtype=torch.float32, device=dev)
        st["rstd"] = torch.empty(n, dtype=torch.float32, device=dev)
        for lo in range(0, n, 65536):
            v = x[lo:lo + 65536].double()
            m = v.mean(1, keepdim=True)
            st["mean"][lo:lo + 65536] = m.squeeze(1).float()
            st["rstd"][lo:lo + 65536] = ((v - m).square().mean(1) + EPS).rsqrt().float()
    return st


# ----------------------------------------------------------------------- run
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    c, op = st["case"], st["case"]["op"]
    layers = _layers()
    if op == "embedding":
        return layers.embedding(st["ids"], st["weight"], scale=c["scale"], dtype=_DT[c["out"]])
    if op == "embedding_grad":
        return layers.embedding_grad(st["ids"], st["grad"], c["rows"], scale=c["scale"],
                                     padding_idx=0 if c["pad"] else None, dtype=_DT[c["out"]])
    if op == "embedding_grad_rows":
        return layers.embedding_grad_rows(st["ids"], st["grad"], c["rows"], scale=c["scale"],
                                          padding_idx=0 if c["pad"] else None, dtype=_DT[c["out"]])
    if op == "layer_norm":
        return layers.layer_norm(st["x"], st["weight"], st["bias"], eps=EPS)
    grads = layers.layer_norm_grad(st["grad"], st["x"], st["mean"], st["rstd"], st["weight"])
    return grads if c["affine"] else grads[:1]


def _run_plain(st):
    c, op = st["case"], st["case"]["op"]
    if op == "embedding":
        return (st["weight"][st["ids"]].float() * c["scale"]).to(_DT[c["out"]])
    if op in ("embedding_grad", "embedding_grad_rows"):
        ids, grad = st["ids"], st["grad"]
        if c["pad"]:
            keep = ids != 0
            ids, grad = ids[keep], grad[keep]
        # hot rows are long sums: 64 bits
        if op == "embedding_grad":
            acc = torch.zeros((c["rows"], c["dim"]), dtype=torch.float64, device=ids.device)
            acc.index_add_(0, ids, grad.double())
            return (acc * c["scale"]).to(_DT[c["out"]])
        rows, slot = torch.unique(ids, sorted=True, return_inverse=True)
        acc = torch.zeros((rows.numel(), c["dim"]), dtype=torch.float64, device=ids.device)
        acc.index_add_(0, slot, grad.double())
        return rows, (acc * c["scale"]).to(_DT[c["out"]])
    x = st["x"].float()
    w = st["weight"].float() if c["affine"] else None
    if op == "layer_norm":
        xc = x - x.mean(1, keepdim=True)
        y = xc * torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
        if c["affine"]:
            y = y * w + st["bias"].float()
        return y.to(st["x"].dtype)
    g = st["grad"].float()
    xh = (x - st["mean"][:, None]) * st["rstd"][:, None]
    t = g * w if c["affine"] else g
    dx = st["rstd"][:, None] * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
    if not c["affine"]:
        return (dx.to(st["x"].dtype),)
    # sums over every row of the batch: 64 bits
    dw = (g * xh).sum(0, dtype=torch.float64)
    db = g.sum(0, dtype=torch.float64)
    return dx.to(st["x"].dtype), dw.to(st["weight"].dtype), db.to(st["weight"].dtype)


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """The definition in 64 bits, row block by row block."""
    st = prepare(case, seed)
    op, n, d = case["op"], case["n"], case["dim"]
    if op == "embedding":
        out = torch.empty((n, d), dtype=torch.float64, device=st["ids"].device)
        for lo in range(0, n, 65536):
            part = torch.index_select(st["weight"], 0, st["ids"][lo:lo + 65536])
            out[lo:lo + 65536] = part.double() * case["scale"]
        return out
    if op in ("embedding_grad", "embedding_grad_rows"):
        ids, order = torch.sort(st["ids"], stable=True)
        if case["pad"]:
            order, ids = order[ids != 0], ids[ids != 0]
        rows, counts = torch.unique_consecutive(ids, return_counts=True)
        ends = torch.cumsum(counts, 0)
        sums = torch.empty((rows.numel(), d), dtype=torch.float64, device=ids.device)
        step = max(1, (1 << 27) // max(1, order.numel()))
        for lo in range(0, d, step):  # differences of the running sum along the sorted rows
            run_sum = torch.cumsum(st["grad"][:, lo:lo + step][order].double(), 0)
            upto = run_sum[ends - 1]
            sums[:, lo:lo + step] = torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1])) if len(rows) else upto
        sums *= case["scale"]
        if op == "embedding_grad_rows":
            return None, sums
        full = torch.zeros((case["rows"], d), dtype=torch.float64, device=ids.device)
        full[rows] = sums
        return full
    w = st["weight"].double() if case["affine"] else torch.ones(d, dtype=torch.float64, device=st["x"].device)
    if op == "layer_norm":
        b = st["bias"].double() if case["affine"] else torch.zeros_like(w)
        out = torch.empty((n, d), dtype=torch.float64, device=w.device)
        for lo in range(0, n, 65536):
            v = st["x"][lo:lo + 65536].double()
            var, mean = torch.var_mean(v, 1, correction=0, keepdim=True)
            out[lo:lo + 65536] = torch.addcmul(b, (v - mean) / torch.sqrt(var + EPS), w)
        return out
    dx = torch.empty((n, d), dtype=torch.float64, device=w.device)
    dw, db = torch.zeros_like(w), torch.zeros_like(w)
    for lo in range(0, n, 65536):
        part = slice(lo, lo + 65536)
        g, r = st["grad"][part].double(), st["rstd"][part].double()
        xh = (st["x"][part].double() - st["mean"][part].double()[:, None]) * r[:, None]
        c2, c1 = torch.mv(g, w) / d, torch.mv(g * xh, w) / d
        dx[part] = r[:, None] * (g * w - c2[:, None] - xh * c1[:, None])
        dw += torch.einsum("ij,ij->j", g, xh)
        db += torch.einsum("ij->j", g)
    return (dx, dw, db) if case["affine"] else (dx,)
