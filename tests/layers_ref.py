"""64-bit references of the input-layer operators and their error bounds.

u = 2^-24 is half a step of float32 relative to the value. A sum of float32
terms whose longest chain of additions is `depth` long is off by at most
depth * u * (sum of magnitudes) (to first order; the bounds below carry a
factor 1.01 for the higher ones). A result rounded to type t is off by another
finfo(t).eps / 2 of its value, or half the smallest subnormal of t.
"""
import ctypes

import torch

import gids_abi

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# (rows, parameters): every pair the norm takes; (table, rows) of the lookup are
# the pairs with the float32 side as the table
PAIRS = [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")]


def rounding(dtype, ref):
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps / 2) + fi.tiny * fi.eps / 2


def close(got, ref, err, what=""):
    """got (any type) within `err` (float32 arithmetic) and one rounding of ref (float64)."""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = 1.01 * err + 1.01 * rounding(got.dtype, ref.abs() + err)
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (what, float(off.max()), float((off / tol)[bad].max()), int(bad.sum()))


def group_sums(ids, grad, num_rows, skip=None):
    """float64 sums of grad's rows by id and the sums of their magnitudes, [num_rows, dim]; counts [num_rows]."""
    ids = ids.reshape(-1).long()
    g = grad.reshape(ids.numel(), grad.shape[-1]).double()
    keep = (ids >= 0) & (ids < num_rows)
    if skip is not None:
        keep &= ids != skip
    ids, g = ids[keep], g[keep]
    s = torch.zeros((num_rows, g.shape[1]), dtype=torch.float64, device=g.device)
    a, c = torch.zeros_like(s), torch.zeros(num_rows, dtype=torch.float64, device=g.device)
    s.index_add_(0, ids, g)
    a.index_add_(0, ids, g.abs())
    c.index_add_(0, ids, torch.ones_like(ids, dtype=torch.float64))
    return s, a, c


def grad_error(ref_abs, counts, scale, ref):
    # at most count additions one after another, then the product with scale
    return U * (counts[:, None] * ref_abs * abs(scale) + ref.abs())


def norm_ref(x, w, b, eps):
    """(y, mean, rstd, error of y) in 64 bits. The error: the mean of the
    differences and of their squares is a tree whose longest chain is `depth`;
    rstd is off by half the variance's relative error and 3 more roundings."""
    x = x.double()
    d = x.shape[-1]
    depth = d / 512 + 80
    m = x.mean(-1, keepdim=True)
    v = (x - m).square().mean(-1, keepdim=True)
    r = 1 / (v + eps).sqrt()
    xh = (x - m) * r
    wd = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    spread = v.sqrt() * r  # 1 unless eps is large beside the variance
    err = U * wd.abs() * (xh.abs() * (depth / 2 + 8) + spread * (depth + 4)) + 2 * U * ((xh * wd).abs() + bd.abs())
    return xh * wd + bd, m.squeeze(-1), r.squeeze(-1), err


def norm_grad_ref(g, x, mean, rstd, w):
    """((dx, dw, db), (their errors)) in 64 bits, from float32 mean and rstd."""
    g, x, m, r = g.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    n, d = x.shape
    wd = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    xh = (x - m) * r
    t = g * wd
    c0, c1 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    dx = r * (t - c0 - xh * c1)
    depth = d / 512 + 80
    e0 = (depth + 3) * t.abs().mean(1, keepdim=True)
    e1 = (depth + 6) * (t * xh).abs().mean(1, keepdim=True)
    edx = U * r * (e0 + xh.abs() * e1 + 6 * (t.abs() + c0.abs() + (xh * c1).abs()))
    rows = n / 64 + 200  # additions of one column, one after another
    edw = U * (rows + 4) * (g * xh).abs().sum(0)
    edb = U * rows * g.abs().sum(0)
    return (dx, (g * xh).sum(0), g.sum(0)), (edx, edw, edb)


def bits(t):
    t = t.detach().contiguous()
    return t.view({2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()])


_abi = None


def abi():
    """The C ABI with the signatures of the input-layer entry points."""
    global _abi
    if _abi is None:
        L = gids_abi.lib()
        vp, i32, i64, u64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float
        P = ctypes.POINTER
        sig = {
            "gids_embedding": [i32, vp, i32, i64, vp, i32, i64, i64, i64, vp, i32, i64, f32, vp],
            "gids_embedding_check": [i32, vp],
            "gids_embedding_grad_workspace": [i64, i64, i64, P(u64)],
            "gids_embedding_grad": [i32, vp, i32, i64, i64, i64, vp, i32, i64, vp, i32, i64, i64, f32, vp, u64, vp],
            "gids_embedding_group": [i32, vp, i32, i64, i64, i64, i64, vp, u64, vp, P(u64), vp],
            "gids_embedding_grad_rows": [i32, vp, vp, i32, i64, i64, i64, i64, vp, i32, i64, i64, f32, vp, u64, vp],
            "gids_layer_norm": [i32, vp, i64, vp, vp, vp, i32, i64, vp, vp, i32, i64, i64, f32, vp],
            "gids_layer_norm_grad_workspace": [i64, i64, P(u64)],
            "gids_layer_norm_grad": [i32, vp, i64, vp, vp, vp, i64, vp, i32, i64, vp, i32, vp, vp, i64, i64, vp, u64,
                                     vp],
        }
        for name, args in sig.items():
            f = getattr(L, name)
            f.restype, f.argtypes = i32, args
        _abi = L
    return _abi
