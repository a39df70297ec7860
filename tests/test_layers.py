"""Refusals of the input-layer operators on the CPU: the C ABI checks its
arguments before it touches a GPU, and GIDS.layers checks tensors first."""
import ctypes

import pytest
import torch

import gids_abi
from gids_abi import GIDS_E_INVAL, GIDS_E_UNSUPPORTED
from layers_ref import abi

P = 1 << 20  # an aligned address that is never read: every call below is refused
N1 = None


def emb(L, **kw):
    a = dict(device=0, out=P, ot=0, os=8, w=P, wt=0, ws=8, rows=10, dim=8, ids=P, ib=8, n=4, scale=1.0)
    a.update(kw)
    return L.gids_embedding(a["device"], a["out"], a["ot"], a["os"], a["w"], a["wt"], a["ws"], a["rows"], a["dim"],
                            a["ids"], a["ib"], a["n"], a["scale"], None)


def grad(L, **kw):
    a = dict(device=0, dw=P, wt=0, dws=8, rows=10, dim=8, g=P, gt=0, gs=8, ids=P, ib=8, n=4, pad=-1, scale=1.0,
             ws=P, wsb=1 << 30)
    a.update(kw)
    return L.gids_embedding_grad(a["device"], a["dw"], a["wt"], a["dws"], a["rows"], a["dim"], a["g"], a["gt"],
                                 a["gs"], a["ids"], a["ib"], a["n"], a["pad"], a["scale"], a["ws"], a["wsb"], None)


def norm(L, **kw):
    a = dict(device=0, y=P, ys=8, mean=P, rstd=P, x=P, xt=0, xs=8, w=P, b=P, pt=0, n=4, dim=8, eps=1e-5)
    a.update(kw)
    return L.gids_layer_norm(a["device"], a["y"], a["ys"], a["mean"], a["rstd"], a["x"], a["xt"], a["xs"], a["w"],
                             a["b"], a["pt"], a["n"], a["dim"], a["eps"], None)


def norm_grad(L, **kw):
    a = dict(device=0, dx=P, dxs=8, dw=P, db=P, g=P, gs=8, x=P, xt=0, xs=8, w=P, pt=0, mean=P, rstd=P, n=4, dim=8,
             ws=P, wsb=1 << 30)
    a.update(kw)
    return L.gids_layer_norm_grad(a["device"], a["dx"], a["dxs"], a["dw"], a["db"], a["g"], a["gs"], a["x"], a["xt"],
                                  a["xs"], a["w"], a["pt"], a["mean"], a["rstd"], a["n"], a["dim"], a["ws"], a["wsb"],
                                  None)


INVALID = {
    emb: [dict(out=None), dict(w=None), dict(ids=None), dict(n=-1), dict(n=1 << 31), dict(dim=0), dict(dim=1 << 31),
          dict(rows=-1), dict(rows=(1 << 32) - 1), dict(ib=2), dict(ot=3), dict(wt=-1), dict(os=7), dict(os=-8),
          dict(ws=-1), dict(out=P + 2), dict(w=P + 1), dict(ids=P + 4), dict(device=-1), dict(device=64)],
    grad: [dict(dw=None), dict(g=None), dict(ids=None), dict(n=-1), dict(dim=0), dict(ib=3), dict(wt=9), dict(gt=9),
           dict(dws=7), dict(gs=-1), dict(pad=-2), dict(pad=10), dict(ws=None), dict(ws=P + 16), dict(wsb=16),
           dict(device=-1), dict(g=P + 2), dict(ids=P + 4)],
    norm: [dict(y=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(n=-1), dict(dim=0),
           dict(dim=(1 << 24) + 1), dict(eps=-1.0), dict(eps=float("nan")), dict(xt=7), dict(ys=7), dict(xs=-8),
           dict(x=P + 2), dict(w=P + 2), dict(b=P + 1), dict(device=-1)],
    norm_grad: [dict(g=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(n=-1), dict(dim=0), dict(dxs=7),
                dict(gs=-1), dict(ws=None), dict(ws=P + 128), dict(wsb=8), dict(dw=P + 2), dict(db=P + 2),
                dict(w=P + 2), dict(device=-1)],
}


@pytest.mark.parametrize("call,kw", [(c, k) for c, ks in INVALID.items() for k in ks],
                         ids=lambda v: getattr(v, "__name__", None) or ",".join(f"{a}={b}" for a, b in v.items()))
def test_abi_refuses_bad_arguments(built, call, kw):
    assert call(abi(), **kw) == GIDS_E_INVAL
    buf = ctypes.create_string_buffer(256)
    assert gids_abi.lib().gids_last_error(buf, 256) > 0


def test_abi_refuses_type_pairs(built):
    L = abi()
    assert emb(L, wt=1, ot=0) == GIDS_E_UNSUPPORTED  # a 16-bit table gives its own type
    assert emb(L, wt=1, ot=2) == GIDS_E_UNSUPPORTED
    assert grad(L, gt=0, wt=1) == GIDS_E_UNSUPPORTED  # a float32 gradient is not rounded to 16 bits
    assert grad(L, gt=1, wt=2) == GIDS_E_UNSUPPORTED
    assert norm(L, xt=0, pt=1) == GIDS_E_UNSUPPORTED
    assert norm(L, xt=1, pt=2) == GIDS_E_UNSUPPORTED
    assert norm_grad(L, xt=2, pt=1) == GIDS_E_UNSUPPORTED


def test_abi_group_and_rows_refusals(built):
    L = abi()
    u = ctypes.c_uint64()
    cnt = ctypes.byref(u)
    ok = [0, P, 8, 4, 10, -1, 8, P, 1 << 30, P, None, None]
    for i, v in [(0, -1), (1, None), (2, 5), (3, -1), (4, -1), (5, 10), (5, -2), (6, 0), (7, None), (7, P + 64), (8, 1)]:
        a = list(ok)
        a[i] = v
        assert L.gids_embedding_group(*a) == GIDS_E_INVAL, (i, v)
    ok = [0, P, P, 0, 8, 3, 10, 8, P, 0, 8, 4, 1.0, P, 1 << 30, None]
    for i, v in [(0, -1), (1, None), (1, P + 4), (2, None), (3, 4), (4, 7), (5, -1), (6, -1), (7, 0), (8, None),
                 (10, -1), (11, -1), (13, None), (14, 4)]:
        a = list(ok)
        a[i] = v
        assert L.gids_embedding_grad_rows(*a) == GIDS_E_INVAL, (i, v)
    assert L.gids_embedding_grad_workspace(-1, 10, 8, cnt) == GIDS_E_INVAL
    assert L.gids_embedding_grad_workspace(4, 10, 8, None) == GIDS_E_INVAL
    assert L.gids_layer_norm_grad_workspace(4, 0, cnt) == GIDS_E_INVAL
    assert L.gids_layer_norm_grad_workspace(4, 8, None) == GIDS_E_INVAL
    assert L.gids_embedding_grad_workspace(1000, 10, 8, cnt) == 0 and u.value > 2 * 8000
    assert L.gids_layer_norm_grad_workspace(1000, 8, cnt) == 0 and u.value >= 64


def test_python_refuses_bad_tensors(built):
    from GIDS import layers

    ids, w, x = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4), torch.zeros(3, 4)
    st = torch.zeros(3)
    for call in (
        lambda: layers.embedding(ids, w),  # CPU tensors
        lambda: layers.embedding(ids.float(), w),
        lambda: layers.embedding(ids, w[0]),
        lambda: layers.embedding(ids, w.double()),
        lambda: layers.embedding(ids, w, dtype=torch.int32),
        lambda: layers.embedding(ids, w, padding_idx=5),
        lambda: layers.embedding(ids, w, padding_idx=-6),
        lambda: layers.embedding(ids, w.t()),
        lambda: layers.embedding_grad(ids, x, 5),
        lambda: layers.embedding_grad(ids[:2], x, 5),
        lambda: layers.embedding_grad(ids, x[:, :0], 5),
        lambda: layers.embedding_grad_rows(ids, x.double(), 5),
        lambda: layers.layer_norm(x),
        lambda: layers.layer_norm(x.double()),
        lambda: layers.layer_norm(x[:, :0]),
        lambda: layers.layer_norm(x, torch.ones(3)),
        lambda: layers.layer_norm(x, torch.ones(4), torch.zeros(4, dtype=torch.float16)),
        lambda: layers.layer_norm(x, torch.ones(4, dtype=torch.float16)),
        lambda: layers.layer_norm(x, torch.ones(8)[::2]),
        lambda: layers.layer_norm_grad(x, x, st, st),
        lambda: layers.layer_norm_grad(x[:2], x, st, st),
        lambda: layers.layer_norm_grad(x.half(), x, st, st),
        lambda: layers.layer_norm_grad(x, x, st, st, param_dtype=torch.float16),
    ):
        with pytest.raises(ValueError):
            call()


def test_modules_build_on_cpu():
    from GIDS import layers

    e = layers.NodeEmbedding(10, 6, padding_idx=-1, dtype=torch.bfloat16)
    assert e.weight.shape == (10, 6) and e.padding_idx == 9 and not e.weight[9].any() and e.weight[:9].any()
    n = layers.LayerNorm(6, bias=False)
    assert n.bias is None and n.weight.shape == (6,)
    assert layers.LayerNorm(6, affine=False).weight is None
    assert "padding_idx=9" in repr(e) and "eps=1e-05" in repr(n)


def test_abi_distinct_refusals(built):
    L = abi()
    u = ctypes.c_uint64()
    f = L.gids_embedding_grad_distinct
    vp, i32, i64, u64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float
    f.restype = i32
    f.argtypes = [i32, vp, vp, i32, i64, i64, i64, i64, vp, i32, i64, vp, i32, i64, i64, f32, vp, u64,
                  ctypes.POINTER(u64), vp]
    ok = [0, P, P, 0, 8, 4, 10, 8, P, 0, 8, P, 8, 4, -1, 1.0, P, 1 << 30, ctypes.byref(u), None]
    for i, v in [(0, -1), (1, None), (2, None), (3, 9), (4, 7), (5, 3), (6, -1), (7, 0), (8, None), (9, 9), (10, -1),
                 (11, None), (12, 3), (13, -1), (14, 10), (16, None), (17, 8), (18, None)]:
        a = list(ok)
        a[i] = v
        assert f(*a) == GIDS_E_INVAL, (i, v)
    a = list(ok)
    a[3] = 1
    assert f(*a) == GIDS_E_UNSUPPORTED


def test_abi_small_calls_may_go_without_a_workspace(built):
    """NULL with 0 bytes is refused where a workspace is needed, and not before the other arguments are
    looked at where none is; NULL with a size is an error everywhere."""
    L = abi()
    none = dict(ws=None, wsb=0)
    assert grad(L, n=129, **none) == GIDS_E_INVAL
    assert grad(L, n=128, ws=None, wsb=256) == GIDS_E_INVAL
    for n, d in ((2049, 128), (2049, 1), (65, 4096), (1, 4097), (1 << 37, 8)):
        assert norm_grad(L, n=n, dim=d, dxs=d, gs=d, xs=d, **none) == GIDS_E_INVAL, (n, d)
    assert norm_grad(L, n=4, dim=8, ws=None, wsb=8) == GIDS_E_INVAL
    u = ctypes.c_uint64()
    a = [0, P, 8, 4, 10, -1, 8, None, 0, P, None, None]
    assert L.gids_embedding_group(*a) == GIDS_E_INVAL
    b = [0, P, P, 0, 8, 3, 10, 8, P, 0, 8, 4, 1.0, None, 0, None]
    assert L.gids_embedding_grad_rows(*b) == GIDS_E_INVAL
    vp, i32, i64, u64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float
    f = L.gids_embedding_grad_distinct
    f.argtypes = [i32, vp, vp, i32, i64, i64, i64, i64, vp, i32, i64, vp, i32, i64, i64, f32, vp, u64,
                  ctypes.POINTER(u64), vp]
    assert f(0, P, P, 0, 8, 10, 10, 8, P, 0, 8, P, 8, 129, -1, 1.0, None, 0, ctypes.byref(u), None) == GIDS_E_INVAL


def test_few_constants_match_the_header(built):
    import pathlib
    import re

    from GIDS import layers

    text = (pathlib.Path(gids_abi.__file__).parents[1] / "include" / "gids_b200.h").read_text()
    assert int(re.search(r"#define GIDS_FEW_IDS (\d+)", text)[1]) == layers._FEW_IDS
    assert eval(re.search(r"#define GIDS_FEW_NORM (.+)", text)[1]) == layers._FEW_NORM


def test_abi_refuses_an_unaligned_count(built):
    """The kernels store the number of rows as one 64-bit word."""
    L = abi()
    for off in (1, 2, 4):
        a = [0, P, 8, 4, 10, -1, 8, P, 1 << 30, P + off, None, None]
        assert L.gids_embedding_group(*a) == GIDS_E_INVAL, off
    a = [0, None, 8, 0, 10, -1, 8, P, 1 << 30, P + 4, None, None]  # no ids: still set
    assert L.gids_embedding_group(*a) == GIDS_E_INVAL
