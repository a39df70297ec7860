"""The input-layer operators (csrc/embedding.cu, csrc/layer_norm.cu) against
64-bit references, through GIDS.layers and the C ABI: every type pair, one row
to many, odd widths, strides, empty inputs, ids outside the table, long runs of
one id, and the ways they are called (streams, graphs, autograd, in place)."""
import ctypes

import pytest
import torch

import gids_abi
from gids_abi import GIDS_E_RANGE, GIDS_E_STATE, check
from layers_ref import (CODES, PAIRS, TYPES, U, abi, bits, close, grad_error, group_sums, norm_grad_ref, norm_ref)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def layers(built):
    from GIDS import layers

    return layers


def randn(*shape, seed=0, dtype="f32"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(TYPES.get(dtype, dtype))


def randint(hi, shape, seed=0, dtype=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, hi, shape, generator=g, device=DEV, dtype=dtype)


# ------------------------------------------------------------------- lookup
def check_embedding(layers, ids, w, scale, dtype):
    out = layers.embedding(ids, w, scale=scale, dtype=dtype)
    assert out.shape == (*ids.shape, w.shape[1]) and out.dtype == dtype
    ref = w.double()[ids.long()] * scale
    close(out, ref, U * ref.abs(), (ids.shape, tuple(w.shape)))


@pytest.mark.parametrize("table,out", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"),
                                       ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [1, 2, 3, 8, 31, 128, 130, 1000, 1001, 1024, 8192])
def test_embedding_types_and_widths(layers, table, out, dim):
    w = randn(500, dim, seed=dim, dtype=table)
    for n in (1, 5, 257):
        check_embedding(layers, randint(500, (n,), seed=n), w, 32.0, TYPES[out])
    check_embedding(layers, randint(500, (3, 7), dtype=torch.int32), w, 0.75, TYPES[out])


def test_embedding_is_exact_without_scale(layers):
    for t in TYPES:
        w = randn(300, 96, dtype=t)
        w[5, :3] = torch.tensor([float("inf"), float("nan"), -0.0], device=DEV)
        ids = randint(300, (1000,))
        ids[:4] = 5
        assert torch.equal(bits(layers.embedding(ids, w)), bits(w[ids]))


def test_embedding_shapes_and_strides(layers):
    w = randn(200, 64)
    assert layers.embedding(torch.zeros(0, dtype=torch.int64, device=DEV), w).shape == (0, 64)
    assert layers.embedding(torch.zeros((2, 0), dtype=torch.int64, device=DEV), w).shape == (2, 0, 64)
    assert layers.embedding(torch.zeros((), dtype=torch.int64, device=DEV), w).shape == (64,)
    assert layers.embedding(randint(200, (4,)), w[:, :0]).shape == (4, 0)
    ids = randint(100, (60,))
    for view in (w[:, 3:50], w[::2], w[:, :33], w[1:, 1:2], randn(100, 1).expand(100, 1), w[:1].expand(100, 64)):
        i = ids.clamp(max=view.shape[0] - 1)
        check_embedding(layers, i, view, 2.0, torch.float32)
        check_embedding(layers, i[::3], view, 1.0, torch.bfloat16)


def test_embedding_ids_outside_the_table(layers):
    w = randn(100, 40)
    for bad in (100, -1, 1 << 40, -(1 << 62)):
        ids = randint(100, (50,))
        ids[7] = bad
        out = layers.embedding(ids, w)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside its table"):
            layers.embedding(ids[:1], w)
        good = torch.arange(50, device=DEV) != 7
        assert torch.equal(out[good], w[ids[good]]) and not out[7].any()
        layers.embedding(ids[:1], w)  # reported once
        layers.check_ids(DEV)
    ids = randint(100, (50,), dtype=torch.int32)
    ids[0] = -5
    layers.embedding(ids, w)
    with pytest.raises(RuntimeError, match="outside its table"):
        layers.check_ids()
    layers.check_ids()


def test_embedding_abi_row_strides_leave_gaps(layers):
    L = abi()
    w = randn(50, 20)
    ids = randint(50, (33,))
    out = torch.full((33, 29), 7.0, device=DEV)
    check(L.gids_embedding(0, out[:, 2:].data_ptr(), 0, 29, w.data_ptr(), 0, 20, 50, 20, ids.data_ptr(), 8, 33, 1.0,
                           None))
    torch.cuda.synchronize()
    assert torch.equal(out[:, 2:22], w[ids]) and bool((out[:, :2] == 7).all()) and bool((out[:, 22:] == 7).all())


def test_embedding_of_a_table_past_32_bit_offsets(layers):
    rows, dim = (1 << 22) + 3, 1024  # 2^32 elements and more
    w = torch.empty((rows, dim), dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([0, rows - 1, rows // 2 + 1, (1 << 21) + 1, rows - 1], device=DEV)
    w[ids] = randn(5, dim, dtype="bf16")
    assert torch.equal(bits(layers.embedding(ids, w)), bits(w[ids]))


# ----------------------------------------------------------- lookup's gradient
def check_grad(layers, ids, grad, num_rows, scale=1.0, pad=None, dtype=None):
    dtype = grad.dtype if dtype is None else dtype
    skip = None if pad is None else pad % num_rows
    s, a, c = group_sums(ids, grad, num_rows, skip)
    ref, err = s * scale, grad_error(a, c, scale, s * scale)
    dw = layers.embedding_grad(ids, grad, num_rows, scale, pad, dtype)
    assert dw.dtype == dtype
    close(dw, ref, err, "dense")
    rows, values = layers.embedding_grad_rows(ids, grad, num_rows, scale, pad, dtype)
    assert rows.dtype == torch.int64 and torch.equal(rows, torch.nonzero(c).squeeze(1))
    assert torch.equal(bits(values), bits(dw[rows]))  # the same sums, in the same order
    again = layers.embedding_grad(ids, grad, num_rows, scale, pad, dtype)
    assert torch.equal(bits(again), bits(dw))


@pytest.mark.parametrize("grad,out", [("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("f16", "f16"),
                                      ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [1, 3, 8, 24, 128, 129, 510, 1024, 2048])
def test_grad_types_and_widths(layers, grad, out, dim):
    for n, rows in ((1, 1), (7, 3), (100, 40), (1000, 64)):
        check_grad(layers, randint(rows, (n,), seed=n), randn(n, dim, seed=n, dtype=grad), rows, 0.5, None, TYPES[out])


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 511, 513, 1023, 1025, 2047, 2048, 2049, 4096, 5000, 65536,
                               303109])
def test_grad_lengths(layers, n):
    for seed, rows in enumerate((1, 2, 1000, 70001)):
        ids = randint(rows, (n,), seed=seed)
        check_grad(layers, ids, randn(n, 16, seed=n), rows)


@pytest.mark.parametrize("rows", [1, 2, 3, 255, 256, 511, 512, 513, 4097, 262143, 262144, 262145, 3000000])
def test_grad_table_sizes(layers, rows):
    for n in (40, 3000):
        ids = torch.cat([randint(rows, (n,), seed=rows), torch.tensor([0, rows - 1, rows // 2], device=DEV)])
        check_grad(layers, ids, randn(n + 3, 4, seed=3), rows, 3.0, None)


@pytest.mark.parametrize("rows", [1 << 27, (1 << 31) + 5, (1 << 32) - 2])
def test_grad_rows_of_huge_tables(layers, rows):
    for n in (50, 4000):
        base = randint(1 << 62, (n,), seed=n) % rows
        ids = torch.cat([base, base[: n // 2], torch.tensor([0, rows - 1, rows - 1], device=DEV)])
        g = randn(len(ids), 8)
        r, v = layers.embedding_grad_rows(ids, g, rows, 1.0)
        want, inv = torch.unique(ids, return_inverse=True)
        s, a, c = group_sums(inv, g, len(want))
        assert torch.equal(r, want)
        close(v, s, grad_error(a, c, 1.0, s))


@pytest.mark.parametrize("n", [64, 5000, 300000])
def test_grad_long_runs_of_one_id(layers, n):
    # all the same; runs that start and end inside chunks, at their borders, and span many
    for lead in (0, 1, 31, 32, 33, 64, 100):
        if lead >= n:
            continue
        ids = torch.full((n,), 5, device=DEV)
        ids[:lead] = torch.arange(lead, device=DEV) % 5
        ids[n - 1] = 9
        perm = torch.randperm(n, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
        check_grad(layers, ids[perm], randn(n, 24, seed=lead, dtype="bf16"), 10, 1.0, None, torch.float32)


def test_grad_skewed_ids_of_two_runs(layers):
    n = 200000
    u = torch.rand(n, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    ids = (u ** 8 * 5000).long()
    check_grad(layers, ids, randn(n, 136, dtype="f16"), 5003, 0.125, 0)


def test_grad_padding(layers):
    g = randn(500, 32)
    ids = randint(50, (500,))
    for pad in (0, 49, -1, -50, 7):
        check_grad(layers, ids, g, 50, 2.0, pad)
    same = torch.full((500,), 7, device=DEV)
    assert not layers.embedding_grad(same, g, 50, padding_idx=7).any()
    rows, values = layers.embedding_grad_rows(same, g, 50, padding_idx=7)
    assert rows.shape == (0,) and values.shape == (0, 32)


def test_grad_padding_rows_are_never_read(layers):
    # what a padded position's gradient holds does not matter
    for n in (40, 3000):
        g = randn(n, 16)
        ids = randint(20, (n,))
        g[ids == 3] = float("nan")
        dw = layers.embedding_grad(ids, g, 20, padding_idx=3)
        assert bool(torch.isfinite(dw).all()) and not dw[3].any()
        # an infinite or NaN gradient stays in its own row
        g = randn(n, 16)
        g[0, 2] = float("inf")
        dw = layers.embedding_grad(ids, g, 20)
        other = torch.ones_like(dw, dtype=torch.bool)
        other[ids[0], 2] = False
        assert torch.isinf(dw[ids[0], 2]) and bool(torch.isfinite(dw[other]).all())


def test_grad_ids_outside_the_table(layers):
    for n in (40, 3000):
        g = randn(n, 16)
        for bad in (30, -1, 1 << 33, -(1 << 50)):
            ids = randint(30, (n,))
            ids[4] = bad
            s, a, c = group_sums(ids, g, 30)
            dw = layers.embedding_grad(ids, g, 30)
            close(dw, s, grad_error(a, c, 1.0, s))
            with pytest.raises(RuntimeError, match="outside its table"):
                layers.check_ids(DEV)
            rows, values = layers.embedding_grad_rows(ids, g, 30)
            with pytest.raises(RuntimeError, match="outside its table"):
                layers.check_ids(DEV)
            assert torch.equal(rows, torch.nonzero(c).squeeze(1)) and torch.equal(bits(values), bits(dw[rows]))
    none = torch.full((10,), 99, device=DEV)
    assert not layers.embedding_grad(none, randn(10, 16), 30).any()
    with pytest.raises(RuntimeError):
        layers.check_ids(DEV)
    rows, _ = layers.embedding_grad_rows(none, randn(10, 16), 30)
    assert rows.numel() == 0
    with pytest.raises(RuntimeError):
        layers.check_ids(DEV)


def test_grad_empty(layers):
    ids = torch.zeros(0, dtype=torch.int64, device=DEV)
    g = torch.zeros((0, 8), device=DEV)
    assert torch.equal(layers.embedding_grad(ids, g, 12), torch.zeros((12, 8), device=DEV))
    assert layers.embedding_grad(ids, g, 0).shape == (0, 8)
    rows, values = layers.embedding_grad_rows(ids, g, 12)
    assert rows.shape == (0,) and values.shape == (0, 8)


def test_grad_strides(layers):
    base = randn(300, 80)
    ids = randint(40, (300,))
    for view in (base[:, :64], base[:, 3:67], base[:, 1:], base[::1, ::2], base[:1].expand(300, 80),
                 base[:, :1].expand(300, 80), torch.ones((), device=DEV).expand(300, 16)):
        check_grad(layers, ids, view, 40)
    check_grad(layers, ids.view(30, 10), base.view(30, 10, 80), 40)
    check_grad(layers, ids.view(10, 30).t(), base.view(30, 10, 80), 40)


def test_grad_abi_writes_only_its_rows(layers):
    L = abi()
    n, rows, dim = 200, 60, 20
    ids, g = randint(rows, (n,)), randn(n, dim)
    b = ctypes.c_uint64()
    check(L.gids_embedding_grad_workspace(n, rows, dim, ctypes.byref(b)))
    ws = torch.empty(b.value, dtype=torch.uint8, device=DEV)
    dw = torch.full((rows + 2, 29), 7.0, device=DEV)
    check(L.gids_embedding_grad(0, dw[1:, 2:].data_ptr(), 0, 29, rows, dim, g.data_ptr(), 0, dim, ids.data_ptr(), 8, n,
                                -1, 1.0, ws.data_ptr(), b.value, None))
    torch.cuda.synchronize()
    assert torch.equal(dw[1:-1, 2:22], layers.embedding_grad(ids, g, rows))
    dw[1:-1, 2:22] = 7.0
    assert bool((dw == 7.0).all())
    # fewer result rows than distinct ids: the first `capacity` of them, nothing behind
    count = torch.zeros(1, dtype=torch.int64, device=DEV)
    check(L.gids_embedding_group(0, ids.data_ptr(), 8, n, rows, -1, dim, ws.data_ptr(), b.value, count.data_ptr(),
                                 None, None))
    cap = 11
    r = torch.full((rows,), -9, dtype=torch.int64, device=DEV)
    v = torch.full((rows, dim), 7.0, device=DEV)
    check(L.gids_embedding_grad_rows(0, r.data_ptr(), v.data_ptr(), 0, dim, cap, rows, dim, g.data_ptr(), 0, dim, n,
                                     1.0, ws.data_ptr(), b.value, None))
    want_r, want_v = layers.embedding_grad_rows(ids, g, rows)
    assert int(count) == len(want_r)
    assert torch.equal(r[:cap], want_r[:cap]) and torch.equal(v[:cap], want_v[:cap])
    assert bool((r[cap:] == -9).all()) and bool((v[cap:] == 7).all())


# ------------------------------------------------------------------ layer norm
def norm_inputs(n, d, pair, seed=0):
    x = randn(n, d, seed=seed) * (0.5 + torch.rand(d, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV))
    x = (x + 0.3).to(TYPES[pair[0]])
    w = (1 + 0.2 * randn(d, seed=seed + 1)).to(TYPES[pair[1]])
    b = (0.2 * randn(d, seed=seed + 2)).to(TYPES[pair[1]])
    return x, w, b


def check_norm(layers, x, w, b, eps=1e-5):
    y, mean, rstd = layers.layer_norm_stats(x, w, b, eps)
    x2 = x.reshape(-1, x.shape[-1])
    ref, m, r, err = norm_ref(x2, w, b, eps)
    close(y.reshape(x2.shape), ref, err, (tuple(x.shape), x.dtype))
    depth = x.shape[-1] / 512 + 90
    close(mean, m, U * depth * x2.double().abs().mean(1), "mean")
    close(rstd, r, U * depth * r, "rstd")
    assert torch.equal(bits(layers.layer_norm(x, w, b, eps)), bits(y))
    return mean, rstd


def check_norm_grad(layers, x, w, g, mean, rstd):
    (dx, dw, db), (ex, ew, eb) = norm_grad_ref(g, x, mean, rstd, w)
    got = layers.layer_norm_grad(g, x, mean, rstd, w)
    close(got[0], dx, ex, ("dx", tuple(x.shape), x.dtype))
    close(got[1], dw, ew, "dweight")
    close(got[2], db, eb, "dbias")
    again = layers.layer_norm_grad(g, x, mean, rstd, w)
    assert all(torch.equal(bits(p), bits(q)) for p, q in zip(got, again))


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("d", [1, 2, 3, 8, 16, 31, 64, 65, 100, 128, 256, 257, 500, 512, 768, 1000, 1001, 1024, 2047,
                               2048, 4096, 5000, 8191, 8192, 16384, 16385, 32768, 40000, 40001])
def test_norm_widths(layers, pair, d):
    for n in (1, 5, 67):
        x, w, b = norm_inputs(n, d, pair, seed=n)
        if d == 1:
            w, b = w.contiguous(), b.contiguous()
        mean, rstd = check_norm(layers, x, w, b)
        check_norm_grad(layers, x, w, randn(n, d, seed=9, dtype=pair[0]), mean, rstd)


@pytest.mark.parametrize("n,d", [(1, 64), (2, 768), (129, 96), (1000, 1024), (20000, 33), (70000, 128), (300001, 8),
                                 (5000, 4096), (300, 20000)])
@pytest.mark.parametrize("pair", [("f32", "f32"), ("bf16", "f32")], ids="-".join)
def test_norm_lengths(layers, n, d, pair):
    x, w, b = norm_inputs(n, d, pair)
    mean, rstd = check_norm(layers, x, w, b)
    check_norm_grad(layers, x, w, randn(n, d, seed=5, dtype=pair[0]), mean, rstd)


def test_norm_without_parameters_and_in_parts(layers):
    for pair in (("f32", "f32"), ("f16", "f16")):
        for n, d in ((50, 384), (9, 77), (4, 40000)):
            x, w, b = norm_inputs(n, d, pair)
            g = randn(n, d, seed=4, dtype=pair[0])
            for ww, bb in ((None, None), (w, None), (None, b)):
                mean, rstd = check_norm(layers, x, ww, bb)
            check_norm_grad(layers, x, None, g, mean, rstd)
            full = layers.layer_norm_grad(g, x, mean, rstd, w)
            for mask in range(8):
                need = tuple(bool(mask >> i & 1) for i in range(3))
                part = layers.layer_norm_grad(g, x, mean, rstd, w, need)
                for have, p, f in zip(need, part, full):
                    assert (p is not None) == have and (p is None or torch.equal(bits(p), bits(f)))


def test_norm_large_means_and_constant_rows(layers):
    # a mean of thousands of spreads: the differences are small beside the mean's half step
    for d in (96, 1000, 1001, 4096, 40000):
        x = (randn(20, d) + 5000.0)
        check_norm(layers, x, None, None)
        x[3] = 7.25
        x[4] = 0.0
        y = layers.layer_norm(x)
        assert not y[4].any() and float(y[3].abs().max()) < 1e-3
        b = randn(d, seed=3)
        assert torch.equal(layers.layer_norm(x, None, b)[4], b)
    one = randn(5, 1)
    assert not layers.layer_norm(one).any()
    assert bool(torch.isnan(layers.layer_norm(one, eps=0.0)).all())  # 0 / 0, as the formula says


def test_norm_extreme_rows_stay_alone(layers):
    for d in (64, 1000, 1001, 40000):
        x, w, b = norm_inputs(9, d, ("f32", "f32"))
        clean = layers.layer_norm(x, w, b)
        x[2, 0], x[5, d - 1] = float("nan"), float("inf")
        y = layers.layer_norm(x, w, b)
        rest = [0, 1, 3, 4, 6, 7, 8]
        assert torch.equal(bits(y[rest]), bits(clean[rest]))
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[5]).any())


def test_norm_strides_and_shapes(layers):
    base = randn(90, 200)
    w, b = randn(64, seed=1), randn(64, seed=2)
    for view in (base[:, :64], base[:, 8:72], base[:, 3:67], base[::3, 100:164], base[:, ::2][:, :64],
                 base[:1, :64].expand(90, 64)):
        mean, rstd = check_norm(layers, view, w, b)
        check_norm_grad(layers, view, w, base[: len(view), 70:134], mean, rstd)
    check_norm(layers, randn(3, 4, 5, 64), w, b)
    check_norm(layers, randn(64), w, b)
    check_norm(layers, randn(10, 64), randn(65)[1:], randn(67)[3:])  # parameters off 16-byte lines
    empty = torch.zeros((0, 64), device=DEV)
    assert layers.layer_norm(empty, w, b).shape == (0, 64)
    z = torch.zeros(0, device=DEV)
    dx, dw, db = layers.layer_norm_grad(empty, empty, z, z, w)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_norm_abi_in_place_and_gaps(layers):
    L = abi()
    for d in (64, 63, 2048, 40000):
        x, w, b = norm_inputs(37, d, ("f32", "f32"))
        y, mean, rstd = layers.layer_norm_stats(x, w, b)
        wide = torch.full((37, d + 9), 7.0, device=DEV)
        wide[:, 4:4 + d] = x
        p = wide[:, 4:].data_ptr()
        check(L.gids_layer_norm(0, p, d + 9, None, None, p, 0, d + 9, w.data_ptr(), b.data_ptr(), 0, 37, d, 1e-5,
                                None))
        torch.cuda.synchronize()
        # a narrower vector may be used: the sums then run in another order
        ref, _, _, err = norm_ref(x, w, b, 1e-5)
        close(wide[:, 4:4 + d], ref, err)
        wide[:, 4:4 + d] = 7.0
        assert bool((wide == 7.0).all())
        g = randn(37, d, seed=8)
        want = layers.layer_norm_grad(g, x, mean, rstd, w)
        u = ctypes.c_uint64()
        check(L.gids_layer_norm_grad_workspace(37, d, ctypes.byref(u)))
        ws = torch.empty(u.value, dtype=torch.uint8, device=DEV)
        for over in (0, 1):  # dx over grad, then over x
            t = [g.clone(), x.clone()]
            dw, db = torch.empty_like(w), torch.empty_like(b)
            check(L.gids_layer_norm_grad(0, t[over].data_ptr(), d, dw.data_ptr(), db.data_ptr(), t[0].data_ptr(), d,
                                         t[1].data_ptr(), 0, d, w.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), 37, d,
                                         ws.data_ptr(), u.value, None))
            torch.cuda.synchronize()
            for a, e in zip((t[over], dw, db), want):
                assert torch.equal(bits(a), bits(e))


# ------------------------------------------------------------- as they are used
def step_ref(ids, table, w, b, scale, pad, up):
    """The input side of a training step in 64 bits by torch autograd."""
    t, w, b = (v.detach().double().requires_grad_() for v in (table, w, b))
    x = t[ids] * scale
    y = torch.nn.functional.layer_norm(x, (t.shape[1],), w, b, 1e-5)
    y.backward(up.double())
    dt = t.grad.clone()
    dt[pad] = t.grad[pad] if pad is None else 0
    return y.detach(), dt, w.grad, b.grad


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("n,dim", [(1, 8), (40, 96), (3000, 256)])
def test_training_step_end_to_end(layers, sparse, n, dim):
    emb = layers.NodeEmbedding(70, dim, scale=dim ** 0.5, padding_idx=3, sparse=sparse, device=DEV)
    norm = layers.LayerNorm(dim, device=DEV)
    with torch.no_grad():
        emb.weight.copy_(randn(70, dim) / dim ** 0.5)
        norm.weight.add_(0.1 * randn(dim, seed=1))
        norm.bias.add_(0.1 * randn(dim, seed=2))
    ids = randint(70, (n,))
    if n > 4:
        ids[::5] = 3
    up = randn(n, dim, seed=3)
    scale = float(torch.tensor(dim ** 0.5, dtype=torch.float32))
    y = norm(emb(ids))
    y.backward(up)
    ry, dt, dw, db = step_ref(ids, emb.weight, norm.weight, norm.bias, scale, 3, up)
    assert emb.weight.grad.is_sparse == sparse
    got = emb.weight.grad
    if sparse:
        got = got.coalesce()  # accumulating into .grad drops torch's flag
        assert 3 not in got.indices()[0].tolist()
        (raw,) = torch.autograd.grad(norm(emb(ids)), emb.weight, up)
        assert raw.is_coalesced() and torch.equal(raw.indices(), got.indices())
        got = got.to_dense()
    # every operator is held to its own bound above; through the chain the
    # relative errors add: 2^-24 x a few hundred of the largest term
    for a, e in ((y.detach(), ry), (got, dt), (norm.weight.grad, dw), (norm.bias.grad, db)):
        assert float((a.double() - e).abs().max()) <= 400 * U * n ** 0.5 * max(1.0, float(e.abs().max()))
    opt = torch.optim.SparseAdam([emb.weight]) if sparse else torch.optim.Adam([emb.weight])
    before = emb.weight.detach().clone()
    opt.step()
    assert torch.equal(emb.weight[3], before[3]) and not torch.equal(emb.weight, before)


def test_gradients_against_differences(layers):
    """Central differences of the 64-bit forward along random directions."""
    n, d = 20, 48
    x, w, b = norm_inputs(n, d, ("f32", "f32"))
    up = randn(n, d, seed=4)
    for t in (x, w, b):
        t.requires_grad_()
    layers.layer_norm(x, w, b).backward(up)

    def f(xx, ww, bb):
        return (norm_ref(xx, ww, bb, 1e-5)[0] * up.double()).sum()

    h = 1e-5
    for i, t in enumerate((x, w, b)):
        v = randn(*t.shape, seed=10 + i).double()
        args = [p.detach().double() for p in (x, w, b)]
        lo, hi = list(args), list(args)
        hi[i], lo[i] = args[i] + h * v, args[i] - h * v
        want = float((f(*hi) - f(*lo)) / (2 * h))
        mag = float((t.grad.double() * v).abs().sum())
        # truncation h^2 x third derivative (|v|^3 over the row's spread, below 1e3) and the
        # gradient's own error, 150 u of its terms
        assert abs(float((t.grad.double() * v).sum()) - want) <= (150 * U + 1e3 * h * h) * mag + 1e-8


def test_autograd_rules(layers):
    w = randn(30, 16).requires_grad_()
    ids = randint(30, (12,))
    out = layers.embedding(ids, w, dtype=torch.bfloat16)
    assert out.dtype == torch.bfloat16
    out.sum().backward()  # an expanded gradient (strides 0)
    c = torch.bincount(ids, minlength=30).float()
    assert w.grad.dtype == torch.float32 and torch.equal(w.grad, c[:, None].expand(30, 16))
    with torch.no_grad():
        assert not layers.embedding(ids, w).requires_grad
    x = randn(6, 24).half().requires_grad_()
    b = torch.zeros(24, device=DEV, requires_grad=True)  # a float32 bias without a weight
    layers.layer_norm(x, None, b).sum().backward()
    assert b.grad.dtype == torch.float32 and bool((b.grad == 6).all()) and x.grad.dtype == torch.float16
    x2 = randn(6, 24)  # gathered features need no gradient, their norm's weight does
    g = torch.ones(24, device=DEV, requires_grad=True)
    y = layers.layer_norm(x2, g)
    y.backward(torch.ones_like(y))
    assert x2.grad is None and g.grad is not None
    with pytest.raises(RuntimeError):  # saved rows that changed
        z = randn(4, 8).requires_grad_()
        t = z * 1
        y = layers.layer_norm(t)
        t.add_(1)
        y.sum().backward()
    with pytest.raises(RuntimeError):  # no second derivative
        z = randn(4, 8).requires_grad_()
        (gz,) = torch.autograd.grad(layers.layer_norm(z).square().sum(), z, create_graph=True)
        gz.sum().backward()


def test_other_streams(layers):
    w, x = randn(5000, 256), randn(4000, 256)
    ids = randint(5000, (4000,))
    want = (layers.embedding(ids, w, scale=2.0), layers.embedding_grad(ids, x, 5000), layers.layer_norm(x))
    rows = layers.embedding_grad_rows(ids, x, 5000)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams * 3:  # in flight together: each call has a workspace of its own
        with torch.cuda.stream(s):
            got.append((layers.embedding(ids, w, scale=2.0), layers.embedding_grad(ids, x, 5000),
                        layers.layer_norm(x), layers.embedding_grad_rows(ids, x, 5000)))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(g[:3], want))
        assert torch.equal(g[3][0], rows[0]) and torch.equal(bits(g[3][1]), bits(rows[1]))


def test_captured_graphs(layers):
    """A step captured twice, replayed in turn and at once, on new inputs."""
    w = randn(400, 96)
    nw, nb = 1 + 0.1 * randn(96, seed=1), 0.1 * randn(96, seed=2)

    def step(ids, g):
        e = layers.embedding(ids, w, scale=3.0)
        y, mean, rstd = layers.layer_norm_stats(e, nw, nb)
        dx, dw, db = layers.layer_norm_grad(g, e, mean, rstd, nw)
        return y, dw, db, layers.embedding_grad(ids, dx, 400, 3.0, 0)

    graphs = []
    for n in (50, 3000):
        ids, g = randint(400, (n,)), randn(n, 96)
        step(ids, g)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(ids, g)
        graphs.append((gr, ids, g, out))
    s = [torch.cuda.Stream() for _ in graphs]
    for rep in range(4):
        for gr, ids, g, out in graphs:
            ids.copy_(randint(400, ids.shape, seed=rep + 20))
            g.copy_(randn(*g.shape, seed=rep + 30))
        torch.cuda.synchronize()
        for st, (gr, *_) in zip(s, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for gr, ids, g, out in graphs:
            for a, e in zip(out, step(ids, g)):
                assert torch.equal(bits(a), bits(e))


def test_captured_backward(layers):
    emb = layers.NodeEmbedding(200, 64, device=DEV)
    norm = layers.LayerNorm(64, device=DEV)
    ids, up = randint(200, (500,)), randn(500, 64)

    def step():
        emb.zero_grad(set_to_none=True)
        norm.zero_grad(set_to_none=True)
        norm(emb(ids)).backward(up)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    want = [p.grad.clone() for p in (emb.weight, norm.weight, norm.bias)]
    gr = torch.cuda.CUDAGraph()
    emb.zero_grad(set_to_none=True)
    norm.zero_grad(set_to_none=True)
    with torch.cuda.graph(gr):
        norm(emb(ids)).backward(up)
    gr.replay()
    torch.cuda.synchronize()
    for p, e in zip((emb.weight, norm.weight, norm.bias), want):
        assert torch.equal(bits(p.grad), bits(e))


def test_counting_rows_is_refused_in_a_capture(layers):
    L = abi()
    ids = randint(50, (30,))
    b = ctypes.c_uint64()
    check(L.gids_embedding_grad_workspace(30, 50, 8, ctypes.byref(b)))
    ws = torch.empty(b.value, dtype=torch.uint8, device=DEV)
    cd = torch.zeros(1, dtype=torch.int64, device=DEV)
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        st = torch.cuda.current_stream().cuda_stream
        args = (0, ids.data_ptr(), 8, 30, 50, -1, 8, ws.data_ptr(), b.value)
        rc = L.gids_embedding_group(*args, None, ctypes.byref(ctypes.c_uint64()), st)
        check(L.gids_embedding_group(*args, cd.data_ptr(), None, st))  # the count stays on the device
    assert rc == GIDS_E_STATE
    gr.replay()
    torch.cuda.synchronize()
    assert int(cd) == len(torch.unique(ids))


def test_abi_reports_bad_ids(layers):
    L = abi()
    w, out = randn(10, 8), torch.empty((4, 8), device=DEV)
    ids = torch.tensor([1, 10, 2, 3], device=DEV)
    args = (0, out.data_ptr(), 0, 8, w.data_ptr(), 0, 8, 10, 8, ids.data_ptr(), 8, 4, 1.0, None)
    check(L.gids_embedding(*args))
    assert L.gids_embedding_check(0, None) == GIDS_E_RANGE
    assert L.gids_embedding_check(0, None) == gids_abi.GIDS_OK
    assert torch.equal(out[[0, 2, 3]], w[[1, 2, 3]]) and not out[1].any()


@pytest.mark.parametrize("pair", [p for p in PAIRS], ids="-".join)
def test_rows_behind_the_batch_are_left(layers, pair):
    L = abi()
    x, w, b = norm_inputs(5, 200, pair)
    y = torch.full((8, 200), 3.0, device=DEV, dtype=x.dtype)
    mean = torch.full((8,), 3.0, device=DEV)
    rstd = torch.full((8,), 3.0, device=DEV)
    check(L.gids_layer_norm(0, y.data_ptr(), 200, mean.data_ptr(), rstd.data_ptr(), x.data_ptr(), CODES[x.dtype], 200,
                            w.data_ptr(), b.data_ptr(), CODES[w.dtype], 5, 200, 1e-5, None))
    torch.cuda.synchronize()
    assert torch.equal(bits(y[:5]), bits(layers.layer_norm(x, w, b)))
    assert bool((y[5:] == 3).all()) and bool((mean[5:] == 3).all()) and bool((rstd[5:] == 3).all())


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current_one(layers):
    w = randn(50, 16).to("cuda:1")
    ids = randint(50, (20,)).to("cuda:1")
    with torch.cuda.device(0):
        assert torch.equal(layers.embedding(ids, w), w[ids])
        layers.layer_norm(w)
        layers.embedding_grad_rows(ids, w[ids], 50)
    assert torch.cuda.current_device() == 0


def test_fetch_feature_trains_its_input_layers(layers):
    """Gathered and embedded types through fetch_feature, a norm behind each, and
    the gradients of a step, on the GPU."""
    import numpy as np

    import GIDS
    from oracle import oracle

    dim, rows = 96, 1000
    t = oracle.synth_table(oracle.KIND_F32_UNIFORM, 3, rows, dim)
    emb = layers.NodeEmbedding(500, dim, scale=2.0, sparse=True, device=DEV)
    norms = {k: layers.LayerNorm(dim, device=DEV) for k in ("paper", "author")}
    g = GIDS.GIDS(page_size=4096, cache_dim=dim, num_ele=t.size, num_ssd=2, cache_size=1, ctrl_idx=0, heterograph=True,
                  heterograph_map={"paper": 0, "fos": 600}, node_embeddings={"author": emb}, feature_norm=norms,
                  accumulator_flag=True)
    g.required_accesses = 300
    g.BAM_FS.write_range(t.ctypes.data, t.nbytes, 0)
    rng = np.random.default_rng(0)
    bs = [[{"paper": torch.as_tensor(rng.integers(0, 600, 150)), "author": torch.as_tensor(rng.integers(0, 500, 90)),
            "fos": torch.as_tensor(rng.integers(0, 400, 60))}, f"s{i}"] for i in range(6)]
    it = iter([list(b) for b in bs])
    opt = torch.optim.SparseAdam([emb.weight], lr=0.1)
    for b in bs[:3]:
        table = emb.weight.detach().clone()
        f = g.fetch_feature(dim, it, DEV)[-1]
        paper = torch.as_tensor(oracle.gather(t, b[0]["paper"].numpy())).to(DEV)
        fos = torch.as_tensor(oracle.gather(t, b[0]["fos"].numpy(), key_off=600)).to(DEV)
        assert torch.equal(f["fos"], fos)
        ref, _, _, err = norm_ref(paper, None, None, 1e-5)
        close(f["paper"].detach(), ref, err)
        ref, _, _, err = norm_ref(2.0 * table[b[0]["author"].to(DEV)], None, None, 1e-5)
        close(f["author"].detach(), ref, err)
        up = {k: randn(*f[k].shape, seed=5) for k in norms}
        for k in norms:
            norms[k].zero_grad(set_to_none=True)
        opt.zero_grad(set_to_none=True)
        torch.autograd.backward([f[k] for k in norms], [up[k] for k in norms])
        for k in norms:
            n = f[k].shape[0]
            close(norms[k].bias.grad, up[k].double().sum(0), U * n * up[k].double().abs().sum(0))
        grad = emb.weight.grad.coalesce()
        assert torch.equal(grad.indices()[0], torch.unique(b[0]["author"]).to(DEV))
        opt.step()
        assert not torch.equal(emb.weight.detach(), table)  # the next batch sees the new rows
    g.close()


@pytest.mark.parametrize("n", [126, 127, 128, 129, 1024, 1025, 8191, 8192, 8193, 16384, 16385, 32767, 32768, 32769,
                               303104, 303105])
def test_grad_lengths_where_the_sort_changes(layers, n):
    for seed, rows in enumerate((5, 3000, 1 << 18)):
        check_grad(layers, randint(rows, (n,), seed=seed), randn(n, 8, seed=n, dtype="bf16"), rows, 1.0, 0,
                   torch.float32)


@pytest.mark.parametrize("dim", [1, 9, 129, 1024])
def test_grad_few_hot_ids(layers, dim):
    for n in (2, 33, 100, 128, 200):
        for kind in range(3):
            ids = torch.full((n,), 7, device=DEV)
            if kind == 1:
                ids[::3] = 2
            if kind == 2:
                ids[n // 2:] = torch.arange(n - n // 2, device=DEV) % 11
            check_grad(layers, ids, randn(n, dim, seed=n, dtype="f16"), 11, 0.5, None)


def test_odd_rows_and_bad_ids(layers):
    for table, out in (("f32", "bf16"), ("f16", "f16")):
        w = randn(300, 1030, dtype=table)[:, 1:1002]
        for dt in (torch.int64, torch.int32):
            ids = randint(300, (700,), dtype=dt)
            check_embedding(layers, ids, w, 1.5, TYPES[out])
            ids[5], ids[699] = 300, -1
            got = layers.embedding(ids, w, scale=1.5, dtype=TYPES[out])
            with pytest.raises(RuntimeError, match="outside its table"):
                layers.check_ids(DEV)
            assert not got[5].any() and not got[699].any()
            close(got[6:699], w[ids[6:699].long()].double() * 1.5, U * w[ids[6:699].long()].double().abs() * 1.5)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_norm_rows_that_meet_vectors_differently(layers, pair):
    """Views whose rows start anywhere, alike or not in the matrices of a call."""
    for n, d, off, pitch in ((3000, 257, 1, 260), (1500, 1001, 3, 1010), (700, 768, 5, 775), (40, 5003, 7, 5013)):
        wide, _, _ = norm_inputs(n, pitch, pair)
        x = wide[:, off:off + d]
        w, b = norm_inputs(1, d, pair)[1:]
        mean, rstd = check_norm(layers, x, w, b)
        g = randn(n, pitch, seed=3, dtype=pair[0])
        check_norm_grad(layers, x, w, g[:, off:off + d], mean, rstd)  # dx contiguous, x and grad alike
        check_norm_grad(layers, x, w, g[:, :d], mean, rstd)
        c = x.contiguous()
        check_norm_grad(layers, c, w, g[:, :d].contiguous(), mean, rstd)  # all alike


def test_captured_long_lists(layers):
    L = abi()
    for n, rows in ((5000, 3000), (40000, 70000), (350000, 1 << 20)):
        ids, g = randint(rows, (n,)), randn(n, 16)
        b = ctypes.c_uint64()
        check(L.gids_embedding_grad_workspace(n, rows, 16, ctypes.byref(b)))
        ws = torch.empty(b.value, dtype=torch.uint8, device=DEV)
        count = torch.zeros(1, dtype=torch.int64, device=DEV)
        r = torch.full((n,), -9, dtype=torch.int64, device=DEV)
        v = torch.zeros((n, 16), device=DEV)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            st = torch.cuda.current_stream().cuda_stream
            dw = layers.embedding_grad(ids, g, rows)
            check(L.gids_embedding_group(0, ids.data_ptr(), 8, n, rows, -1, 16, ws.data_ptr(), b.value,
                                         count.data_ptr(), None, st))
            check(L.gids_embedding_grad_rows(0, r.data_ptr(), v.data_ptr(), 0, 16, n, rows, 16, g.data_ptr(), 0, 16,
                                             n, 1.0, ws.data_ptr(), b.value, st))
        for rep in range(3):
            ids.copy_(randint(rows // (rep + 1), (n,), seed=rep + 1))
            g.copy_(randn(n, 16, seed=rep + 1))
            r.fill_(-9)
            gr.replay()
            torch.cuda.synchronize()
            want_r, want_v = layers.embedding_grad_rows(ids, g, rows)
            k = int(count)
            assert k == len(want_r) and torch.equal(r[:k], want_r) and bool((r[k:] == -9).all())
            assert torch.equal(bits(v[:k]), bits(want_v))
            assert torch.equal(bits(dw), bits(layers.embedding_grad(ids, g, rows)))


def test_calls_from_several_threads(layers):
    import threading

    jobs = []
    for t in range(4):
        n = (100, 3000, 40000, 9000)[t]
        ids, w, g = randint(700, (n,), seed=t), randn(700, 72, seed=t), randn(n, 72, seed=t + 9)
        want = (layers.embedding(ids, w, scale=0.5), layers.embedding_grad(ids, g, 700), layers.layer_norm(g),
                *layers.embedding_grad_rows(ids, g, 700))
        jobs.append((ids, w, g, want))
    torch.cuda.synchronize()
    bad = []

    def run(ids, w, g, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = (layers.embedding(ids, w, scale=0.5), layers.embedding_grad(ids, g, 700),
                           layers.layer_norm(g), *layers.embedding_grad_rows(ids, g, 700))
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want)):
                        bad.append("differs")
        except Exception as e:  # reported by the main thread
            bad.append(repr(e))

    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad, bad[:3]


def test_counting_rows_in_a_capture_leaves_python_usable(layers):
    ids, g = randint(50, (300,)), randn(300, 8)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = layers.layer_norm(g)
        with pytest.raises(RuntimeError, match="captured"):
            layers.embedding_grad_rows(ids, g, 50)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(bits(y), bits(layers.layer_norm(g)))
    layers.embedding_grad_rows(ids, g, 50)


def test_rows_of_another_list_stay_inside_the_gradient(layers):
    """gids_embedding_grad_rows after gids_embedding_group of fewer ids, on the same
    workspace: the call's own bounds hold, whatever the words say."""
    L = abi()
    g = randn(3000, 8)
    b = ctypes.c_uint64()
    check(L.gids_embedding_grad_workspace(3000, 50, 8, ctypes.byref(b)))
    ws = torch.full((b.value,), 0x11, dtype=torch.uint8, device=DEV)
    ids = randint(50, (100,))
    count = torch.zeros(1, dtype=torch.int64, device=DEV)
    check(L.gids_embedding_group(0, ids.data_ptr(), 8, 100, 50, -1, 8, ws.data_ptr(), b.value, count.data_ptr(), None,
                                 None))
    r = torch.full((60,), -9, dtype=torch.int64, device=DEV)
    v = torch.full((60, 8), 7.0, device=DEV)
    check(L.gids_embedding_grad_rows(0, r.data_ptr(), v.data_ptr(), 0, 8, 40, 50, 8, g.data_ptr(), 0, 8, 3000, 1.0,
                                     ws.data_ptr(), b.value, None))
    torch.cuda.synchronize()
    assert bool((r[40:] == -9).all()) and bool((v[40:] == 7).all())


@pytest.mark.parametrize("rows,dim", [(33, 7), (1, 3), (5, 1), (1001, 129)])
def test_grad_tables_of_odd_size(layers, rows, dim):
    for n in (5, 300, 40000):
        for t in ("f32", "f16"):
            ids, g = randint(max(1, rows // 2), (n,)), randn(n, dim, dtype=t)
            big = torch.full((rows * dim + 8,), 5.0, device=DEV, dtype=TYPES[t])
            dw = layers.embedding_grad(ids, g, rows)
            L = abi()
            b = ctypes.c_uint64()
            check(L.gids_embedding_grad_workspace(n, rows, dim, ctypes.byref(b)))
            ws = torch.empty(b.value, dtype=torch.uint8, device=DEV)
            check(L.gids_embedding_grad(0, big.data_ptr(), CODES[big.dtype], dim, rows, dim, g.data_ptr(),
                                        CODES[g.dtype], dim, ids.data_ptr(), 8, n, -1, 1.0, ws.data_ptr(), b.value,
                                        None))
            torch.cuda.synchronize()
            assert torch.equal(bits(big[:rows * dim].view(rows, dim)), bits(dw))
            assert bool((big[rows * dim:] == 5).all())
            check_grad(layers, ids, g, rows)


def test_checking_ids_in_a_capture_is_refused(layers):
    g = randn(30, 8)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = layers.layer_norm(g)
        assert abi().gids_embedding_check(0, torch.cuda.current_stream().cuda_stream) == GIDS_E_STATE
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(bits(y), bits(layers.layer_norm(g)))


def test_distinct_rows_in_one_call_and_in_two(layers, monkeypatch):
    for n, rows in ((1, 1), (90, 40), (4000, 700), (60000, 3000)):
        ids, g = randint(rows, (n,), seed=n), randn(n, 40, seed=n, dtype="bf16")
        got = []
        for limit in (0, 1 << 40):
            monkeypatch.setattr(layers, "_ONE_CALL_BYTES", limit)
            got.append(layers.embedding_grad_rows(ids, g, rows, 0.5, 0, torch.float32))
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(*got))
        assert got[1][0].is_contiguous() and got[1][1].is_contiguous()


@pytest.mark.parametrize("n", [1, 2, 31, 33, 64, 100, 127, 128])
def test_distinct_rows_of_few_ids(layers, n):
    for rows, dim, t in ((5, 16, "f32"), (1 << 31, 8, "bf16"), (300, 1024, "f16")):
        ids = (randint(1 << 40, (n,), seed=n) * 7919) % rows
        ids[n // 2:] = ids[: n - n // 2].clone()
        g = randn(n, dim, seed=n, dtype=t)
        r, v = layers.embedding_grad_rows(ids, g, rows, 2.0)
        want, inv = torch.unique(ids, return_inverse=True)
        s, a, c = group_sums(inv, g, len(want))
        assert torch.equal(r, want)
        close(v, 2.0 * s, grad_error(a, c, 2.0, 2.0 * s))
        # padding and bad ids are left out
        bad = ids.clone()
        bad[0] = rows if n > 1 else ids[0]
        pad = int(ids[-1])
        r, v = layers.embedding_grad_rows(bad, g, rows, 2.0, pad)
        if n > 1:
            with pytest.raises(RuntimeError, match="outside its table"):
                layers.check_ids(DEV)
        keep = (bad < rows) & (bad != pad)
        assert torch.equal(r, torch.unique(bad[keep]))


@pytest.mark.parametrize("d", [1, 5, 24, 96, 200, 257, 768, 1001, 1024, 4096, 4100, 8192, 9000, 16384])
def test_norm_gradient_of_few_rows(layers, d):
    """Around the row counts where one cluster stops doing all of it."""
    for n in (1, 3, 8, 9, 31, 33, 64, 100, 129, 160, 320, 512, 513, 641, 1300, 2050):
        if n * d > 3000000:
            continue
        for pair in (("bf16", "f32"), ("f32", "f32")):
            x, w, _ = norm_inputs(n, d, pair, seed=n)
            _, mean, rstd = layers.layer_norm_stats(x)
            check_norm_grad(layers, x, w, randn(n, d, seed=2, dtype=pair[0]), mean, rstd)


@pytest.mark.parametrize("n,rows,dim", [(128, 300, 24), (129, 300, 24), (4000, 700, 40), (40000, 3000, 72)])
def test_distinct_rows_through_the_abi(layers, n, rows, dim):
    """Rows of the result are strided here, with room for more of them; what lies between and behind stays."""
    ids, g = randint(rows, (n,), seed=n), randn(n, dim, seed=n, dtype="f16")
    want_rows, want = layers.embedding_grad_rows(ids, g, rows, 0.5, 7, torch.float32)
    most, stride = min(n, rows) + 5, dim + 8
    out_rows = torch.full((most,), -5, dtype=torch.int64, device=DEV)
    out = torch.full((most, stride), -5.0, device=DEV)
    ws = torch.empty(layers._store_module().embedding_grad_workspace(n, rows, dim), dtype=torch.uint8, device=DEV)
    L, count = abi(), ctypes.c_uint64()
    vp, i32, i64, u64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float
    L.gids_embedding_grad_distinct.argtypes = [i32, vp, vp, i32, i64, i64, i64, i64, vp, i32, i64, vp, i32, i64, i64,
                                               f32, vp, u64, ctypes.POINTER(u64), vp]
    assert L.gids_embedding_grad_distinct(
        0, out_rows.data_ptr(), out.data_ptr(), 0, stride, most, rows, dim, g.data_ptr(), 1, dim, ids.data_ptr(), 8, n,
        7, 0.5, ws.data_ptr(), ws.numel(), ctypes.byref(count), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    k = count.value
    assert k == len(want_rows) and torch.equal(out_rows[:k], want_rows)
    assert torch.equal(bits(out[:k, :dim]), bits(want))
    assert bool((out_rows[k:] == -5).all()) and bool((out[k:] == -5).all()) and bool((out[:, dim:] == -5).all())


@pytest.mark.parametrize("dim", [1, 3, 4, 7, 8, 33, 129, 1001])
def test_few_ids_and_rows_of_any_width(layers, dim):
    """Up to 128 ids, tables dense and as distinct rows: whole blocks of zero rows, blocks with
    some, rows on and off 16 bytes."""
    for n, rows in ((1, 1), (3, 31), (64, 33), (128, 1000), (128, 20000), (5, 70001)):
        for pair in (("f32", "f32"), ("bf16", "f32"), ("f16", "f16")):
            g = randn(n, dim, seed=n, dtype=pair[0])
            check_grad(layers, randint(rows, (n,), seed=rows), g, rows, 0.5, rows // 2, TYPES[pair[1]])
    # the same bits as the sums of a sorted list that ends in padding
    ids, g = randint(40, (128,), seed=3), randn(128, dim, seed=3)
    more = torch.cat([ids + 1, torch.zeros(72, dtype=ids.dtype, device=DEV)])
    dw = layers.embedding_grad(ids + 1, g, 41, 2.0, 0)
    assert not bool(dw[0].any())
    s, a, c = group_sums(more, torch.cat([g, randn(72, dim)]), 41, 0)
    close(layers.embedding_grad(more, torch.cat([g, randn(72, dim)]), 41, 2.0, 0), 2.0 * s, grad_error(a, c, 2.0, 2.0 * s))
    close(dw, 2.0 * s, grad_error(a, c, 2.0, 2.0 * s))


def test_few_ids_into_a_gapped_table(layers):
    L = abi()
    for dim, stride, t, code in ((8, 12, torch.float32, 0), (5, 7, torch.float16, 1), (8, 24, torch.bfloat16, 2)):
        ids, g = randint(500, (90,), seed=dim), randn(90, dim).to(t)
        dw = torch.full((502, stride), 7.0, device=DEV, dtype=t)
        check(L.gids_embedding_grad(0, dw[1:].data_ptr(), code, stride, 500, dim, g.data_ptr(), code, dim,
                                    ids.data_ptr(), 8, 90, 3, 1.0, None, 0, None))
        torch.cuda.synchronize()
        assert torch.equal(bits(dw[1:-1, :dim].contiguous()), bits(layers.embedding_grad(ids, g, 500, 1.0, 3)))
        assert bool((dw[0] == 7).all()) and bool((dw[-1] == 7).all()) and bool((dw[1:-1, dim:] == 7).all())


@pytest.mark.parametrize("n,d", [(2048, 1), (2048, 128), (1000, 8), (341, 768), (63, 4096), (64, 4096), (261, 1001),
                                 (2000, 130)])
def test_norm_gradient_without_a_workspace(layers, n, d):
    """As large as it may be, also where the matrices do not meet 16 bytes alike."""
    for pair in (("bf16", "f32"), ("f32", "f32"), ("f16", "f16")):
        x, w, _ = norm_inputs(n, d, pair, seed=n)
        g = randn(n, d, seed=2, dtype=pair[0])
        _, mean, rstd = layers.layer_norm_stats(x)
        check_norm_grad(layers, x, w, g, mean, rstd)
        wide = torch.zeros(n, d + 3, dtype=x.dtype, device=DEV)
        wide[:, 1:d + 1] = x
        check_norm_grad(layers, wide[:, 1:d + 1], w, g, mean, rstd)


@pytest.mark.parametrize("n", [32768, 32769, 33280, 75775, 75776, 75777, 303104, 303105])
def test_sort_shapes(layers, n):
    """Around the lengths where the sort changes its kernels and what a thread takes."""
    for rows in (7, 70000, 1 << 22):
        ids, g = randint(rows, (n,), seed=n), randn(n, 4, seed=3)
        r, v = layers.embedding_grad_rows(ids, g, rows, 1.0, 3)
        want, inv = torch.unique(ids, return_inverse=True)
        s, a, c = group_sums(inv, g, len(want))
        keep = want != 3
        assert torch.equal(r, want[keep])
        close(v, s[keep], grad_error(a, c, 1.0, s)[keep])


@pytest.mark.parametrize("dim,t", [(4096, "f16"), (4104, "bf16"), (2052, "f32"), (5120, "bf16")])
def test_sums_of_long_rows_over_many_ids(layers, dim, t):
    """Two vectors a thread: whole teams, and teams that end in the first or the second vector."""
    n = 40001
    for rows in (30, 30000):
        ids = randint(rows, (n,), seed=dim)
        ids[: n // 3] = rows // 2  # a run over many blocks
        check_grad(layers, ids, randn(n, dim, seed=1, dtype=t), rows, 0.5, 1)


def test_few_ids_next_to_one_another(layers):
    """Named rows at the ends of the stretches that are zeroed together, and side by side."""
    for dim, rows in ((1, 1000), (4, 640), (64, 40), (600, 9)):
        step = max(1, min(128, 2048 // (4 * dim)))
        at = [r for b in range(0, rows, step) for r in (b, b + 1, b + step - 1) if r < rows][:127] + [rows - 1]
        check_grad(layers, torch.tensor(at, device=DEV), randn(len(at), dim, seed=dim), rows, 1.0)
    ids = torch.arange(128, device=DEV)
    check_grad(layers, ids, randn(128, 2, seed=1), 128, 1.0)
    check_grad(layers, ids + 3, randn(128, 2, seed=1), 400, 1.0, 5)


CAPTURE_BESIDE = """
import threading
import torch
from GIDS import layers

DEV = "cuda:0"
s = torch.cuda.Stream()
ids = torch.arange(100, device=DEV) % 40
g = torch.randn(100, 16, device=DEV)
x = torch.randn(64, 32, device=DEV)
with torch.cuda.stream(s):  # kernels and the allocator's blocks, but no call that returns a count yet
    dense = layers.embedding_grad(ids, g, 50)
    room = [torch.empty(50, dtype=torch.int64, device=DEV), torch.empty(50, 16, device=DEV)]
    del room
y = layers.layer_norm(x)
torch.cuda.synchronize()
got, bad = [], []

def other():
    try:
        with torch.cuda.stream(s):
            got.append(layers.embedding_grad_rows(ids, g, 50))
            layers.check_ids(DEV)
    except Exception as e:
        bad.append(repr(e))

gr = torch.cuda.CUDAGraph()
with torch.cuda.graph(gr):
    z = layers.layer_norm(x)
    t = threading.Thread(target=other)
    t.start()
    t.join()
assert not bad, bad
gr.replay()
torch.cuda.synchronize()
assert torch.equal(z, y)
rows, values = got[0]
assert torch.equal(rows, torch.arange(40, device=DEV)) and torch.equal(values, dense[:40])
"""


def test_counting_rows_beside_another_threads_capture(layers):
    """The first call that returns a count, while another thread captures a graph in torch's default mode."""
    import os
    import subprocess
    import sys

    run = subprocess.run([sys.executable, "-c", CAPTURE_BESIDE], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": os.pathsep.join(p for p in sys.path if p)})
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [1, 8, 33, 768, 1001, 4096, 20000])
def test_norm_statistics_of_rows_that_are_not_finite(layers, d, t):
    """NaN or infinities anywhere in a row make its mean (or, for infinities, at least its variance) NaN: rstd
    is NaN with it, and the rows beside it keep their bits."""
    x = randn(9, d, seed=d, dtype=t)
    want = layers.layer_norm_stats(x)
    x[1, d // 2] = float("nan")
    x[4, 0] = float("inf")
    x[7, d - 1] = -float("inf")
    x[7, d // 3] = float("inf") if d > 1 else -float("inf")
    y, mean, rstd = layers.layer_norm_stats(x)
    ref = (x.double() - x.double().mean(1, keepdim=True)).square().mean(1)
    bad = torch.isnan(ref)
    assert bad.tolist() == [i in (1, 4, 7) for i in range(9)]
    assert torch.equal(torch.isnan(rstd), bad) and bool(torch.isnan(y[bad]).all())
    assert not bool(torch.isfinite(mean[bad]).any())
    for a, b in zip((y, mean, rstd), want):
        assert torch.equal(bits(a[~bad]), bits(b[~bad]))


@pytest.mark.parametrize("d", [8, 33, 1024, 20000])
def test_norm_of_rows_out_of_range(layers, d):
    """What float32 statistics cannot hold: a sum out of range gives NaN, squares alone out of range rstd = 0."""
    x, b = randn(4, d, seed=d), randn(d, seed=1)
    x[1] = 3e38
    x[2, ::2] = 1e25
    x[2, 1::2] = -1e25
    y, mean, rstd = layers.layer_norm_stats(x, None, b)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(rstd[1]))
    assert float(rstd[2]) == 0 and torch.equal(y[2], b) and bool(torch.isfinite(mean[2]))
    ref, _, _, err = norm_ref(x[[0, 3]], None, b, 1e-5)
    close(y[[0, 3]], ref, err)
