"""How GIDS.layers meets torch's transforms, on the CPU with a stand-in for the
kernels: a call either takes part in them or is refused."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd


def _array(ptr, *shape):
    count = 1
    for s in shape:
        count *= s
    return torch.frombuffer((ctypes.c_float * max(count, 1)).from_address(ptr), dtype=torch.float32)[:count].view(shape)


class Kernels:
    """The compiled module's calls on contiguous float32 host memory, in the formulas of their definitions."""

    def __init__(self):
        self.calls = 0

    def embedding_grad_workspace(self, n, num_rows, dim):
        return 256

    layer_norm_grad_workspace = embedding_grad_workspace

    def embedding(self, device, out, ot, os, weight, wt, ws, num_rows, dim, ids, ib, n, scale, stream):
        self.calls += 1
        i = torch.frombuffer((ctypes.c_int64 * n).from_address(ids), dtype=torch.int64)
        _array(out, n, dim).copy_(scale * _array(weight, num_rows, dim)[i])

    def embedding_grad(self, device, dw, wt, dws, num_rows, dim, grad, gt, gs, ids, ib, n, pad, scale, ws, wsb, stream):
        self.calls += 1
        i = torch.frombuffer((ctypes.c_int64 * n).from_address(ids), dtype=torch.int64)
        keep = i != pad
        _array(dw, num_rows, dim).zero_().index_add_(0, i[keep], scale * _array(grad, n, dim)[keep])

    def embedding_grad_distinct(self, device, rows, values, wt, vs, capacity, num_rows, dim, grad, gt, gs, ids, ib, n,
                                pad, scale, ws, wsb, stream):
        self.calls += 1
        i = torch.frombuffer((ctypes.c_int64 * n).from_address(ids), dtype=torch.int64)
        u, slot = torch.unique(i, return_inverse=True)
        torch.frombuffer((ctypes.c_int64 * capacity).from_address(rows), dtype=torch.int64)[:len(u)].copy_(u)
        _array(values, capacity, dim)[:len(u)].zero_().index_add_(0, slot, scale * _array(grad, n, dim))
        return len(u)

    def layer_norm(self, device, y, ys, mean, rstd, x, xt, xs, weight, bias, pt, n, dim, eps, stream):
        self.calls += 1
        v = _array(x, n, dim)
        m = v.mean(1, keepdim=True)
        r = ((v - m).square().mean(1, keepdim=True) + eps).rsqrt()
        out = (v - m) * r
        if weight:
            out = out * _array(weight, dim)
        if bias:
            out = out + _array(bias, dim)
        _array(y, n, dim).copy_(out)
        if mean:
            _array(mean, n).copy_(m[:, 0])
            _array(rstd, n).copy_(r[:, 0])

    def layer_norm_grad(self, device, dx, dxs, dw, db, grad, gs, x, xt, xs, weight, pt, mean, rstd, n, dim, ws, wsb,
                        stream):
        self.calls += 1
        g, v, r = _array(grad, n, dim), _array(x, n, dim), _array(rstd, n)[:, None]
        xh = (v - _array(mean, n)[:, None]) * r
        t = g * _array(weight, dim) if weight else g
        if dx:
            _array(dx, n, dim).copy_(r * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True)))
        if dw:
            _array(dw, dim).copy_((g * xh).sum(0))
        if db:
            _array(db, dim).copy_(g.sum(0))


@pytest.fixture
def layers(monkeypatch):
    from GIDS import layers

    k = Kernels()
    monkeypatch.setattr(layers, "_module", k)
    monkeypatch.setattr(layers, "_device_of", lambda *t: 0)
    monkeypatch.setattr(layers, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(layers, "kernels", k, raising=False)
    return layers


IDS = torch.tensor([2, 0, 2, 4])


def test_the_stand_in_agrees_with_torch(layers):
    w, x = torch.randn(5, 8).requires_grad_(), torch.randn(6, 8).requires_grad_()
    for sparse in (False, True):
        (gw,) = torch.autograd.grad(layers.embedding(IDS, w, 2.0, sparse=sparse).square().sum(), w)
        (want,) = torch.autograd.grad((2.0 * w[IDS]).square().sum(), w)
        torch.testing.assert_close(gw.to_dense(), want)
    p, b = torch.randn(8).requires_grad_(), torch.randn(8).requires_grad_()
    got = torch.autograd.grad(layers.layer_norm(x, p, b).square().sum(), (x, p, b))
    want = torch.autograd.grad(torch.nn.functional.layer_norm(x, (8,), p, b).square().sum(), (x, p, b))
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_tangents_are_refused(layers, requires_grad):
    w, x = torch.randn(5, 8).requires_grad_(requires_grad), torch.randn(6, 8).requires_grad_(requires_grad)
    p, st = torch.ones(8), torch.ones(6)
    with fwd.dual_level():
        dw, dx, dp, ds = (fwd.make_dual(t, torch.ones_like(t)) for t in (w, x, p, st))
        for call in (lambda: layers.embedding(IDS, dw), lambda: layers.layer_norm(dx),
                     lambda: layers.layer_norm(x, dp), lambda: layers.layer_norm(x, None, dp),
                     lambda: layers.layer_norm_stats(dx), lambda: layers.embedding_grad(IDS, dx[:4], 5),
                     lambda: layers.embedding_grad_rows(IDS, dx[:4], 5),
                     lambda: layers.layer_norm_grad(dx, x, st, st), lambda: layers.layer_norm_grad(x, dx, st, st),
                     lambda: layers.layer_norm_grad(x, x, ds, st), lambda: layers.layer_norm_grad(x, x, st, st, dp)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        # others' tangents are none of its business
        assert fwd.unpack_dual(layers.layer_norm(x, p)).tangent is None
        assert layers.embedding(IDS, w).shape == (4, 8)


def test_a_gradient_with_a_tangent_is_refused(layers):
    x = torch.randn(6, 8).requires_grad_()
    w = torch.randn(5, 8).requires_grad_()
    for out, leaf in ((layers.layer_norm(x), x), (layers.embedding(IDS, w), w),
                      (layers.embedding(IDS, w, sparse=True), w)):
        with fwd.dual_level():
            g = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, g)


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_traced_modules_run_their_kernels(layers, requires_grad, grad_mode):
    emb, norm = layers.NodeEmbedding(5, 8, scale=2.0), layers.LayerNorm(8)
    model = torch.nn.Sequential(emb, norm).requires_grad_(requires_grad)
    with torch.set_grad_enabled(grad_mode):
        traced = torch.jit.trace(model, (IDS,))
        before = layers.kernels.calls
        other = torch.tensor([4, 4, 1, 3])
        got = traced(other)
        assert layers.kernels.calls == before + 2
        want = torch.nn.functional.layer_norm(2.0 * emb.weight[other], (8,), norm.weight, norm.bias)
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-4)
        assert got.requires_grad == (requires_grad and grad_mode)


def test_what_a_recording_would_miss_is_refused(layers):
    from torch.fx.experimental.proxy_tensor import make_fx

    w, x, st = torch.randn(5, 8), torch.randn(4, 8), torch.ones(4)
    calls = (lambda t: layers.embedding_grad(IDS, t, 5), lambda t: layers.embedding_grad_rows(IDS, t, 5)[1],
             lambda t: layers.layer_norm_grad(t, x, st, st)[0], lambda t: layers.layer_norm_stats(t)[0])
    for call in calls:
        with pytest.raises(RuntimeError, match="jit.trace"):
            torch.jit.trace(call, (x,))
    for call in (*calls, lambda t: layers.layer_norm(t), lambda t: layers.embedding(IDS, t)):
        for requires_grad in (False, True):
            with pytest.raises(RuntimeError, match="make_fx"):
                make_fx(call)(x.clone().requires_grad_(requires_grad))
            for mode in ("fake", "symbolic"):
                with pytest.raises(RuntimeError):
                    make_fx(call, tracing_mode=mode)(x.clone().requires_grad_(requires_grad))
    # other modes see the operations and leave the call as it is
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    want = layers.layer_norm(x)
    with Watch():
        assert torch.equal(layers.layer_norm(x), want) and torch.equal(layers.embedding(IDS, w), w[IDS])


def test_transforms_of_functions_are_refused(layers):
    w, x = torch.randn(5, 8), torch.randn(4, 8)
    for call in (lambda: torch.vmap(lambda i: layers.embedding(i, w))(IDS),
                 lambda: torch.vmap(lambda t: layers.embedding(IDS, t))(torch.randn(2, 5, 8)),
                 lambda: torch.vmap(layers.layer_norm)(torch.randn(2, 4, 8)),
                 lambda: torch.func.jvp(layers.layer_norm, (x,), (x,)),
                 lambda: torch.func.jvp(lambda t: layers.embedding(IDS, t), (w,), (w,)),
                 lambda: torch.func.grad(lambda t: layers.layer_norm(t).sum())(x),
                 lambda: torch.func.grad(lambda t: layers.embedding(IDS, t).sum())(w),
                 lambda: torch.export.export(layers.LayerNorm(8), (x,))):
        with pytest.raises(Exception):
            call()


@pytest.mark.parametrize("sparse", [False, True])
def test_second_derivatives_are_refused(layers, sparse):
    x, w = torch.randn(4, 8), torch.randn(5, 8)
    p = torch.ones(8)
    losses = [(lambda t: layers.layer_norm(t).square().sum(), x), (lambda t: layers.layer_norm(x, t).square().sum(), p),
              (lambda t: layers.layer_norm(x, p, t).pow(3).sum(), torch.zeros(8)),
              (lambda t: layers.embedding(IDS, t, 2.0, sparse=sparse).pow(3).sum(), w)]
    for loss, at in losses:
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.functional.hvp(loss, at, torch.ones_like(at))
        if not sparse:
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.functional.hessian(loss, at)
        leaf = at.clone().requires_grad_()
        (g,) = torch.autograd.grad(loss(leaf), leaf, create_graph=True)
        (want,) = torch.autograd.grad(loss(leaf), leaf)
        assert torch.equal(g.detach().to_dense(), want.to_dense()) and g.is_sparse == want.is_sparse
        with pytest.raises(RuntimeError, match="second derivative"):
            (g.to_dense() if g.is_sparse else g).square().sum().backward()
        loss(leaf).backward(create_graph=True)  # a graph that nobody differentiates
        assert torch.equal(leaf.grad.detach().to_dense(), want.to_dense())
        leaf.grad = None
    # what does not depend on the gradient is no one's second derivative
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(layers.layer_norm(leaf).sum(), leaf)
    assert not g.requires_grad


@pytest.mark.parametrize("create_graph", [False, True])
def test_checkpointed_layers(layers, create_graph):
    """torch.utils.checkpoint recomputes what the backward pass reads, and lets it be read once."""
    from torch.utils.checkpoint import checkpoint

    emb, norm = layers.NodeEmbedding(5, 8), layers.LayerNorm(8)
    out = checkpoint(lambda i: norm(emb(i)), IDS, use_reentrant=False)
    params = (emb.weight, norm.weight, norm.bias)
    got = torch.autograd.grad(out.square().sum(), params, create_graph=create_graph)
    want = torch.autograd.grad(norm(emb(IDS)).square().sum(), params)
    assert all(torch.equal(a.detach(), b) for a, b in zip(got, want))


def test_compiled_callers_run_the_kernels(layers):
    """torch.compile breaks its graph at the kernels and calls them."""
    emb, norm = layers.NodeEmbedding(5, 8), layers.LayerNorm(8)
    step = torch.compile(lambda i: (norm(emb(i) * 2.0) + 1.0).square().sum(), backend="eager")
    for requires_grad in (True, False):
        for p in (*emb.parameters(), *norm.parameters()):
            p.requires_grad_(requires_grad)
            p.grad = None
        for _ in range(2):
            before = layers.kernels.calls
            loss = step(IDS)
            assert layers.kernels.calls >= before + 2
            torch.testing.assert_close(loss, (norm(emb(IDS) * 2.0) + 1.0).square().sum())
        if requires_grad:
            loss.backward()
            got = emb.weight.grad.clone()
            (want,) = torch.autograd.grad((norm(emb(IDS) * 2.0) + 1.0).square().sum(), emb.weight)
            torch.testing.assert_close(got, want)
