"""A model's input layers: what a trainer does with node ids and gathered rows
before its first layer (no reference counterpart; there it is torch code of the
training scripts).

* ``embedding`` / ``NodeEmbedding``: rows of a learnable table, times a scale,
  for node types without stored features (or tokens), with the gradient by
  sorted ids: dense, or as the distinct rows for tables too large for that.
* ``layer_norm`` / ``LayerNorm``: layer norm of gathered rows, forward and
  backward.

``GIDS.GIDS(node_embeddings=..., feature_norm=...)`` applies them to the batches
it hands out. All run as hand-written kernels in the library behind
``BAM_Feature_Store`` (imported on first use) on the current stream, take
float32, float16 and bfloat16 CUDA tensors, sum in float32 and repeat bit for
bit. Workspaces come from torch's allocator for each call, so calls on several
streams and in several captured graphs share nothing.

An id outside its table gives a zero row and no gradient, and raises at the next
embedding call on that device (of any thread and stream; that call did nothing and can
be repeated), or at ``check_ids``.

Derivatives are reverse-mode and first: inputs with a forward-mode tangent are
refused, and so are second derivatives. ``embedding`` and ``layer_norm`` can be
traced by torch.jit.trace (for a replay in Python); what else records torch
operations is refused. A backward pass that is captured into a CUDA graph must not
meet an eager graph of the same parameters that is still alive (torch's rule for
every op): drop eager losses and outputs first.
"""
from __future__ import annotations

import functools
import math

import torch
import torch.autograd.forward_ad as _forward_ad

from .sampler import _store_module as _import_module

try:  # the stream's handle without building a Stream object for every call
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:  # pragma: no cover - a build of torch without CUDA
    _raw_stream = None

_module = None


def _store_module():
    global _module
    if _module is None:
        _module = _import_module()
    return _module


_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _type(t: torch.dtype, what: str) -> int:
    if t not in _TYPES:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, not {t}")
    return _TYPES[t]


def _device_of(first: torch.Tensor, *others) -> int:
    """Index of the CUDA device that the tensors (or None) are all on."""
    device = first.get_device()
    if device < 0:
        raise ValueError(f"CUDA tensors expected, not {first.device}")
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError(f"a tensor is on {t.device}, the others on {first.device}")
    return device


_is_tracing = torch._C._is_tracing  # by torch.jit.trace
_dispatch_modes = torch._C._len_torch_dispatch_stack


def _check_transforms(*tensors):
    """What autograd would not see, or a recording would miss, is refused: for
    calls inside a forward_ad.dual_level or a dispatch mode (the callers look, as
    that is all that most calls pay for).

    The operators have no forward-mode derivative, so a tangent would be dropped without a
    word where no input requires grad. A recording of torch operations (make_fx) sees a
    kernel's empty result but not the kernel."""
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("GIDS.layers has no forward-mode derivatives (an input carries a tangent)")
    if _dispatch_modes():
        from torch.fx.experimental.proxy_tensor import get_proxy_mode

        if get_proxy_mode() is not None:
            raise RuntimeError("GIDS.layers cannot be recorded by make_fx")


def _check_transforms_and_trace(what, *tensors):
    """The same for the operators that torch.jit.trace cannot record as a function of their own."""
    if _is_tracing():
        raise RuntimeError(f"{what} cannot be traced by torch.jit.trace")
    _check_transforms(*tensors)


def _check_ids(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be int32 or int64, not {ids.dtype}")
    return ids.contiguous()


def _as_rows(t: torch.Tensor, dim: int):
    """t as a matrix of rows [*, dim] whose columns are consecutive (a view where there is one), and its row stride."""
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    if t.is_contiguous():  # (asking for this costs less than one stride)
        return t, dim
    if (dim > 1 and t.stride(1) != 1) or t.stride(0) < 0:
        return t.contiguous(), dim
    return t, t.stride(0)


def _new_like(t: torch.Tensor) -> torch.Tensor:
    """An empty contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _padding(padding_idx, num_rows: int) -> int:
    if padding_idx is None:
        return -1
    p = int(padding_idx)
    if not -num_rows <= p < num_rows:
        raise ValueError(f"padding_idx {p} is outside the table of {num_rows} rows")
    return p + num_rows if p < 0 else p


def check_ids(device=None):
    """Wait for the current stream of ``device`` and raise RuntimeError if an
    embedding call there met an id outside its table since the last check."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    _store_module().embedding_check(device.index, _raw_stream(device.index))


# ------------------------------------------------------------------ embedding
def _embedding_forward(ids, weight, scale, dtype):
    if weight.dim() != 2:
        raise ValueError(f"weight must be a matrix, not {tuple(weight.shape)}")
    num_rows, dim = weight.shape
    wt = ot = _type(weight.dtype, "weight")
    if dtype is not weight.dtype:
        ot = _type(dtype, "dtype")
    device = _device_of(weight, ids)
    stride = dim
    if not weight.is_contiguous():
        stride = weight.stride(0)
        if dim > 1 and weight.stride(1) != 1:
            raise ValueError("the columns of weight must be consecutive (stride 1)")
    ids = _check_ids(ids)
    shape = (*ids.shape, dim)
    out = weight.new_empty(shape) if ot == wt else weight.new_empty(shape, dtype=dtype)
    if dim:
        _store_module().embedding(device, out.data_ptr(), ot, dim, weight.data_ptr(), wt,
                                  stride, num_rows, dim, ids.data_ptr(), ids.element_size(), ids.numel(),
                                  scale, _raw_stream(device))
    return out


def _grad_args(ids, grad, num_rows, dtype):
    ids = _check_ids(ids)
    shape = grad.shape
    if len(shape) < 1 or shape[:-1] != ids.shape:
        raise ValueError(f"grad {tuple(shape)} does not hold one row for each of the ids {tuple(ids.shape)}")
    dim = shape[-1]
    if dim < 1:
        raise ValueError("grad has no columns")
    given = grad.dtype
    gt = wt = _type(given, "grad")
    if dtype is None:
        dtype = given
    elif dtype is not given:
        wt = _type(dtype, "dtype")
    return ids, *_as_rows(grad, dim), dim, dtype, gt, wt, _device_of(grad, ids)


def _grad_workspace(grad, n, num_rows, dim):
    return grad.new_empty(_store_module().embedding_grad_workspace(n, num_rows, dim), dtype=torch.uint8)


_FEW_IDS = 128  # GIDS_FEW_IDS: up to here one kernel, without a workspace
_FEW_NORM = 1 << 18  # GIDS_FEW_NORM


def embedding_grad(ids, grad, num_rows, scale=1.0, padding_idx=None, dtype=None):
    """The gradient of ``embedding`` as a dense table [num_rows, dim]: row v is
    ``scale`` times the sum of the rows of ``grad`` whose id is v (in position
    order, in float32), rounded to ``dtype`` (grad's by default, or float32).
    Ids equal to ``padding_idx`` are left out."""
    if _forward_ad._current_level >= 0 or _dispatch_modes() or _is_tracing():
        _check_transforms_and_trace("embedding_grad", grad)
    num_rows = int(num_rows)
    pad = _padding(padding_idx, num_rows)
    ids, g, stride, dim, dtype, gt, wt, device = _grad_args(ids, grad, num_rows, dtype)
    n = ids.numel()
    ws = None if n <= _FEW_IDS else _grad_workspace(grad, n, num_rows, dim)
    dw = grad.new_empty((num_rows, dim), dtype=dtype)
    _store_module().embedding_grad(device, dw.data_ptr(), wt, dim, num_rows, dim, g.data_ptr(), gt,
                                   stride, ids.data_ptr(), ids.element_size(), n, pad, scale,
                                   *_span(ws), _raw_stream(device))
    return dw


def embedding_grad_rows(ids, grad, num_rows, scale=1.0, padding_idx=None, dtype=None):
    """The gradient of ``embedding`` as its distinct rows: ``(rows, values)``,
    the ids that occur (ascending, int64; without ``padding_idx``) and for each
    the row ``embedding_grad`` would hold. Waits once, for the number of
    rows, so it cannot be captured into a graph."""
    if _forward_ad._current_level >= 0 or _dispatch_modes() or _is_tracing():
        _check_transforms_and_trace("embedding_grad_rows", grad)
    num_rows = int(num_rows)
    pad = _padding(padding_idx, num_rows)
    ids, g, stride, dim, dtype, gt, wt, device = _grad_args(ids, grad, num_rows, dtype)
    m, stream = _store_module(), _raw_stream(device)
    n = ids.numel()
    most = min(n, num_rows)
    ws = None if n <= _FEW_IDS else _grad_workspace(grad, n, num_rows, dim)
    if most * dim * dtype.itemsize <= _ONE_CALL_BYTES:
        rows = grad.new_empty(most, dtype=torch.int64)
        values = grad.new_empty((most, dim), dtype=dtype)
        count = m.embedding_grad_distinct(device, rows.data_ptr(), values.data_ptr(), wt, dim, most, num_rows, dim,
                                          g.data_ptr(), gt, stride, ids.data_ptr(), ids.element_size(), n, pad,
                                          scale, *_span(ws), stream)
        return rows.resize_(count), values.resize_(count, dim)
    if ws is None:
        ws = _grad_workspace(grad, n, num_rows, dim)
    count = m.embedding_group(device, ids.data_ptr(), ids.element_size(), n, num_rows, pad, dim, ws.data_ptr(),
                              ws.numel(), 0, stream)
    rows = grad.new_empty(count, dtype=torch.int64)
    values = grad.new_empty((count, dim), dtype=dtype)
    m.embedding_grad_rows(device, rows.data_ptr(), values.data_ptr(), wt, dim, count, num_rows, dim, g.data_ptr(),
                          gt, stride, n, scale, ws.data_ptr(), ws.numel(), stream)
    return rows, values


# Results up to this size get room for every row there can be, so that one call sorts and
# sums without a gap between (7,910 ids x 448 bf16: 32 us a pass instead of 37; 200,000 x 128
# fp32: 83 instead of 92); larger ones wait for the count and hold no more than the rows there are.
_ONE_CALL_BYTES = 1 << 28


class _Underivable(torch.autograd.Function):
    """Hands on gradients that depend on ``inputs`` and refuses to be differentiated."""

    @staticmethod
    def forward(ctx, grads, *inputs):
        return grads

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the gradients of GIDS.layers have no derivative (second derivatives are not supported)")


def _first_derivative(backward):
    """A backward pass of kernels that autograd does not see. Where a graph of it is
    asked for (create_graph), the gradients stay tied to what they depend on, so that
    a second derivative is an error: torch's once_differentiable leaves them
    untied, and torch.autograd.functional.hvp and hessian then take it as zero."""

    @functools.wraps(backward)
    def wrapper(ctx, grad):
        saved = ctx.saved_tensors  # once: torch.utils.checkpoint allows no second look
        with torch.no_grad():
            out = backward(ctx, saved, grad)
        if not torch.is_grad_enabled():
            return out
        at = [i for i, t in enumerate(out) if t is not None]
        tied = _Underivable.apply(tuple(out[i] for i in at), grad, *saved)
        out = list(out)
        for i, t in zip(at, tied):
            out[i] = t
        return tuple(out)

    return wrapper


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, sparse, dtype):
        ctx.save_for_backward(ids)
        ctx.conf = (weight.shape[0], scale, padding_idx, sparse, weight.dtype)
        return _embedding_forward(ids, weight, scale, dtype)

    @staticmethod
    @_first_derivative
    def backward(ctx, saved, grad):
        (ids,) = saved
        num_rows, scale, padding_idx, sparse, dtype = ctx.conf
        if not sparse:
            dw = embedding_grad(ids, grad, num_rows, scale, padding_idx, dtype)
        else:
            rows, values = embedding_grad_rows(ids, grad, num_rows, scale, padding_idx, dtype)
            dw = torch.sparse_coo_tensor(rows.unsqueeze(0), values, (num_rows, grad.shape[-1]), is_coalesced=True)
        return None, dw, None, None, None, None


def embedding(ids, weight, scale=1.0, padding_idx=None, sparse=False, dtype=None):
    """``scale * weight[ids]`` as a tensor [*ids.shape, dim] of ``dtype`` (the
    table's; any of the three types if the table is float32). Differentiable in
    ``weight``: rows of ``padding_idx`` get no gradient, and with ``sparse`` the
    gradient is a coalesced sparse tensor of the distinct rows (for
    torch.optim.SparseAdam and the like) instead of a dense table."""
    if _forward_ad._current_level >= 0 or _dispatch_modes():
        _check_transforms(weight)
    dtype = weight.dtype if dtype is None else dtype
    scale = float(scale)
    if padding_idx is not None:
        padding_idx = _padding(padding_idx, weight.shape[0])
    # a trace records the function, whose replay runs the kernel
    if (weight.requires_grad and torch.is_grad_enabled()) or _is_tracing():
        return _Embedding.apply(ids, weight, scale, padding_idx, bool(sparse), dtype)
    return _embedding_forward(ids, weight, scale, dtype)


class NodeEmbedding(torch.nn.Module):
    """A learnable table of ``num_rows`` rows, looked up by id (``embedding``).

    ``padding_idx`` starts as a zero row and gets no gradient; ``sparse`` gives
    the gradient as its distinct rows; ``out_dtype`` is the type of the looked
    up rows (a float32 table can feed a 16-bit model)."""

    def __init__(self, num_rows, dim, scale=1.0, padding_idx=None, sparse=False, dtype=torch.float32, out_dtype=None,
                 device=None):
        super().__init__()
        self.num_rows, self.dim = int(num_rows), int(dim)
        self.scale = float(scale)
        self.padding_idx = None if padding_idx is None else _padding(padding_idx, self.num_rows)
        self.sparse = bool(sparse)
        self.out_dtype = out_dtype
        self.weight = torch.nn.Parameter(torch.empty((self.num_rows, self.dim), dtype=dtype, device=device))
        self.reset_parameters()

    def reset_parameters(self):
        with torch.no_grad():
            self.weight.normal_(0.0, 1.0 / math.sqrt(self.dim))
            if self.padding_idx is not None:
                self.weight[self.padding_idx].zero_()

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx, self.sparse, self.out_dtype)

    def extra_repr(self):
        return f"{self.num_rows}, {self.dim}, scale={self.scale}, padding_idx={self.padding_idx}, sparse={self.sparse}"


# ----------------------------------------------------------------- layer norm
def _params(x, weight, bias):
    """dim and the type code of weight and bias (x's where there are none)."""
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"x must have rows of at least one column, not {tuple(shape)}")
    dim = shape[-1]
    xt = _type(x.dtype, "x")
    pt = None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (dim,):
            raise ValueError(f"{name} must have shape ({dim},), not {tuple(p.shape)}")
        if not p.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        t = _type(p.dtype, name)
        if pt is not None and t != pt:
            raise ValueError("weight and bias must have one type")
        pt = t
    if pt is None:
        pt = xt
    if pt not in (xt, 0):
        raise ValueError("weight and bias must have x's type or float32")
    return dim, xt, pt


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _span(ws):
    """Address and bytes of a workspace, or none."""
    return (0, 0) if ws is None else (ws.data_ptr(), ws.numel())


def _layer_norm_forward(x, weight, bias, eps, stats):
    dim, xt, pt = _params(x, weight, bias)
    device = _device_of(x, weight, bias)
    rows, stride = _as_rows(x, dim)
    n = rows.shape[0]
    y = _new_like(x)
    mean = rstd = None
    if stats:
        mean = x.new_empty(n, dtype=torch.float32)
        rstd = x.new_empty(n, dtype=torch.float32)
    _store_module().layer_norm(device, y.data_ptr(), dim, _ptr(mean), _ptr(rstd), rows.data_ptr(), xt,
                               stride, _ptr(weight), _ptr(bias), pt, n, dim, eps, _raw_stream(device))
    return y, mean, rstd


def layer_norm_grad(grad, x, mean, rstd, weight=None, need=(True, True, True), param_dtype=None):
    """``(dx, dweight, dbias)`` of ``layer_norm`` from the gradient of its
    output and the mean and rstd of every row (float32, as
    ``layer_norm_stats`` returns them). ``need`` says which are wanted (None for
    the others). dweight and dbias have weight's type; without a weight,
    ``param_dtype`` (x's by default, or float32)."""
    if _forward_ad._current_level >= 0 or _dispatch_modes() or _is_tracing():
        _check_transforms_and_trace("layer_norm_grad", grad, x, mean, rstd, weight)
    dim, xt, pt = _params(x, weight, None)
    ptype = weight.dtype if weight is not None else param_dtype or x.dtype
    if weight is None:
        if ptype not in (x.dtype, torch.float32):
            raise ValueError("param_dtype must be x's type or float32")
        pt = _TYPES[ptype]
    if grad.shape != x.shape or grad.dtype != x.dtype:
        raise ValueError(f"grad must be like x: {tuple(x.shape)} {x.dtype}, not {tuple(grad.shape)} {grad.dtype}")
    device = _device_of(x, grad, mean, rstd, weight)
    xr, x_stride = _as_rows(x, dim)
    gr, g_stride = _as_rows(grad, dim)
    n = xr.shape[0]
    for name, s in (("mean", mean), ("rstd", rstd)):
        if s.dtype != torch.float32 or s.numel() != n or not s.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 tensor of {n} elements")
    m = _store_module()
    few = dim <= 4096 and n * max(dim, 128) <= _FEW_NORM
    dx = _new_like(x) if need[0] else None
    like = weight if weight is not None else x.new_empty(0, dtype=ptype)
    dw = like.new_empty(dim) if need[1] else None
    db = like.new_empty(dim) if need[2] else None
    ws = None  # few rows, and dx alone, need none
    if not few and (need[1] or need[2]):
        ws = x.new_empty(m.layer_norm_grad_workspace(n, dim), dtype=torch.uint8)
    m.layer_norm_grad(device, _ptr(dx), dim if need[0] else 0, _ptr(dw), _ptr(db), gr.data_ptr(),
                      g_stride, xr.data_ptr(), xt, x_stride, _ptr(weight), pt, mean.data_ptr(),
                      rstd.data_ptr(), n, dim, *_span(ws), _raw_stream(device))
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _layer_norm_forward(x, weight, bias, eps, True)
        ctx.bias_type = None if bias is None else bias.dtype
        ctx.save_for_backward(x, mean, rstd, weight)
        return y

    @staticmethod
    @_first_derivative
    def backward(ctx, saved, grad):
        x, mean, rstd, weight = saved
        return *layer_norm_grad(grad, x, mean, rstd, weight, ctx.needs_input_grad[:3], ctx.bias_type), None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension of ``x``: ``(x - mean) / sqrt(var +
    eps) * weight + bias`` in x's type; weight and bias [dim] are of x's type or
    float32, or None. Differentiable in all three."""
    if _forward_ad._current_level >= 0 or _dispatch_modes():
        _check_transforms(x, weight, bias)
    if _is_tracing() or (
            torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                         or (bias is not None and bias.requires_grad))):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _layer_norm_forward(x, weight, bias, float(eps), False)[0]


def layer_norm_stats(x, weight=None, bias=None, eps=1e-5):
    """``(y, mean, rstd)``: ``layer_norm`` (without autograd) and the float32
    statistics of every row that ``layer_norm_grad`` takes."""
    if _forward_ad._current_level >= 0 or _dispatch_modes() or _is_tracing():
        _check_transforms_and_trace("layer_norm_stats", x, weight, bias)
    return _layer_norm_forward(x, weight, bias, float(eps), True)


class LayerNorm(torch.nn.Module):
    """``layer_norm`` with learnable weight and bias (``affine``; ``bias=False`` leaves the bias out)."""

    def __init__(self, dim, eps=1e-5, affine=True, bias=True, dtype=torch.float32, device=None):
        super().__init__()
        self.dim, self.eps = int(dim), float(eps)
        self.weight = torch.nn.Parameter(torch.ones(self.dim, dtype=dtype, device=device)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(self.dim, dtype=dtype, device=device)) if affine and bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}, affine={self.weight is not None}"
