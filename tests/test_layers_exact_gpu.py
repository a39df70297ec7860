"""The embedding gradient on small whole numbers, whose float32 sums are exact in any
order: results are compared for equality, so that one row too few or too
many in a long sum shows. Also int32 ids, and the one-kernel form of few ids
against the sorted form bit for bit."""
import ctypes

import pytest
import torch

from gids_abi import GIDS_E_RANGE, check
from layers_ref import CODES, TYPES, abi, bits

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def layers(built):
    from GIDS import layers

    return layers


def whole(n, dim, dtype, seed=0):
    """-3 .. 3, zero left out: every sum of up to 2^22 of them is a float32 number, whatever the order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    v = torch.randint(1, 4, (n, dim), generator=g, device=DEV)
    sign = torch.randint(0, 2, (n, dim), generator=g, device=DEV) * 2 - 1
    return (v * sign).to(TYPES[dtype])


def sums(ids, grad, num_rows, pad=None):
    """The exact sums by id, as float32, and which ids occur."""
    ids = ids.long()
    keep = (ids >= 0) & (ids < num_rows)
    if pad is not None:
        keep &= ids != pad
    s = torch.zeros((num_rows, grad.shape[1]), dtype=torch.int64, device=DEV)
    s.index_add_(0, ids[keep], grad[keep].long())
    return s.float(), torch.unique(ids[keep])


def check_exact(layers, ids, grad, num_rows, pad=None):
    want, rows = sums(ids, grad, num_rows, pad)
    dw = layers.embedding_grad(ids, grad, num_rows, 1.0, pad, torch.float32)
    assert torch.equal(dw, want)
    r, v = layers.embedding_grad_rows(ids, grad, num_rows, 1.0, pad, torch.float32)
    assert torch.equal(r, rows) and torch.equal(v, want[rows])
    half = layers.embedding_grad(ids, grad, num_rows, 0.5, pad, torch.float32)  # a power of two is exact too
    assert torch.equal(half, 0.5 * want)
    return dw


# 256 blocks of sums and more, where a run's partial sums are found by a scan and
# added by several teams, lie behind 262,144 ids
@pytest.mark.parametrize("dim,t", [(1, "f32"), (3, "bf16"), (8, "f16"), (33, "f32"), (128, "f32"), (130, "bf16"),
                                   (264, "f16")])
@pytest.mark.parametrize("n", [300, 65536, 300000, 303109])
@pytest.mark.parametrize("rows", [1, 2, 7])
def test_long_runs_are_exact(layers, n, rows, dim, t):
    ids = torch.arange(n, device=DEV) * rows // n  # runs of equal length
    ids = ids[torch.randperm(n, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)]
    grad = whole(n, dim, t, seed=dim)
    dw = check_exact(layers, ids, grad, rows)
    # the comparison sees a single row that is left out, and so a block of them
    short, _ = sums(ids[:-1], grad[:-1], rows)
    assert not torch.equal(dw, short)
    check_exact(layers, ids, grad, rows, pad=rows - 1)


@pytest.mark.parametrize("dim,t", [(1024, "bf16"), (1001, "f32"), (2056, "f16")])
@pytest.mark.parametrize("n", [5000, 70001])
def test_wide_rows_are_exact(layers, n, dim, t):
    for rows in (1, 3, 400):
        ids = torch.randint(0, rows, (n,), generator=torch.Generator(device=DEV).manual_seed(dim), device=DEV)
        check_exact(layers, ids, whole(n, dim, t), rows)


@pytest.mark.parametrize("n", [127, 128, 129, 1000, 8193, 32769, 75777, 200000, 303105])
@pytest.mark.parametrize("dim,t", [(4, "f32"), (24, "f16"), (67, "bf16")])
def test_skewed_ids_are_exact(layers, n, dim, t):
    """A few ids take most of the list, the others occur once or not at all; ids behind the table are left out."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    for num_rows in (50, 70000):
        ids = (torch.rand(n, generator=gen, device=DEV, dtype=torch.float64).pow(8) * num_rows).long()
        check_exact(layers, ids, whole(n, dim, t, seed=n), num_rows, pad=num_rows // 2)
    ids[n // 2] = num_rows
    ids[0] = -1
    want, _ = sums(ids, grad := whole(n, dim, t, seed=n), num_rows)
    dw = layers.embedding_grad(ids, grad, num_rows, 1.0, None, torch.float32)
    assert torch.equal(dw, want)
    with pytest.raises(RuntimeError, match="outside its table"):
        layers.check_ids(DEV)


@pytest.mark.parametrize("n", [1, 5, 128, 129, 1024, 5000, 32768, 32769, 75777, 310001])
@pytest.mark.parametrize("rows", [3, 70000, (1 << 31) + 5])
def test_int32_ids(layers, n, rows):
    """The gradient of int32 ids is that of the same int64 ids; a negative one is outside every table."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    ids = torch.randint(0, min(rows, (1 << 31) - 1), (n,), generator=gen, device=DEV, dtype=torch.int32)
    grad = torch.randn(n, 20, generator=gen, device=DEV)
    for bad in (False, True):
        if bad:
            ids[n // 2] = -7
        got = layers.embedding_grad_rows(ids, grad, rows, 2.0, 1)
        if bad:
            with pytest.raises(RuntimeError, match="outside its table"):
                layers.check_ids(DEV)
        want = layers.embedding_grad_rows(ids.long(), grad, rows, 2.0, 1)
        if bad:
            with pytest.raises(RuntimeError, match="outside its table"):
                layers.check_ids(DEV)
        assert torch.equal(got[0], want[0]) and torch.equal(bits(got[1]), bits(want[1]))
        assert got[0].tolist() == [i for i in torch.unique(ids).tolist() if i >= 0 and i != 1]
    if rows <= 70000:
        ids[n // 2] = 0
        assert torch.equal(bits(layers.embedding_grad(ids, grad, rows, 2.0, 1)),
                           bits(layers.embedding_grad(ids.long(), grad, rows, 2.0, 1)))
        check_exact(layers, ids, whole(n, 20, "f32"), rows, 1)


@pytest.mark.parametrize("dim", [1, 8, 24, 130, 257, 1024])
@pytest.mark.parametrize("n", [1, 2, 31, 33, 64, 100, 127, 128])
def test_few_ids_add_as_the_sorted_list_does(layers, n, dim):
    """One kernel for up to 128 ids, and the sort with its sums: the same bits."""
    L = abi()
    st = torch.cuda.current_stream().cuda_stream
    gen = torch.Generator(device=DEV).manual_seed(n)
    rows = 90
    lists = [torch.full((n,), 5, device=DEV), torch.randint(0, rows, (n,), generator=gen, device=DEV),
             torch.randint(0, 3, (n,), generator=gen, device=DEV), (torch.arange(n, device=DEV) * 3) // max(n, 1)]
    for gt, vt in (("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")):
        grad = torch.randn(n, dim, generator=gen, device=DEV).to(TYPES[gt])
        for ids in lists:
            b, count = ctypes.c_uint64(), ctypes.c_uint64()
            check(L.gids_embedding_grad_workspace(n, rows, dim, ctypes.byref(b)))
            ws = torch.empty(b.value, dtype=torch.uint8, device=DEV)
            check(L.gids_embedding_group(0, ids.data_ptr(), 8, n, rows, 2, dim, ws.data_ptr(), b.value, None,
                                         ctypes.byref(count), st))
            r = torch.empty(n, dtype=torch.int64, device=DEV)
            v = torch.empty(n, dim, dtype=TYPES[vt], device=DEV)
            check(L.gids_embedding_grad_rows(0, r.data_ptr(), v.data_ptr(), CODES[v.dtype], dim, n, rows, dim,
                                             grad.data_ptr(), CODES[grad.dtype], dim, n, 0.3, ws.data_ptr(), b.value,
                                             st))
            k = count.value
            few = layers.embedding_grad_rows(ids, grad, rows, 0.3, 2, v.dtype)
            dense = layers.embedding_grad(ids, grad, rows, 0.3, 2, v.dtype)
            assert torch.equal(few[0], r[:k]) and torch.equal(bits(few[1]), bits(v[:k]))
            assert torch.equal(bits(dense[few[0]]), bits(v[:k]))


def test_int32_ids_through_the_abi_report(layers):
    L = abi()
    ids = torch.tensor([4, -1, 9], dtype=torch.int32, device=DEV)
    grad, dw = whole(3, 8, "f32"), torch.empty(9, 8, device=DEV)
    check(L.gids_embedding_grad(0, dw.data_ptr(), 0, 8, 9, 8, grad.data_ptr(), 0, 8, ids.data_ptr(), 4, 3, -1, 1.0, None,
                                0, None))
    assert L.gids_embedding_check(0, None) == GIDS_E_RANGE
    assert torch.equal(dw[4], grad[0]) and not dw[:4].any() and not dw[5:].any()
