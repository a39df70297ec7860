"""GIDS.fetch_feature with the model's input layers (node_embeddings,
feature_norm): which rows are gathered, marked and looked up, on the CPU
against a fake store."""
import types

import numpy as np
import pytest
import torch

from oracle import oracle
from test_gids_policy import FakeStore, batches, fake  # noqa: F401


class Table:
    """Stands in for a NodeEmbedding on the CPU: remembers its ids."""

    def __init__(self, rows, dim):
        self.rows = torch.arange(rows * dim, dtype=torch.float32).view(rows, dim)
        self.seen = []

    def __call__(self, ids):
        self.seen.append(ids.tolist())
        return self.rows[ids]


def hetero(n, seed=0, sizes=None):
    rng = np.random.default_rng(seed)
    sizes = sizes or {"paper": 30, "author": 20, "fos": 10}
    return [[{k: torch.as_tensor(rng.integers(0, 100, size=m)) for k, m in sizes.items()}, f"seeds{i}", f"blocks{i}"]
            for i in range(n)]


MAP = {"paper": 0, "author": 300, "fos": 600}


def expect(ids, off=0):
    return oracle.gather(FakeStore.table, ids.numpy(), key_off=off)


def test_embedded_types_are_not_gathered(fake):  # noqa: F811
    t = Table(100, 8)
    g = fake(heterograph=True, heterograph_map={k: v for k, v in MAP.items() if k != "author"},
             node_embeddings={"author": t}, window_buffer=True, wb_size=2)
    bs = hetero(6)
    it = iter([list(b) for b in bs])
    for b in bs[:3]:
        out = g.fetch_feature(64, it, "cpu")
        feats = out[-1]
        assert list(feats) == ["paper", "author", "fos"] and out[1] == b[1]
        assert torch.equal(feats["author"], t.rows[b[0]["author"]])
        for k in ("paper", "fos"):
            assert np.array_equal(feats[k].numpy(), expect(b[0][k], MAP[k]))
    calls = g.BAM_FS.calls
    assert [c[2] for c in calls if c[0] == "read_feature_hetero"] == [[30, 10]] * 3
    marked = [c[1] for c in calls if c[0] == "wb"]
    assert len(marked) == 2 * 5 and all(len(m) in (30, 10) for m in marked)
    g.drop_window_buffer()
    assert sum(c[0] == "unset_window_buffering" for c in g.BAM_FS.calls) == 2 * 2


def test_accumulator_looks_up_when_a_batch_is_handed_out(fake):  # noqa: F811
    t = Table(100, 4)
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": t}, accumulator_flag=True)
    g.required_accesses = 100  # three batches of 40 stored rows each
    bs = hetero(7, seed=2)
    it = iter([list(b) for b in bs])
    out = [g.fetch_feature(64, it, "cpu")]
    assert [c[1] for c in g.BAM_FS.calls if c[0] == "read_feature_hetero"] == [6]
    t.rows = t.rows + 1000.0  # the optimiser's step between two batches
    out.append(g.fetch_feature(64, it, "cpu"))
    assert torch.equal(out[0][-1]["author"], t.rows[bs[0][0]["author"]] - 1000.0)
    assert torch.equal(out[1][-1]["author"], t.rows[bs[1][0]["author"]])
    assert np.array_equal(out[1][-1]["paper"].numpy(), expect(bs[1][0]["paper"]))


def test_empty_and_missing_embedded_types(fake):  # noqa: F811
    t = Table(50, 8)
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": t, "venue": t})
    b = hetero(1, sizes={"paper": 5, "author": 0})[0]
    feats = g.fetch_feature(64, iter([b]), "cpu")[-1]
    assert set(feats) == {"paper", "author"} and feats["author"].shape == (0, 8)


def test_norm_of_homogeneous_and_typed_features(fake):  # noqa: F811
    g = fake(feature_norm=lambda x: x * 2)
    b = batches(1, 12)[0]
    out = g.fetch_feature(64, iter([list(b)]), "cpu")
    assert np.array_equal(out[-1].numpy(), 2 * expect(b[0]))
    t = Table(100, 64)
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": t},
             feature_norm={"paper": lambda x: x + 1, "author": lambda x: -x})
    h = hetero(1)[0]
    f = g.fetch_feature(64, iter([list(h)]), "cpu")[-1]
    assert np.array_equal(f["paper"].numpy(), expect(h[0]["paper"]) + 1)
    assert torch.equal(f["author"], -t.rows[h[0]["author"]])
    assert np.array_equal(f["fos"].numpy(), expect(h[0]["fos"], 600))
    g = fake(heterograph=True, heterograph_map=MAP, feature_norm=lambda x: x * 3)
    f = g.fetch_feature(64, iter([list(h)]), "cpu")[-1]
    assert all(np.array_equal(f[k].numpy(), 3 * expect(h[0][k], MAP[k])) for k in MAP)


def test_constructor_refusals(fake):  # noqa: F811
    with pytest.raises(ValueError, match="heterograph"):
        fake(node_embeddings={"author": Table(3, 4)})
    with pytest.raises(ValueError, match="heterograph"):
        fake(feature_norm={"author": Table(3, 4)})


def test_accumulator_with_nothing_stored_takes_one_batch_at_a_time(fake):  # noqa: F811
    t = Table(100, 4)
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": t}, accumulator_flag=True)
    bs = hetero(5, seed=3, sizes={"author": 7})
    it = iter([list(b) for b in bs])
    for i, b in enumerate(bs):
        out = g.fetch_feature(64, it, "cpu")
        assert out[1] == b[1] and torch.equal(out[-1]["author"], t.rows[b[0]["author"]])
    assert len(t.seen) == 5


class Plus(torch.nn.Module):
    def __init__(self, by):
        super().__init__()
        self.by = by

    def forward(self, x):
        return x + self.by


@pytest.mark.parametrize("accumulator", [False, True])
def test_norms_in_a_module_dict(fake, accumulator):  # noqa: F811
    """The way a model registers its norms by node type."""
    t = Table(100, 64)
    norms = torch.nn.ModuleDict({"paper": Plus(1.0), "author": Plus(2.0)})
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": t}, feature_norm=norms,
             accumulator_flag=accumulator)
    bs = hetero(2, seed=8)
    it = iter([list(b) for b in bs])
    f = g.fetch_feature(64, it, "cpu")[-1]
    assert np.array_equal(f["paper"].numpy(), expect(bs[0][0]["paper"]) + 1)
    assert torch.equal(f["author"], t.rows[bs[0][0]["author"]] + 2)
    assert np.array_equal(f["fos"].numpy(), expect(bs[0][0]["fos"], 600))
    norms["fos"] = Plus(3.0)  # the loader holds the model's dict, not a copy
    f = g.fetch_feature(64, it, "cpu")[-1]
    assert np.array_equal(f["fos"].numpy(), expect(bs[1][0]["fos"], 600) + 3)
    h = hetero(1)[0]
    g = fake(heterograph=True, heterograph_map=MAP, feature_norm=types.MappingProxyType({"paper": Plus(1.0)}))
    f = g.fetch_feature(64, iter([list(h)]), "cpu")[-1]
    assert np.array_equal(f["paper"].numpy(), expect(h[0]["paper"]) + 1)
    for typed in (norms, types.MappingProxyType({"paper": Plus(1.0)})):
        with pytest.raises(ValueError, match="heterograph"):
            fake(feature_norm=typed)


class Reports(Table):
    """Raises in the calls named, as the table's lookup does for ids of an earlier call."""

    def __init__(self, rows, dim, at):
        super().__init__(rows, dim)
        self.at = at

    def __call__(self, ids):
        if len(self.seen) in self.at:
            self.seen.append(None)
            raise RuntimeError("an id of an earlier embedding call lay outside its table")
        return super().__call__(ids)


@pytest.mark.parametrize("kw", [{}, dict(window_buffer=True, wb_size=2), dict(accumulator_flag=True)],
                         ids=lambda kw: next(iter(kw), "plain"))
def test_a_report_loses_no_batch(fake, kw):  # noqa: F811
    t = Reports(100, 8, {1, 3})
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": t}, **kw)
    g.required_accesses = 100
    bs = hetero(9, seed=5)
    it = iter([list(b) for b in bs])
    got, raised = [], 0
    while len(got) < 4:
        try:
            got.append(g.fetch_feature(64, it, "cpu"))
        except RuntimeError:
            raised += 1
    assert raised == 2
    for out, b in zip(got, bs):
        assert out[1] == b[1] and torch.equal(out[-1]["author"], t.rows[b[0]["author"]])
        assert np.array_equal(out[-1]["paper"].numpy(), expect(b[0]["paper"]))
        assert len(out) == 4


def test_a_batch_that_raises_twice_is_given_up(fake):  # noqa: F811
    t = Reports(100, 8, {0, 1})
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": t})
    bs = hetero(2, seed=6)
    it = iter([list(b) for b in bs])
    for _ in range(2):
        with pytest.raises(RuntimeError, match="earlier"):
            g.fetch_feature(64, it, "cpu")
    assert g.fetch_feature(64, it, "cpu")[1] == bs[1][1]
    g = fake(heterograph=True, heterograph_map=MAP, node_embeddings={"author": Reports(100, 8, {0})})
    it = iter([list(b) for b in bs])
    with pytest.raises(RuntimeError):
        g.fetch_feature(64, it, "cpu")
    g.drop_window_buffer()  # nothing of the old window is left
    assert g.fetch_feature(64, it, "cpu")[1] == bs[1][1]
