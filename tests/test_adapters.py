"""The pool of low-rank adapters on the CPU: shapes, loading, and the rows of a step."""

import pytest
import torch

from fms_model_optimizer_b200.adapters import LoraAdapters

SHAPES = dict(q=(64, 32), down=(32, 96))


def test_pool_and_loading():
    pool = LoraAdapters(SHAPES, 2, 3, 12, "cpu")
    assert pool.a[1, "q"].shape == (3, 16, 32) and pool.b[0, "down"].shape == (3, 32, 16) and pool.scale.tolist() == [1.0] * 3
    g = torch.Generator().manual_seed(0)
    a, b = torch.randn(12, 32, generator=g), torch.randn(64, 12, generator=g)
    pool.load(2, 1, "q", a, b)
    assert torch.equal(pool.a[1, "q"][2, :12], a.bfloat16()) and torch.equal(pool.b[1, "q"][2, :, :12], b.bfloat16())
    assert int(pool.a[1, "q"][2, 12:].count_nonzero()) == 0 and int(pool.a[1, "q"][:2].count_nonzero()) == 0
    pool.load(2, 1, "q", a[:4], b[:, :4])  # a lower rank in the same place
    assert int(pool.a[1, "q"][2, 4:].count_nonzero()) == 0 and int(pool.b[1, "q"][2, :, 4:].count_nonzero()) == 0
    for bad in ((a[:, :31], b), (a, b[:63]), (a, b[:, :11]), (torch.zeros(13, 32), torch.zeros(64, 13))):
        with pytest.raises(RuntimeError, match="weights"):
            pool.load(0, 0, "q", *bad)
    assert set(LoraAdapters(SHAPES, 1, 1, 8, "cpu", names=["down"]).a) == {(0, "down")}
    for bad in (dict(rank=0), dict(rank=129), dict(adapters=0), dict(layers=0), dict(dtype=torch.float32)):
        with pytest.raises(RuntimeError):
            LoraAdapters(SHAPES, **{**dict(layers=1, adapters=1, rank=8, dev="cpu"), **bad})


def test_rows_of_a_step():
    pool = LoraAdapters(SHAPES, 1, 3, 8, "cpu")
    which = pool.which([2, -1, 0], [2, 3, 1], "cpu", 2)
    assert which.tolist() == [-1, -1, 2, 2, -1, -1, -1, 0]
    step = pool.step(which)
    assert step.starts.tolist() == [0, 1, 1, 3] and step.rows[:3].tolist() == [7, 2, 3]
    y = torch.zeros(8, 32)
    assert LoraAdapters(SHAPES, 1, 3, 8, "cpu", names=["q"]).step(which).add_(0, "down", y, y) is y  # no adapters there
    for bad in (([3, 0], [1, 1]), ([-2, 0], [1, 1]), ([0], [1, 1])):
        with pytest.raises(RuntimeError, match="every prompt"):
            pool.which(*bad, "cpu")
