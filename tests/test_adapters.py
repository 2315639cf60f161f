"""The pool of low-rank adapters on the CPU: shapes, loading, and the rows of a step."""

import pytest
import torch

from fms_model_optimizer_b200 import ops
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


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_rows_of_adapters_from_integers_of_any_width(dtype):
    rows, starts = ops.lora_groups(torch.tensor([1, 0, 127, 1], dtype=dtype), 300)
    assert rows.tolist() == [1, 0, 3, 2]
    assert starts.tolist() == [0, 1] + [3] * 126 + [4] * 173


def test_the_pool_takes_trained_weights_without_their_graph_and_names_what_it_lacks():
    pool = LoraAdapters({"q": (16, 8)}, 1, 2, 8, "cpu")
    a, b = torch.nn.Parameter(torch.ones(8, 8)), torch.nn.Parameter(torch.ones(16, 8))
    pool.load(1, 0, "q", a, b)
    assert not pool.a[0, "q"].requires_grad and not pool.b[0, "q"].requires_grad
    for adapter, layer, name in ((-1, 0, "q"), (2, 0, "q"), (0, 1, "q"), (0, 0, "k")):
        with pytest.raises(RuntimeError, match="there is no adapter"):
            pool.load(adapter, layer, name, a, b)
    with pytest.raises(RuntimeError, match="has weights"):
        pool.load(0, 0, "q", torch.tensor(1.0), b)
