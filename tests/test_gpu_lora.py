"""Low-rank adapters of many requests added to a projection's output, against 64 bits.

Bounds (w: width, r: rank).  v = x a^T is an fp32 sum of w products, (w + 16) 2^-23 of sum |x a| off; as two 16-bit numbers it keeps 2^-16 of itself in
bf16, in fp16 2^-21 of the row's largest.  What v is off by reaches y through |b|; the second sum, of 2 r products, is (2 r + 16) 2^-23 of
sum |v b| off.  y is rounded once, half a step.
"""

import pytest
import torch

from fms_model_optimizer_b200 import ops
from oracle import requests as OR

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _half_step(want, dtype):
    exponent = torch.frexp(want.abs())[1].clamp(min={torch.float16: -13, torch.bfloat16: -125}[dtype])
    return torch.ldexp(torch.full_like(want, U[dtype]), exponent - 1)


def _near(got, y, x, a, b, which, scale):
    dtype = y.dtype
    want, v, size, rows = OR.lora(y, x, a, b, which, scale)
    bound = _half_step(want, dtype) * (1 + 2.0**-10)
    w, r = x.shape[1], a.shape[1]
    for i, at in rows.items():
        if at.numel() == 0:
            continue
        off = (w + 16) * 2.0**-23 * size[i]
        off += 2.0**-16 * v[i].abs() if dtype == torch.bfloat16 else 2.0**-21 * v[i].abs().amax(-1, keepdim=True)
        off += (2 * r + 16) * 2.0**-23 * v[i].abs()
        bound[at] += scale[i].abs().double() * (off @ b[i].double().abs().t())
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    none = ~((which >= 0) & (which < a.shape[0]))
    assert torch.equal(got[none], y[none]), "rows without an adapter were written"


def _inputs(seed, tokens, adapters, rank, width, out, dtype, without=0.2):
    g = torch.Generator().manual_seed(seed)
    x, y = (torch.randn((tokens, n), generator=g).to(dtype) for n in (width, out))
    a = (torch.randn((adapters, rank, width), generator=g) * width**-0.5).to(dtype)
    b = torch.randn((adapters, out, rank), generator=g).to(dtype)
    which = torch.randint(0, max(adapters, 1), (tokens,), generator=g)
    which[torch.rand(tokens, generator=g) < without] = -1
    return y, x, a, b, which, torch.rand(adapters, generator=g) + 0.5


def _run(dev, y, x, a, b, which, scale):
    d = [t.to(dev) for t in (y, x, a, b)]
    rows, starts = ops.lora_groups(which.to(dev), a.shape[0])
    got = ops.lora_add_(*d, rows, starts, scale.to(dev))
    assert got.data_ptr() == d[0].data_ptr()
    ops.check_status(dev)
    return got.cpu()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,adapters,rank,width,out", [
    (1, 1, 16, 4096, 4096), (1, 40, 8, 64, 72), (17, 3, 16, 264, 520), (64, 16, 16, 1024, 2056), (200, 5, 24, 776, 8), (33, 2, 32, 8, 1000), (70, 3, 64, 2048, 136),
    (45, 2, 128, 1096, 264), (300, 1, 40, 512, 512), (5000, 3, 16, 520, 264), (6001, 7, 64, 136, 328), (5003, 100, 32, 264, 72), (16, 4, 120, 4104, 4096)])  # fmt: skip
def test_against_64_bits(cuda_dev, dtype, tokens, adapters, rank, width, out):
    case = _inputs(tokens + rank, tokens, adapters, rank, width, out, dtype, 0.0 if tokens == 1 else 0.2)
    _near(_run(cuda_dev, *case), *case)


def test_groups():
    """The rows of each adapter, in rising order, whatever the type of `which`; on the CPU too."""
    which = torch.tensor([2, -1, 0, 2, 7, 1, 0, -100, 2])
    for w in (which, which.int(), which.to(torch.int16)):
        rows, starts = ops.lora_groups(w, 4)
        assert starts.tolist() == [0, 2, 3, 6, 6] and rows.dtype == starts.dtype == torch.int32
        assert rows[:6].tolist() == [2, 6, 5, 0, 3, 8]
    rows, starts = ops.lora_groups(which[:0], 2)
    assert starts.tolist() == [0, 0, 0] and rows.numel() == 0
    for bad in (which.float(), which.view(3, 3)):
        with pytest.raises(RuntimeError):
            ops.lora_groups(bad, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_views_and_strides(cuda_dev, dtype):
    """Columns of a wider output (a fused projection's), rows with a pitch, adapters that are every other one of a pool, and rows that fit no 16 bytes."""
    y, x, a, b, which, scale = _inputs(5, 50, 3, 16, 256, 128, dtype)
    rows, starts = ops.lora_groups(which.to(cuda_dev), 3)
    wide = torch.zeros(50, 512, dtype=dtype, device=cuda_dev)
    wide[:, 64:192] = y.to(cuda_dev)
    dx = torch.zeros(50, 300, dtype=dtype, device=cuda_dev)
    dx[:, 3:259] = x.to(cuda_dev)
    pool_a, pool_b = torch.zeros(6, 20, 264, dtype=dtype, device=cuda_dev), torch.zeros(6, 128, 24, dtype=dtype, device=cuda_dev)
    pool_a[::2, 2:18, :256], pool_b[::2, :, 8:] = a.to(cuda_dev), b.to(cuda_dev)
    got = ops.lora_add_(wide[:, 64:192], dx[:, 3:259], pool_a[::2, 2:18, :256], pool_b[::2, :, 8:], rows, starts, scale.to(cuda_dev))
    _near(got.cpu(), y, x, a, b, which, scale)
    assert int(wide[:, :64].count_nonzero()) == 0 and int(wide[:, 192:].count_nonzero()) == 0
    odd = torch.zeros(50, 131, dtype=dtype, device=cuda_dev)
    odd[:, 1:129] = y.to(cuda_dev)
    got = ops.lora_add_(odd[:, 1:129], x.to(cuda_dev).t().contiguous().t(), a.to(cuda_dev), b.to(cuda_dev).transpose(1, 2).contiguous().transpose(1, 2), rows, starts, scale.to(cuda_dev))
    _near(got.cpu(), y, x, a, b, which, scale)
    assert got.data_ptr() == odd[:, 1:].data_ptr() and int(odd[:, 129:].count_nonzero()) == 0


def test_rows_in_any_order(cuda_dev):
    """A row's result does not depend on its place among the rows of its adapter, nor on what others there are."""
    y, x, a, b, which, scale = _inputs(6, 80, 2, 32, 512, 256, torch.bfloat16, 0.0)
    first = _run(cuda_dev, y, x, a, b, which, scale)
    rows, starts = ops.lora_groups(which.to(cuda_dev), 2)
    n = int(starts[1])
    mixed = torch.cat([rows[:n].flip(0), rows[n:].flip(0)])
    dev = [t.to(cuda_dev) for t in (x, a, b)]
    assert torch.equal(ops.lora_add_(y.to(cuda_dev), *dev, mixed, starts, scale.to(cuda_dev)).cpu(), first)
    again = ops.lora_add_(y.to(cuda_dev), *dev, rows, starts, scale.to(cuda_dev)).cpu()
    assert torch.equal(again, first)


def test_large_sums_in_fp16(cuda_dev):
    """v far outside fp16, on both sides, where y is not."""
    y, x, a, b, which, scale = _inputs(7, 40, 2, 16, 512, 64, torch.float16, 0.0)
    for up, down in ((2.0**9, 2.0**-13), (2.0**-10, 2.0**8)):
        xs, bs = x * up, b * down
        a2 = (a * 2.0**8 if up > 1 else a * 2.0**-6).half()
        s = scale * (1.0 if up > 1 else 2.0**8)
        _near(_run(cuda_dev, y, xs, a2, bs, which, s), y, xs, a2, bs, which, s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_and_nan_stay_in_their_rows(cuda_dev, dtype):
    y, x, a, b, which, scale = _inputs(8, 30, 2, 16, 128, 64, dtype, 0.0)
    clean = _run(cuda_dev, y, x, a, b, which, scale)
    x[4, 7] = float("nan")
    x[9, 0] = float("inf")
    got = _run(cuda_dev, y, x, a, b, which, scale)
    keep = torch.ones(30, dtype=torch.bool)
    keep[[4, 9]] = False
    assert torch.equal(got[keep], clean[keep]) and bool(got[4].isnan().all())
    want = OR.lora(y, x, a, b, which, scale)[0][9].to(dtype)
    assert torch.equal(got[9].isnan(), want.isnan()) and torch.equal(got[9].nan_to_num(1.0, 2.0, 3.0), want.nan_to_num(1.0, 2.0, 3.0))
    # what a row without an adapter holds reaches nobody
    which[4] = -1
    assert torch.equal(_run(cuda_dev, y, x, a, b, which, scale)[4], y[4])


def test_empty_calls(cuda_dev):
    y, x, a, b, which, scale = _inputs(9, 12, 2, 16, 64, 64, torch.bfloat16)
    none = torch.full_like(which, -1)
    assert torch.equal(_run(cuda_dev, y, x, a, b, none, scale), y)
    assert torch.equal(_run(cuda_dev, y, x, a[:0], b[:0], none, scale[:0]), y)
    assert _run(cuda_dev, y[:0], x[:0], a, b, which[:0], scale).shape == (0, 64)


def test_offsets_beyond_32_bits(cuda_dev):
    """Rows of x and y, and adapters, more than 2^31 elements apart."""
    pitch = (1 << 30) + 8
    y, x, a, b, which, scale = _inputs(10, 3, 3, 16, 64, 64, torch.bfloat16, 0.0)
    which[:] = torch.tensor([2, 0, 1])
    room = torch.zeros(2 * pitch + 4096, dtype=torch.bfloat16, device=cuda_dev)
    dx, dy = room.as_strided((3, 64), (pitch, 1), 0), room.as_strided((3, 64), (pitch, 1), 64)
    da, db = room.as_strided((3, 16, 64), (pitch, 64, 1), 128), room.as_strided((3, 64, 16), (pitch, 16, 1), 128 + 1024)
    for to, t in ((dx, x), (da, a), (db, b)):
        to.copy_(t)
    dy.copy_(y)
    rows, starts = ops.lora_groups(which.to(cuda_dev), 3)
    got = ops.lora_add_(y.to(cuda_dev), dx, da, db, rows, starts, scale.to(cuda_dev))
    _near(got.cpu(), y, x, a, b, which, scale)
    got = ops.lora_add_(dy, x.to(cuda_dev), a.to(cuda_dev), b.to(cuda_dev), rows, starts, scale.to(cuda_dev))
    _near(got.cpu(), y, x, a, b, which, scale)


def test_bad_rows_and_starts_are_reported(cuda_dev):
    y, x, a, b, which, scale = _inputs(11, 20, 2, 16, 64, 64, torch.bfloat16, 0.0)
    dev = [t.to(cuda_dev) for t in (x, a, b)]
    rows, starts = ops.lora_groups(which.to(cuda_dev), 2)
    good = ops.lora_add_(y.to(cuda_dev), *dev, rows, starts, scale.to(cuda_dev)).cpu()
    for bad in (-1, 20, 1 << 30):
        some = rows.clone()
        gone = int(some[3])
        some[3] = bad
        got = ops.lora_add_(y.to(cuda_dev), *dev, some, starts, scale.to(cuda_dev)).cpu()
        keep = torch.arange(20) != gone
        assert torch.equal(got[keep], good[keep]) and torch.equal(got[gone], y[gone])
        with pytest.raises(RuntimeError, match="status"):
            ops.check_status(cuda_dev)
    n = int(starts[1])
    for bad in ([0, n, 21], [0, n, n - 1], [-1, n, 20], [0, -5, 20], [1, n, 20]):
        ops.lora_add_(y.to(cuda_dev), *dev, rows, torch.tensor(bad, dtype=torch.int32, device=cuda_dev), scale.to(cuda_dev))
        with pytest.raises(RuntimeError, match="status"):
            ops.check_status(cuda_dev)


def test_refusals(cuda_dev):
    y, x, a, b, which, scale = (t.to(cuda_dev) for t in _inputs(12, 20, 2, 16, 64, 64, torch.bfloat16))
    rows, starts = ops.lora_groups(which, 2)
    ops.lora_add_(y.clone(), x, a, b, rows, starts, scale)
    for args in ((y.float(), x, a, b, rows, starts, scale), (y, x.half(), a, b, rows, starts, scale), (y, x[:, :60], a[:, :, :60], b, rows, starts, scale),
                 (y, x, a[:, :12], b[:, :, :12], rows, starts, scale), (y, x, a, b[:, :60], rows, starts, scale), (y, x, a, b, rows.long(), starts, scale),
                 (y, x, a, b, rows, starts[:2], scale), (y, x, a, b, rows, starts, scale[:1]), (y[:1].expand(20, 64), x, a, b, rows, starts, scale),
                 (y, x.cpu(), a, b, rows, starts, scale), (y, x, a[:1], b, rows, starts, scale), (y, x[:19], a, b, rows, starts, scale)):  # fmt: skip
        with pytest.raises(RuntimeError):
            ops.lora_add_(*args)
    with pytest.raises(RuntimeError, match="rank"):
        ops.lora_add_(y, x, x.new_zeros(2, 136, 64), x.new_zeros(2, 64, 136), rows, starts, scale)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.lora_add_(y, x, a.clone().requires_grad_(True), b, rows, starts, scale)


def test_streams_and_graphs(cuda_dev):
    y, x, a, b, which, scale = _inputs(13, 24, 4, 16, 512, 384, torch.bfloat16)
    rows, starts = ops.lora_groups(which.to(cuda_dev), 4)
    sy, sx, sa, sb, ss = (t.to(cuda_dev) for t in (y, x, a, b, scale))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _near(ops.lora_add_(sy.clone(), sx, sa, sb, rows, starts, ss).cpu(), y, x, a, b, which, scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.lora_add_(sy, sx, sa, sb, rows, starts, ss)
    for seed in (14, 15):  # other rows, adapters and requests of the same sizes
        y, x, a, b, which, scale = _inputs(seed, 24, 4, 16, 512, 384, torch.bfloat16)
        for to, t in ((sy, y), (sx, x), (sa, a), (sb, b), (ss, scale)):
            to.copy_(t)
        for to, t in zip((rows, starts), ops.lora_groups(which.to(cuda_dev), 4)):
            to.copy_(t)
        graph.replay()
        _near(sy.cpu(), y, x, a, b, which, scale)


def test_inputs_that_share_memory_with_the_output(cuda_dev):
    """x beside y in one buffer, and x that is y: read as they were before."""
    y, x, a, b, which, scale = _inputs(16, 300, 3, 16, 128, 128, torch.bfloat16)
    rows, starts = ops.lora_groups(which.to(cuda_dev), 3)
    da, db, ds = (t.to(cuda_dev) for t in (a, b, scale))
    both = torch.cat([x, y], 1).to(cuda_dev)
    _near(ops.lora_add_(both[:, 128:], both[:, :128], da, db, rows, starts, ds).cpu(), y, x, a, b, which, scale)
    assert torch.equal(both[:, :128].cpu(), x)
    same = y.to(cuda_dev)
    _near(ops.lora_add_(same, same, da, db, rows, starts, ds).cpu(), y, y, a, b, which, scale)


def _same_extremes(got, want):
    """NaN, infinities and their signs where 64 bits have them."""
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[want.isinf()].double(), want[want.isinf()])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,adapters,rank", [(30, 2, 8), (30, 2, 16), (5000, 2, 16), (30, 2, 32), (30, 2, 64), (5000, 2, 64), (30, 2, 128)])
def test_infinite_weights_reach_y_as_they_are(cuda_dev, dtype, tokens, adapters, rank):
    """Infinities and NaN in b: v times an infinity is one, whatever v's parts are, and outputs beside it stay as near as ever."""
    y, x, a, b, which, scale = _inputs(17, tokens, adapters, rank, 136, 72, dtype, 0.0)
    inf, clean = float("inf"), b.clone()
    b[0, 5, 3], b[1, 6, 0], b[1, 9, 2], b[1, 9, 7], b[0, 11, 1] = inf, -inf, inf, -inf, float("nan")
    got, want = _run(cuda_dev, y, x, a, b, which, scale), OR.lora(y, x, a, b, which, scale)[0]
    assert int(want.isinf().sum()) > tokens / 2
    _same_extremes(got, want)
    got[~want.isfinite()] = 0.0
    keep = want.isfinite()
    plain = _run(cuda_dev, y, x, a, clean, which, scale)
    assert torch.equal(got[keep], plain[keep])


def test_an_infinite_weight_meets_a_small_v(cuda_dev):
    """v in fp16 that is 2^-28 of the row's largest, below the last place of both its parts, is not zero where an infinity meets it."""
    y, x, a, b, which, scale = _inputs(18, 40, 2, 16, 136, 72, torch.float16, 0.0)
    a, b = a * 64, b / 64
    a[:, 3] = a[:, 3].sign() * 2.0**-24
    b[0, 5, 3], b[1, 6, 3] = float("inf"), float("-inf")
    v = OR.lora(y, x, a, b, which, scale)[1]
    assert all(bool((v[i][:, 3].abs() < 2.0**-25 * v[i].abs().amax(-1)).all()) and bool((v[i][:, 3] != 0).all()) for i in v)
    _same_extremes(_run(cuda_dev, y, x, a, b, which, scale), OR.lora(y, x, a, b, which, scale)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_infinite_sum_beside_large_ones(cuda_dev, dtype):
    """One infinite number of v leaves the others as they are, outside fp16 too: y is that infinity, not the difference of two."""
    y, x, a, b, which, scale = _inputs(19, 40, 2, 16, 136, 72, dtype, 0.0)
    x, a, b = x * 2.0**9, a * 2.0**12, (b * 2.0**-12).abs() * torch.randn(b.shape, generator=torch.Generator().manual_seed(20)).sign().to(dtype)
    a[0, 3, 7], a[1, 9, 0] = float("inf"), float("-inf")
    want, v, _, _ = OR.lora(y, x, a, b, which, scale)
    assert all(float(v[i][v[i].isfinite()].abs().max()) > 65504 for i in v)
    _same_extremes(_run(cuda_dev, y, x, a, b, which, scale), want)


def test_rows_of_y_that_overlap_are_refused(cuda_dev):
    """Blocks that write the same bytes would leave what comes last; rows that only lie between one another are fine."""
    y, x, a, b, which, scale = _inputs(21, 20, 2, 16, 64, 64, torch.bfloat16, 0.0)
    rows, starts = ops.lora_groups(which.to(cuda_dev), 2)
    rest = [t.to(cuda_dev) for t in (x, a, b)]
    room = torch.zeros(20 * 256, dtype=torch.bfloat16, device=cuda_dev)
    for strides in ((32, 1), (0, 1), (64, 0), (8, 8), (1, 1), (4, 6), (63, 1)):
        with pytest.raises(RuntimeError, match="share memory"):
            ops.lora_add_(room.as_strided((20, 64), strides), *rest, rows, starts, scale.to(cuda_dev))
    assert int(room.count_nonzero()) == 0
    for strides in ((64, 1), (1, 20), (2, 41), (192, 3), (3, 64)):
        at = room.as_strided((20, 64), strides)
        at.copy_(y)
        _near(ops.lora_add_(at, *rest, rows, starts, scale.to(cuda_dev)).cpu(), y, x, a, b, which, scale)
