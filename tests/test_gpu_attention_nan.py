"""NaN and infinities among the values of prompts: a query that sees one has it in its output, one that does not is as without it, and
neither makes the call slow or ends it.

Rows that see none of them: the tile's product may carry 0 * NaN, so they are computed a second time, in fp32 throughout, which moves
them by the roundings of the first one: weights and output to 16 bits, 2 u of the largest |v|, on either side, hence 4 u.
"""

import math

import pytest
import torch

from fms_model_optimizer_b200 import ops

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _prompt(dev, seed, n, m, hq, hkv, dim, dtype, batch=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(batch * n, hq, dim, generator=g, device=dev).to(dtype)
    k, v = (torch.randn(batch * m, hkv, dim, generator=g, device=dev).to(dtype) for _ in range(2))
    cu = [torch.arange(0, batch * x + 1, x, dtype=torch.int32, device=dev) for x in (n, m)]
    return q, k, v, *cu, n


def _seen(n, m, window, sinks, dev):
    i, j = torch.arange(n, device=dev)[:, None] + m - n, torch.arange(m, device=dev)[None]
    seen = j <= i
    return seen & ((j > i - window) | (j < sinks)) if window else seen


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,m,hq,hkv,dim,window,sinks", [(300, 300, 4, 2, 128, 0, 0), (300, 300, 4, 2, 64, 50, 2), (40, 3000, 8, 1, 128, 0, 0), (2000, 2000, 8, 1, 96, 0, 0),
                                                         (2000, 2000, 8, 1, 64, 1300, 140), (700, 1500, 5, 1, 40, 200, 130), (513, 513, 12, 12, 128, 0, 0)])  # fmt: skip
def test_values_that_are_not_finite(cuda_dev, dtype, n, m, hq, hkv, dim, window, sinks):
    q, k, v, cu_q, cu_k, most = _prompt(cuda_dev, n + dim, n, m, hq, hkv, dim, dtype)
    run = lambda v: ops.prompt_attention(q, k, v, cu_q, cu_k, most, window=window, sinks=sinks)  # noqa: E731
    clean = run(v).float()
    seen = _seen(n, m, window, sinks, cuda_dev)
    # (key, head dimension, value), first of one kind each, then all of them
    places = [(0, 3, math.nan), (m // 2 + 1, 0, math.inf), (m - n // 3, dim - 1, math.nan), (m - 1, 5, -math.inf), (m - 2, 7, math.nan), (m // 3, 9, math.inf),
              (m - n // 2, 9, -math.inf), (130 if m > 130 else 7, dim - 2, math.inf)]  # fmt: skip
    for some in [[p] for p in places] + [places]:
        bad = v.clone()
        for j, d, x in some:
            bad[j, :, d] = x
        got = run(bad).float()
        total = torch.zeros(n, dim, device=cuda_dev)  # what a row's visible values that are not finite add up to
        for j, d, x in some:
            total[:, d] += torch.where(seen[:, j], x, 0.0)
        want_nan = total.isnan()[:, None].expand_as(got)
        plus, minus = ((total == x)[:, None].expand_as(got) for x in (math.inf, -math.inf))
        assert torch.equal(got.isnan(), want_nan), some
        assert bool((got[plus] == math.inf).all()) and bool((got[minus] == -math.inf).all()), some
        rest = ~(want_nan | plus | minus)
        assert float((got - clean)[rest].abs().max()) <= 4 * U[dtype] * float(v.abs().max()), some
    ops.check_status(cuda_dev)


def _time(run):
    run()
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(3):
        run()
    end.record()
    torch.cuda.synchronize()
    return begin.elapsed_time(end) / 3


@pytest.mark.parametrize("key", [0, 700, 2040])
@pytest.mark.parametrize("columns", [1, 128])
def test_a_visible_nan_does_not_make_the_call_slow(cuda_dev, key, columns):
    """Rows that see a NaN value have their answer.  To know it they read values again, no more than a fraction of the work of their
    logits: ten times the time without is far above that, and far below a second computation of the rows by themselves."""
    q, k, v, cu_q, cu_k, most = _prompt(cuda_dev, 5, 2048, 2048, 32, 8, 128, torch.bfloat16, batch=4)
    bad = v.clone()
    bad[key::2048, :, :columns] = math.nan
    run = lambda v: lambda: ops.prompt_attention(q, k, v, cu_q, cu_k, most)  # noqa: E731
    got = run(bad)().view(4, 2048, 32, 128)
    assert got[:, key:, :, :columns].isnan().all() and not got[:, :key].isnan().any() and not got[..., columns:].isnan().any()
    clean, slow = _time(run(v)), _time(run(bad))
    assert slow < 10 * clean, (clean, slow)
    ops.check_status(cuda_dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,m,hq,hkv,dim,window,sinks", [(300, 700, 8, 2, 128, 0, 0), (300, 700, 6, 1, 8, 90, 40), (2000, 2000, 8, 1, 72, 500, 1), (130, 130, 128, 1, 64, 0, 0)])
def test_keys_queries_and_values_that_are_nan(cuda_dev, dtype, n, m, hq, hkv, dim, window, sinks):
    """A NaN in a key that a row sees, or in its query, is a row of NaN; beside NaN among the values each row has what it sees."""
    q, k, v, cu_q, cu_k, most = _prompt(cuda_dev, n + dim, n, m, hq, hkv, dim, dtype)
    run = lambda q, k, v: ops.prompt_attention(q, k, v, cu_q, cu_k, most, window=window, sinks=sinks).float()  # noqa: E731
    clean = run(q, k, v)
    seen = _seen(n, m, window, sinks, cuda_dev)
    bad_keys, bad_rows, bad_values = [m - n // 2, m - 3], [n // 4], [(m - n + n // 3, 1), (m - n + 1, 0), (m - 2, 5)]
    q, k, v = q.clone(), k.clone(), v.clone()
    q[bad_rows, :, 0] = math.nan
    k[bad_keys, :, dim - 1] = math.nan
    want = torch.zeros(n, dim, dtype=torch.bool, device=cuda_dev)
    want[bad_rows] = True
    for j in bad_keys:
        want |= seen[:, j, None]
    for j, d in bad_values:
        v[j, :, d] = math.nan
        want[:, d] |= seen[:, j]
    got = run(q, k, v)
    want = want[:, None].expand_as(got)
    assert torch.equal(got.isnan(), want)
    assert float((got - clean)[~want].abs().max()) <= 4 * U[dtype] * float(clean.abs().max().clamp(min=float(v[~v.isnan()].abs().max())))
    ops.check_status(cuda_dev)
