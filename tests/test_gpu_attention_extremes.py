"""Attention whose logits are as large as its types allow: finite in fp32, and with one key far above the others the answer is its value.

Bound: with a weight of 1 - 2^-30 or more for one key the output is its value, but for the roundings of that weight and of the output
to 16 bits, 2 u of the largest |v| (the rows of other keys, nearer to one another than fp32 can tell such logits apart, are left out).
"""

import pytest
import torch

from fms_model_optimizer_b200 import ops

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _check(got, q, k, v, scale, first, dtype, what):
    """got, q [n, heads, d] from position `first` on, k and v [m, d]."""
    x = torch.einsum("ihd,jd->ihj", q.double(), k.double()) * scale
    pos = first + torch.arange(q.shape[0], device=q.device)[:, None, None]
    x = x.masked_fill(torch.arange(k.shape[0], device=q.device) > pos, -torch.inf)
    two = x.topk(min(2, x.shape[-1]), -1).values
    size = torch.einsum("ihd,jd->ihj", q.double().abs(), k.double().abs()).amax(-1) * scale
    clear = two[..., 0] - two[..., -1] > 2 * (q.shape[-1] + 16) * 2.0**-23 * size + 25 if x.shape[-1] > 1 else torch.ones_like(size, dtype=torch.bool)
    clear |= pos[..., 0] == 0
    assert float(clear.float().mean()) > 0.5, what
    err = (got.double() - v.double()[x.argmax(-1)]).abs().amax(-1)
    assert not got.isnan().any(), (what, int(got.isnan().sum()))
    assert float(err[clear].max()) <= 2 * U[dtype] * float(v.double().abs().max()), what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [30.0, 1e3, 1e4, 6e4, 1e6, 1e12, 1e18])
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("which", ["prompt", "token", "token, e4m3"])
def test_large_logits(cuda_dev, dtype, size, rising, which):
    if dtype == torch.float16 and size > 65504:
        pytest.skip("not an fp16 number")
    if rising and size == 30.0:
        pytest.skip("the first keys are as good as alike")
    g = torch.Generator(device=cuda_dev).manual_seed(41)
    for n, m, hq, hkv, dim in ((300, 300, 2, 1, 64), (70, 3000, 8, 1, 128)):  # the second shared by two blocks
        q = (torch.randn(n, hq, dim, generator=g, device=cuda_dev).sign() * size).to(dtype)
        k = ((torch.rand(m, hkv, dim, generator=g, device=cuda_dev) * 2 - 1) * size).to(dtype)
        if rising:  # the maximum grows from tile to tile, now by little, now by much
            k = (k.float() * torch.linspace(1e-6, 1, m, device=cuda_dev)[:, None, None] ** 2).to(dtype)
        v = torch.randn(m, hkv, dim, generator=g, device=cuda_dev).to(dtype)
        cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=cuda_dev) for x in (n, m))
        if which == "prompt":
            _check(ops.prompt_attention(q, k, v, cu_q, cu_k, n), q, k[:, 0], v[:, 0], dim**-0.5, m - n, dtype, which)
            continue
        pages, scales = [t.transpose(0, 1)[None].contiguous() for t in (k, v)], {}
        if which == "token, e4m3":
            pages = [(t.float() / t.float().abs().max() * 448).to(F8) for t in pages]
            scales = dict(k_scale=torch.ones(1, device=cuda_dev), v_scale=torch.ones(1, device=cuda_dev))
        table, lens = torch.zeros(1, 1, dtype=torch.int32, device=cuda_dev), torch.tensor([m], dtype=torch.int32, device=cuda_dev)
        token = ops.paged_attention(q[-1:], *pages, table, lens, **scales)
        _check(token, q[-1:], *(t[0, 0].float() for t in pages), dim**-0.5, m - 1, dtype, which)
    ops.check_status(cuda_dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [20, 700, 9000])
def test_an_infinite_value_of_small_weight(cuda_dev, dtype, n):
    """A value of infinity that is seen with a weight of 2^-58, too small for 16 bits: the output is infinite, not 0 * infinity."""
    g = torch.Generator(device=cuda_dev).manual_seed(42)
    dim = 64
    q, k, v = torch.zeros(1, 2, dim, device=cuda_dev), torch.zeros(n, 1, dim, device=cuda_dev), torch.randn(n, 1, dim, generator=g, device=cuda_dev)
    q[..., 0] = 8  # logits of the first element
    k[:, :, 0] = torch.rand(n, 1, generator=g, device=cuda_dev)
    at = n // 3
    k[at] = 0
    k[at, :, 0] = -40
    v[at, :, 3] = torch.inf
    q, k, v = (t.to(dtype) for t in (q, k, v))
    cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=cuda_dev) for x in (1, n))
    pages = [t.transpose(0, 1)[None].contiguous() for t in (k, v)]
    for got in (ops.prompt_attention(q, k, v, cu_q, cu_k, 1), ops.paged_attention(q, *pages, torch.zeros(1, 1, dtype=torch.int32, device=cuda_dev), cu_k[1:])):
        assert bool((got[..., 3] == torch.inf).all()) and int(got.isfinite().sum()) == 2 * (dim - 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e3, 6e4, 1e15])
@pytest.mark.parametrize("n,m,hq", [(300, 300, 2), (40, 3000, 8), (1500, 1500, 8)])
def test_keys_far_below_the_others_come_first(cuda_dev, dtype, size, n, m, hq):
    """Logits of -size^2 for the first keys and ordinary ones behind: those that see an ordinary key are as without the others."""
    if dtype == torch.float16 and size > 65504:
        pytest.skip("not an fp16 number")
    g = torch.Generator(device=cuda_dev).manual_seed(43)
    dim, low = 64, m - n + 2 * n // 3
    q, k, v = (torch.randn(rows, h, dim, generator=g, device=cuda_dev).to(dtype) for rows, h in ((n, hq), (m, 1), (m, 1)))
    q[..., 0] = size
    k[..., 0] = 0
    k[:low, :, 0] = -size
    cu = [torch.tensor([0, x], dtype=torch.int32, device=cuda_dev) for x in (n, m)]
    got = ops.prompt_attention(q, k, v, *cu, n)
    keep, part = low - (m - n), n - (low - (m - n))
    rest = ops.prompt_attention(q[keep:].contiguous(), k[low:].contiguous(), v[low:].contiguous(), *(torch.tensor([0, part], dtype=torch.int32, device=cuda_dev),) * 2, part)
    assert not got.isnan().any()
    # two ways of one row, each with weights and output in 16 bits
    assert float((got[keep:].float() - rest.float()).abs().max()) <= 4 * U[dtype] * float(v.float().abs().max())
    ops.check_status(cuda_dev)
