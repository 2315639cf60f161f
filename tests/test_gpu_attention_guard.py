"""Stray stores of the generating decoder's kernels: every output and cache between guard bands of poison, rows that nothing writes included."""

import ctypes as C

import pytest
import torch

from fms_model_optimizer_b200 import _lib as L
from fms_model_optimizer_b200 import ops
from oracle import attention as OA
from test_gpu_guard import POISON, Guarded

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DT = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16, torch.float32: L.DT_F32, F8: L.DT_F8E4M3}


def _randn(g, dev, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=dev).to(dtype)


def _poisoned(t):
    return (t.contiguous().view(torch.uint8) == POISON).all()


@pytest.mark.parametrize("dim,rotary", [(16, 16), (48, 32), (80, 80), (96, 48), (128, 128), (512, 512)])
@pytest.mark.parametrize("dtype,f8", [(torch.bfloat16, True), (torch.float16, False), (torch.float32, False)])
@pytest.mark.parametrize("tokens", [3, 1401])  # a block of four warps a token, a warp a token
def test_rotation_stays_inside_its_outputs(cuda_dev, dim, rotary, dtype, f8, tokens):
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    hq, hkv, page = 5, 2, 7
    pages = -(-tokens // page) + 1
    ct = F8 if f8 else dtype
    q, k, v = (_randn(g, cuda_dev, tokens, h, dim, dtype=dtype) for h in (hq, hkv, hkv))
    cos, sin = (_randn(g, cuda_dev, 9, rotary // 2, dtype=torch.float32) for _ in range(2))
    pos = torch.randint(0, 9, (tokens,), generator=g, device=cuda_dev, dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=g, device=cuda_dev)[:tokens]
    scale = torch.full((hkv,), 0.5, device=cuda_dev)
    outs = [Guarded(tokens, h * dim, dtype, cuda_dev) for h in (hq, hkv)]
    caches = [Guarded(pages * hkv * page, dim, ct, cuda_dev, pitch=dim + 16) for _ in range(2)]  # rows with room behind them
    row = dim + 16
    a = L.QkRopeArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=outs[0].t.data_ptr(), k_out=outs[1].t.data_ptr(), cos=cos.data_ptr(), sin=sin.data_ptr(),
                     positions=pos.data_ptr(), k_pages=caches[0].t.data_ptr(), v_pages=caches[1].t.data_ptr(), slots=slots.data_ptr(), k_scale=scale.data_ptr(),
                     v_scale=scale.data_ptr(), q_token=hq * dim, q_head=dim, k_token=hkv * dim, k_head=dim, v_token=hkv * dim, v_head=dim, page_stride=hkv * page * row,
                     head_stride=page * row, slot_stride=row, num_slots=pages * page, tokens=tokens, q_heads=hq, kv_heads=hkv, head_dim=dim, rotary=rotary, table_rows=9,
                     page_size=page, dtype=DT[dtype], weight_dtype=DT[dtype], cache_dtype=DT[ct], eps=1e-6)  # fmt: skip
    L.check(L.load().qlin_qk_rope(C.byref(a), C.c_void_p(torch.cuda.current_stream(cuda_dev).cuda_stream)), "qlin_qk_rope")
    torch.cuda.synchronize()
    for t, what in zip(outs + caches, ("q", "k", "k_pages", "v_pages")):
        t.check(what)
    pool = [torch.zeros(pages, hkv, page, dim, device=cuda_dev).to(ct) for _ in range(2)]
    scales = dict(k_scale=scale, v_scale=scale) if f8 else {}
    want = ops.qk_norm_rope(q, k, cos, sin, pos, v=v, k_pages=pool[0], v_pages=pool[1], slots=slots, **scales)
    assert all(torch.equal(o.t.reshape(w.shape), w) for o, w in zip(outs, want))
    free = torch.ones(pages * page, dtype=torch.bool, device=cuda_dev)
    free[slots] = False
    for got, p in zip(caches, pool):
        got = got.t.view(torch.uint8 if f8 else dtype).reshape(pages, hkv, page, dim).transpose(1, 2).reshape(pages * page, hkv, dim)
        p = p.view(torch.uint8 if f8 else dtype).transpose(1, 2).reshape(pages * page, hkv, dim)
        assert torch.equal(got[slots], p[slots]) and _poisoned(got[free])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 40, 72, 96, 128])
@pytest.mark.parametrize("lens,hq,hkv", [([(1, 1), (130, 130), (7, 300)], 6, 2), ([(900, 1500)], 5, 1), ([(64, 64)] * 40, 8, 8)])
def test_prompt_attention_stays_inside_its_output(cuda_dev, dtype, dim, lens, hq, hkv):
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    nq, nk = sum(n for n, _ in lens), sum(m for _, m in lens)
    q, k, v = (_randn(g, cuda_dev, n, h, dim, dtype=dtype) for n, h in ((nq, hq), (nk, hkv), (nk, hkv)))
    cu = [torch.tensor([0] + torch.tensor(x).cumsum(0).tolist(), dtype=torch.int32, device=cuda_dev) for x in ([n for n, _ in lens], [m for _, m in lens])]
    most = max(n for n, _ in lens)
    out = Guarded(nq, hq * dim, dtype, cuda_dev)
    ops.prompt_attention(q, k, v, *cu, most, out=out.t.view(nq, hq, dim))
    torch.cuda.synchronize()
    ops.check_status(cuda_dev)
    out.check("out")
    assert torch.equal(out.t.view(nq, hq, dim), ops.prompt_attention(q, k, v, *cu, most))


@pytest.mark.parametrize("dtype,f8", [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("dim", [8, 16, 48, 80, 128])
@pytest.mark.parametrize("lens,hq,hkv", [([1, 0, 300], 6, 2), ([5000], 5, 1), ([90] * 80, 24, 1), ([40000], 8, 1)])
def test_paged_attention_stays_inside_its_output(cuda_dev, dtype, f8, dim, lens, hq, hkv):
    """... and its workspace, whose size the C interface names."""
    if f8 and dim % 16:
        pytest.skip("e4m3 rows are multiples of 16")
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    page = 24
    per = -(-max(lens) // page)
    b = len(lens)
    q = _randn(g, cuda_dev, b, hq, dim, dtype=dtype)
    k, v = (_randn(g, cuda_dev, b * per, hkv, page, dim, dtype=torch.float32).to(F8 if f8 else dtype) for _ in range(2))
    table, n = torch.arange(b * per, dtype=torch.int32, device=cuda_dev).view(b, per), torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    one = torch.ones(hkv, device=cuda_dev)
    out = Guarded(b, hq * dim, dtype, cuda_dev)
    a = L.PagedAttentionArgs(q=q.data_ptr(), k_pages=k.data_ptr(), v_pages=v.data_ptr(), block_table=table.data_ptr(), lens=n.data_ptr(), k_scale=one.data_ptr(),
                             v_scale=one.data_ptr(), out=out.t.data_ptr(), q_batch=hq * dim, q_head=dim, page_stride=hkv * page * dim, head_stride=page * dim,
                             slot_stride=dim, table_stride=per, batch=b, q_heads=hq, kv_heads=hkv, head_dim=dim, page_size=page, num_pages=b * per, max_pages=per,
                             dtype=DT[dtype], cache_dtype=DT[k.dtype], scale=dim**-0.5)  # fmt: skip
    lib = L.load()
    work = Guarded(1, max(16, lib.qlin_paged_attention_workspace_bytes(C.byref(a))), torch.uint8, cuda_dev)
    a.workspace = work.t.data_ptr()
    L.check(lib.qlin_paged_attention(C.byref(a), C.c_void_p(torch.cuda.current_stream(cuda_dev).cuda_stream)), "qlin_paged_attention")
    torch.cuda.synchronize()
    out.check("out")
    work.check("workspace")
    scales = dict(k_scale=one, v_scale=one) if f8 else {}
    assert torch.equal(out.t.view(b, hq, dim), ops.paged_attention(q, k, v, table, n, **scales))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rotary,norm,f8", [(1500, 32, 8, 128, 128, True, True), (1332, 12, 12, 64, 32, False, False), (2401, 5, 1, 96, 48, True, False),
                                                              (1400, 2, 2, 512, 256, True, False), (1333, 3, 1, 16, 16, False, True)])  # fmt: skip
def test_rotation_of_prompts(cuda_dev, dtype, tokens, hq, hkv, dim, rotary, norm, f8):
    """As many tokens as take a warp each: against 64 bits, and bit for bit what the form for few tokens gives."""
    g = torch.Generator(device=cuda_dev).manual_seed(tokens)
    q, k, v = (_randn(g, cuda_dev, tokens, h, dim, dtype=torch.float32).mul(3).to(dtype) for h in (hq, hkv, hkv))
    wq, wk = ((1 + 0.2 * _randn(g, cuda_dev, dim, dtype=torch.float32)).to(dtype) if norm else None for _ in range(2))
    ang = torch.outer(torch.arange(300.0, device=cuda_dev), 10000.0 ** (-torch.arange(0, rotary, 2, device=cuda_dev) / rotary))
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, 300, (tokens,), generator=g, device=cuda_dev, dtype=torch.int32)
    page, pages = 16, -(-tokens // 16) + 2
    slots = torch.randperm(pages * page, generator=g, device=cuda_dev)[:tokens]
    scales = dict(k_scale=torch.full((hkv,), 0.03, device=cuda_dev), v_scale=torch.full((hkv,), 0.04, device=cuda_dev)) if f8 else {}
    pools = [[torch.zeros(pages, hkv, page, dim, device=cuda_dev).to(F8 if f8 else dtype) for _ in range(2)] for _ in range(2)]

    def run(part, pool):
        return ops.qk_norm_rope(q[part], k[part], cos, sin, pos[part], q_weight=wq, k_weight=wk, eps=1e-5, v=v[part], k_pages=pool[0], v_pages=pool[1], slots=slots[part], **scales)

    got = run(slice(0, tokens), pools[0])
    parts = [run(slice(i, i + 500), pools[1]) for i in range(0, tokens, 500)]
    ops.check_status(cuda_dev)
    assert all(torch.equal(x, torch.cat(y)) for x, y in zip(got, zip(*parts)))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(*pools))
    u = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}[dtype]
    for x, w, z in ((q, wq, got[0]), (k, wk, got[1])):
        y, want = OA.norm_rope(x, w, 1e-5, cos[pos.long()], sin[pos.long()])
        near = y.abs()
        half = rotary // 2
        near[..., :rotary] = torch.cat([near[..., :half] + near[..., half:rotary]] * 2, -1)
        # fp32 arithmetic of a few dozen roundings, then one rounding, fp16 with subnormal numbers
        tol = u * want.abs() + (2.0**-25 if dtype == torch.float16 else 0.0) + 2.0**-18 * near
        assert bool(((z.double() - want).abs() <= tol).all())
