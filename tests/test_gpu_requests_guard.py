"""Stray stores of the operators that answer many requests at once: every output, workspaces included, between guard bands of poison."""

import ctypes as C

import pytest
import torch

from fms_model_optimizer_b200 import _lib as L
from fms_model_optimizer_b200 import ops
from test_gpu_guard import Guarded

pytestmark = pytest.mark.gpu

DT = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16, torch.float32: L.DT_F32, torch.float8_e4m3fn: L.DT_F8E4M3}


def _stream(dev):
    return C.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top,pitch", [(1, 1, 1, 1), (3, 4099, 32, 4099), (2, 50257, 7, 50261), (500, 1031, 5, 1040), (1, 128256, 20, 128256)])
def test_log_probabilities_stay_inside_their_outputs(cuda_dev, dtype, rows, vocab, top, pitch):
    g = torch.Generator(device=cuda_dev).manual_seed(vocab)
    x = torch.randn(rows * pitch + 3, generator=g, device=cuda_dev).to(dtype)[3:].as_strided((rows, vocab), (pitch, 1))  # a row that begins anywhere
    tokens = torch.randint(-1, vocab, (rows,), generator=g, device=cuda_dev)
    outs = dict(logprobs=Guarded(rows, 1, torch.float32, cuda_dev), entropy=Guarded(rows, 1, torch.float32, cuda_dev), stats=Guarded(rows, 2, torch.float32, cuda_dev),
                top_logprobs=Guarded(rows, top, torch.float32, cuda_dev), top_ids=Guarded(rows, 2 * top, torch.int32, cuda_dev), d_logits=Guarded(rows, vocab, dtype, cuda_dev))  # fmt: skip
    ones = torch.ones(rows, device=cuda_dev)
    a = L.TokenLogprobsArgs(logits=x.data_ptr(), tokens=tokens.data_ptr(), ld=pitch, rows=rows, vocab=vocab, top=top, dtype=DT[dtype], d_logprobs=ones.data_ptr(),
                            d_entropy=ones.data_ptr(), **{n: o.t.data_ptr() for n, o in outs.items()})  # fmt: skip
    for fn in ("qlin_token_logprobs", "qlin_token_logprobs_bwd"):
        L.check(getattr(L.load(), fn)(C.byref(a), _stream(cuda_dev)), fn)
    torch.cuda.synchronize()
    for name, o in outs.items():
        o.check(name)
    lp, entropy, top_lp, ids = ops.token_logprobs(x, tokens, top=top)
    assert torch.equal(outs["logprobs"].t.reshape(-1), lp) and torch.equal(outs["entropy"].t.reshape(-1), entropy)
    assert torch.equal(outs["top_logprobs"].t, top_lp) and torch.equal(outs["top_ids"].t.contiguous().view(torch.int64), ids)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,adapters,rank,width,out", [(1, 1, 8, 8, 8), (37, 3, 16, 264, 72), (40, 2, 64, 520, 1000), (33, 2, 128, 136, 40), (5000, 2, 24, 72, 264), (700, 2, 120, 64, 520)])
def test_adapters_stay_inside_their_rows(cuda_dev, dtype, tokens, adapters, rank, width, out):
    g = torch.Generator(device=cuda_dev).manual_seed(tokens)
    x = torch.randn(tokens, width, generator=g, device=cuda_dev).to(dtype)
    a, b = (torch.randn(shape, generator=g, device=cuda_dev).to(dtype) for shape in ((adapters, rank, width), (adapters, out, rank)))
    rows, starts = ops.lora_groups(torch.randint(-1, adapters, (tokens,), generator=g, device=cuda_dev), adapters)
    y = Guarded(tokens, out, dtype, cuda_dev, pitch=out + 24)
    before = torch.randn(tokens, out, generator=g, device=cuda_dev).to(dtype)
    y.t.copy_(before)
    got = ops.lora_add_(y.t, x, a, b, rows, starts, torch.ones(adapters, device=cuda_dev))
    torch.cuda.synchronize()
    y.check("y")
    assert got.data_ptr() == y.t.data_ptr() and torch.equal(got, ops.lora_add_(before, x, a, b, rows, starts, torch.ones(adapters, device=cuda_dev)))


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("each,groups,prefix,own", [(3, 2, 70, 20), (20, 1, 1000, 9), (40, 1, 1500, 40), (40, 3, 300, 3), (2, 1, 64, 9000)])
def test_prefix_attention_stays_inside_its_output_and_workspace(cuda_dev, f8, dim, each, groups, prefix, own):
    g = torch.Generator(device=cuda_dev).manual_seed(dim + each)
    dtype, ct, page, hq, hkv = torch.bfloat16, torch.float8_e4m3fn if f8 else torch.bfloat16, 16, 8, 2
    batch, pp, per = each * groups, -(-prefix // page), -(-(prefix + own) // page)
    k, v = (torch.randn(200, hkv, page, dim, generator=g, device=cuda_dev).to(ct) for _ in range(2))
    q = torch.randn(batch, hq, dim, generator=g, device=cuda_dev).to(dtype)
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    ptable, table = (i32(torch.randint(0, 200, shape, generator=g, device=cuda_dev)) for shape in ((groups, pp), (batch, per)))
    plens = torch.full((groups,), prefix, dtype=torch.int32, device=cuda_dev)
    lens = i32(prefix + torch.randint(1, own + 1, (batch,), generator=g, device=cuda_dev))
    at = i32(torch.arange(groups + 1, device=cuda_dev) * each)
    scale = torch.ones(hkv, device=cuda_dev)
    out = Guarded(batch, hq * dim, dtype, cuda_dev)
    a = L.PrefixAttentionArgs(
        own=L.PagedAttentionArgs(q=q.data_ptr(), k_pages=k.data_ptr(), v_pages=v.data_ptr(), block_table=table.data_ptr(), lens=lens.data_ptr(), k_scale=scale.data_ptr(),
                                 v_scale=scale.data_ptr(), out=out.t.data_ptr(), q_batch=hq * dim, q_head=dim, page_stride=hkv * page * dim, head_stride=page * dim, slot_stride=dim,
                                 table_stride=per, batch=batch, q_heads=hq, kv_heads=hkv, head_dim=dim, page_size=page, num_pages=200, max_pages=per, dtype=DT[dtype], cache_dtype=DT[ct],
                                 scale=dim**-0.5),
        prefix_table=ptable.data_ptr(), prefix_lens=plens.data_ptr(), groups=at.data_ptr(), prefix_stride=pp, num_groups=groups, max_prefix_pages=pp)  # fmt: skip
    need = L.load().qlin_prefix_attention_workspace_bytes(C.byref(a))
    assert need > 0
    work = Guarded(1, need, torch.uint8, cuda_dev)
    a.own.workspace = work.t.data_ptr()
    L.check(L.load().qlin_prefix_attention(C.byref(a), _stream(cuda_dev)), "qlin_prefix_attention")
    torch.cuda.synchronize()
    out.check("out")
    work.check("workspace")
    scales = dict(k_scale=scale, v_scale=scale) if f8 else {}
    assert torch.equal(out.t.reshape(batch, hq, dim), ops.prefix_attention(q, k, v, ptable, plens, at, table, lens, **scales))
