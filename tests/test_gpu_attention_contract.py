"""What the attention calls promise around their arithmetic: gradients refused, outputs that overlap inputs, caches without room."""

import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from fms_model_optimizer_b200 import _lib as L
from fms_model_optimizer_b200 import ops

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g).to(dtype)


class _Calls:
    """The three calls with every floating-point argument by name."""

    def __init__(self, dev, f8):
        g = torch.Generator().manual_seed(31)
        r = lambda *shape, dtype=torch.bfloat16: _randn(g, *shape, dtype=dtype).to(dev)  # noqa: E731
        self.i = torch.tensor([0, 1], dtype=torch.int32, device=dev)
        self.cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
        self.n = torch.tensor([3, 7], dtype=torch.int32, device=dev)
        pages = lambda: r(4, 2, 8, 64, dtype=torch.float32).to(F8 if f8 else torch.bfloat16)  # noqa: E731
        scales = dict(k_scale=torch.ones(2, device=dev), v_scale=torch.ones(2, device=dev)) if f8 else {}
        qkv = dict(q=r(2, 4, 64), k=r(2, 2, 64), v=r(2, 2, 64))
        self.args = {
            "rotate": dict(qkv, cos=r(4, 32, dtype=torch.float32), sin=r(4, 32, dtype=torch.float32), q_weight=r(64), k_weight=r(64), k_pages=pages(), v_pages=pages(), **scales),
            "token": dict(q=r(2, 4, 64), k_pages=pages(), v_pages=pages(), out=r(2, 4, 64), **scales),
            "prompt": dict(qkv, out=r(2, 4, 64)),
        }

    def __call__(self, which, **other):
        a = dict(self.args[which], **other)
        if which == "rotate":
            return ops.qk_norm_rope(a.pop("q"), a.pop("k"), a.pop("cos"), a.pop("sin"), self.i, slots=self.i.long(), **a)
        if which == "token":
            return ops.paged_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), self.i[:, None], self.n, **a)
        return ops.prompt_attention(a.pop("q"), a.pop("k"), a.pop("v"), self.cu, self.cu, 2, **a)


@pytest.mark.parametrize("which", ["rotate", "token", "prompt"])
@pytest.mark.parametrize("f8", [False, True])
def test_no_gradient_is_cut_off_silently(cuda_dev, which, f8):
    calls = _Calls(cuda_dev, f8)
    calls(which)
    for name, t in calls.args[which].items():
        if t.dtype != F8:  # no gradient reaches codes
            wanting = t.clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no gradient"):
                calls(which, **{name: wanting})
            with torch.no_grad():
                calls(which, **{name: wanting})
            with fwAD.dual_level(), torch.no_grad():  # tangents pass through no_grad
                dual = fwAD.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="no gradient"):
                    calls(which, **{name: dual})
    ops.check_status(cuda_dev)


@pytest.mark.parametrize("lens,dim", [([5000], 128), ([40, 2000, 7], 64)])
def test_an_output_may_lie_over_an_input(cuda_dev, lens, dim):
    """Queries, keys or values that the output takes the place of: the result is the one of an output of its own."""
    g = torch.Generator().manual_seed(32)
    hq, hkv, page = 16, 1, 16
    b, per = len(lens), -(-max(lens) // page)
    q = _randn(g, b, hq, dim).to(cuda_dev)
    pages = [_randn(g, b * per, hkv, page, dim).to(cuda_dev) for _ in range(2)]
    table, n = torch.arange(b * per, dtype=torch.int32, device=cuda_dev).view(b, per), torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    want = ops.paged_attention(q, *pages, table, n)
    own = torch.empty_like(q)
    assert ops.paged_attention(q, *pages, table, n, out=own) is own and torch.equal(own, want)
    for over in ("q", "k", "v"):
        mine, k, v = q.clone(), *(p.clone() for p in pages)
        out = dict(q=mine, k=k.view(-1)[: q.numel()].view(q.shape), v=v.view(-1)[-q.numel() :].view(q.shape))[over]
        got = ops.paged_attention(mine, k, v, table, n, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(got, want), over
    x = [_randn(g, 2000, 8, dim).to(cuda_dev) for _ in range(3)]
    cu = torch.tensor([0, 2000], dtype=torch.int32, device=cuda_dev)
    want = ops.prompt_attention(*x, cu, cu, 2000)
    for i in range(3):
        mine = [t.clone() for t in x]
        assert torch.equal(ops.prompt_attention(*mine, cu, cu, 2000, out=mine[i]), want), i
    x[2][100, 3, 5] = math.nan  # rows before the 100th are computed again from what they see
    want = ops.prompt_attention(*x, cu, cu, 2000)
    assert not want[:100].isnan().any()
    mine = [t.clone() for t in x]
    assert torch.equal(ops.prompt_attention(*mine, cu, cu, 2000, out=mine[0])[:100], want[:100])
    ops.check_status(cuda_dev)


def test_a_cache_without_pages_reports_every_slot(cuda_dev):
    calls = _Calls(cuda_dev, False)
    none = torch.empty(0, 2, 8, 64, dtype=torch.bfloat16, device=cuda_dev)
    ops.check_status(cuda_dev)
    a = dict(calls.args["rotate"], k_pages=none, v_pages=none)
    rotate = lambda slots: ops.qk_norm_rope(a["q"], a["k"], a["cos"], a["sin"], calls.i, q_weight=a["q_weight"], k_weight=a["k_weight"], v=a["v"], k_pages=none,  # noqa: E731
                                            v_pages=none, slots=torch.tensor(slots, device=cuda_dev))  # fmt: skip
    want = rotate([-1, -1])
    ops.check_status(cuda_dev)
    got = rotate([-1, 0])
    with pytest.raises(RuntimeError, match="status"):
        ops.check_status(cuda_dev)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_cache_whose_places_share_memory_is_refused(cuda_dev):
    """Keys and values in the same pages, or pages that are one and the same: what such a cache held would depend on timing."""
    calls = _Calls(cuda_dev, False)
    one = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16, device=cuda_dev)
    for k, v in ((one, one), (one[:1].expand(4, 2, 8, 64), one[1:2].expand(4, 2, 8, 64)), (one[:, :1].expand(4, 2, 8, 64), one[:, 1:].expand(4, 2, 8, 64))):
        with pytest.raises(RuntimeError, match="share memory"):
            calls("rotate", k_pages=k, v_pages=v)
    calls("token", k_pages=one, v_pages=one)  # reading them is no matter
    calls("token", k_pages=one[:1].expand(4, 2, 8, 64), v_pages=one[:1].expand(4, 2, 8, 64))
    assert not one.any()


@pytest.mark.parametrize("case", ["no sequences", "no queries a sequence", "keys that are not there", "offsets that fall"])
def test_offsets_that_do_not_cover_the_queries_are_reported(cuda_dev, case):
    """... also where there is nothing to compute: the C entry's status word, and outputs that hold no stale value as an answer."""
    x = torch.ones(4, 2, 64, dtype=torch.bfloat16, device=cuda_dev)
    out = torch.full_like(x, 3.0)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    none = case in ("keys that are not there", "offsets that fall")
    cu_q, cu_k = (torch.tensor(c, dtype=torch.int32, device=cuda_dev) for c in (([0, 4, 2] if case == "offsets that fall" else [0, 2, 4]), [0, 3, 3] if "keys" in case else [0, 0, 0]))
    a = L.PromptAttentionArgs(q=x.data_ptr(), k=x.data_ptr(), v=x.data_ptr(), out=out.data_ptr(), cu_q=cu_q.data_ptr(), cu_k=cu_k.data_ptr(), status=status.data_ptr(),
                              q_token=128, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, tokens_q=4, tokens_k=0 if none else 4,
                              batch=0 if case == "no sequences" else 2, max_q=0 if case == "no queries a sequence" else 2, q_heads=2, kv_heads=2, head_dim=64,
                              dtype=L.DT_BF16, scale=0.125)  # fmt: skip
    stream = C.c_void_p(torch.cuda.current_stream(cuda_dev).cuda_stream)
    assert L.load().qlin_prompt_attention(C.byref(a), stream) == L.OK
    assert int(status) == L.ERR_BAD_SHAPE
    if none:  # the call through tensors reports it as well
        ops.check_status(cuda_dev)
        ops.prompt_attention(x, x[:0], x[:0], cu_q, cu_k, 2)
        with pytest.raises(RuntimeError, match="status"):
            ops.check_status(cuda_dev)
        good = torch.tensor([0, 2, 4], dtype=torch.int32, device=cuda_dev)
        assert not ops.prompt_attention(x, x[:0], x[:0], good, torch.zeros_like(good), 2).any()
        ops.check_status(cuda_dev)
    else:
        assert bool((out == 3.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries_whose_logits_are_all_minus_infinity_give_zeros(cuda_dev, dtype, value):
    """... whatever the values hold that they see with a weight of zero: in one block, in blocks that join, and in a second launch."""
    dim = 64
    minus = lambda *shape: torch.full(shape, -math.inf, dtype=dtype, device=cuda_dev)  # noqa: E731
    for n, hq, hkv in ((40, 2, 1), (300, 4, 2), (2000, 8, 1)):  # the last shared by two blocks
        q, k = torch.ones(n, hq, dim, dtype=dtype, device=cuda_dev), torch.ones(n, hkv, dim, dtype=dtype, device=cuda_dev)
        q[::2] = -math.inf
        v = torch.zeros(n, hkv, dim, dtype=dtype, device=cuda_dev)
        v[n // 3 :, :, 5] = value
        cu = torch.tensor([0, n], dtype=torch.int32, device=cuda_dev)
        got = ops.prompt_attention(q, k, v, cu, cu, n)
        assert not got[::2].any(), (n, "rows of minus infinity")
        assert not got[: n // 3].any() and bool((got[1::2][n // 6 + 1 :, :, 5].isnan() if math.isnan(value) else got[1::2][n // 6 + 1 :, :, 5] == value).all())
    for lens, page, f8 in (([3], 4, False), ([700, 2, 90], 16, False), ([9000], 64, False), ([500, 0], 16, True), ([9000], 64, True)):
        if f8 and math.isinf(value):
            continue  # e4m3 has no infinities
        per = -(-max(lens) // page)
        shape = (len(lens) * per, 1, page, dim)
        k, v = torch.ones(shape, dtype=dtype, device=cuda_dev), torch.zeros(shape, dtype=dtype, device=cuda_dev)
        v[..., 5] = value
        one = torch.ones(1, device=cuda_dev) if f8 else None
        if f8:
            k, v = k.to(F8), v.to(F8)
        table = torch.arange(len(lens) * per, dtype=torch.int32, device=cuda_dev).view(len(lens), per)
        n = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
        q = minus(len(lens), 2, dim)
        q[:, 1] = 1
        got = ops.paged_attention(q, k, v, table, n, k_scale=one, v_scale=one)
        assert not got[:, 0].any(), (lens, f8)
        seen = got[:, 1, 5][n > 0]
        assert bool((seen.isnan() if math.isnan(value) else seen == value).all())
    ops.check_status(cuda_dev)
