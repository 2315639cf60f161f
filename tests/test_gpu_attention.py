"""Rotation into a paged cache, attention of prompts and attention of one token over pages, against 64 bits.

Bounds (u: unit roundoff of the 16-bit type, 2^-8 bf16, 2^-11 fp16).  Attention: the weights are rounded to 16 bits as operands
(u * sum w|v|), the output once (u * |o| <= u * sum w|v|), a logit is an fp32 sum of head_dim products, (head_dim + 16) 2^-23 of
sum |q k| scale off at most, which moves a weight by as much; fp16 weights below the normal range lose up to 2^-30 of the largest
each, and an fp16 output is 2^-25 off where it is subnormal.  Rotation: fp32 arithmetic of a few dozen roundings, 2^-18 of the two
rotated elements, and the output's rounding (half of its type's spacing there).  e4m3: half
a step, 2^-4 of the value or 2^-10 of the scale.
"""

import math

import pytest
import torch

from fms_model_optimizer_b200 import ops
from oracle import attention as OA

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
F8 = torch.float8_e4m3fn


def _half_step(want, dtype):
    """Half of the spacing of the type at |want|, its subnormal numbers included: what one rounding may be off."""
    exponent = torch.frexp(want.abs())[1].clamp(min={torch.float16: -13, torch.bfloat16: -125, torch.float32: -125}[dtype])
    return torch.ldexp(torch.full_like(want, U[dtype]), exponent - 1)



def _randn(g, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(dtype)


# ---------------------------------------------------------------------------------------------------- rotation and cache write
def _tables(n, rotary):
    ang = torch.outer(torch.arange(n).float(), 10000.0 ** (-torch.arange(0, rotary, 2).float() / rotary))
    return ang.cos(), ang.sin()


def _rope_close(got, x, weight, eps, cos, sin, dtype):
    y, want = OA.norm_rope(x, weight, eps, cos, sin)
    r = cos.shape[1]
    near = y.abs()
    near[..., : 2 * r] = torch.cat([y[..., :r].abs() + y[..., r : 2 * r].abs()] * 2, -1)
    err = (got.double() - want).abs()
    assert bool((err <= _half_step(want, dtype) + 2.0**-18 * near).all()), float((err - _half_step(want, dtype)).max())
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rotary,page,norm,f8", [
    (1, 32, 8, 128, 128, 16, True, False), (37, 32, 8, 128, 128, 16, True, True), (5, 12, 12, 64, 32, 24, False, False), (130, 7, 1, 96, 48, 7, True, True),
    (3, 2, 2, 16, 16, 1, True, False), (9, 3, 3, 256, 128, 64, True, True), (4, 1, 1, 512, 512, 5, True, False), (6, 5, 5, 80, 80, 3, False, True)])  # fmt: skip
def test_rotation_and_cache_write(cuda_dev, dtype, tokens, hq, hkv, dim, rotary, page, norm, f8):
    g = torch.Generator().manual_seed(tokens * 131 + dim)
    qkv = _randn(g, tokens, (hq + 2 * hkv) * dim, dtype=dtype, std=3.0)
    q, k, v = (t.view(tokens, -1, dim) for t in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
    dq, dk, dv = (t.view(tokens, -1, dim) for t in qkv.to(cuda_dev).split([hq * dim, hkv * dim, hkv * dim], 1))  # views with a pitch
    wq, wk = (_randn(g, dim, dtype=dtype, std=0.2) + 1 if norm else None for _ in range(2))
    cos, sin = _tables(200, rotary)
    pos = torch.randint(0, 200, (tokens,), generator=g, dtype=torch.int32)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[tokens // 2] = -1 if tokens > 2 else slots[tokens // 2]
    ct = F8 if f8 else dtype
    kp, vp = (_randn(g, pages, hkv, page, dim, dtype=torch.float32).to(ct) for _ in range(2))
    ks, vs = (torch.rand(hkv, generator=g) * 0.05 + 0.01 if f8 else None for _ in range(2))
    dev = lambda t: None if t is None else t.to(cuda_dev)  # noqa: E731
    dkp, dvp = dev(kp), dev(vp)
    got_q, got_k = ops.qk_norm_rope(dq, dk, dev(cos), dev(sin), dev(pos), q_weight=dev(wq), k_weight=dev(wk), eps=1e-5, v=dv, k_pages=dkp, v_pages=dvp, slots=dev(slots),
                                    k_scale=dev(ks), v_scale=dev(vs))  # fmt: skip
    ops.check_status(cuda_dev)
    c, s = cos[pos.long()], sin[pos.long()]
    _rope_close(got_q.cpu(), q, wq, 1e-5, c, s, dtype)
    zk = _rope_close(got_k.cpu(), k, wk, 1e-5, c, s, dtype)
    for got, before, want, exact, scale in ((dkp, kp, zk, got_k.cpu(), ks), (dvp, vp, v.double(), v, vs)):
        flat = got.cpu().float().transpose(1, 2).reshape(pages * page, hkv, dim)
        old = before.float().transpose(1, 2).reshape(pages * page, hkv, dim)
        used = slots[slots >= 0]
        rest = torch.ones(pages * page, dtype=torch.bool)
        rest[used] = False
        assert torch.equal(flat[rest], old[rest]), "slots that no token has were written"
        rows = flat[used]
        if f8:
            x = (want[slots >= 0] / scale.double()[:, None]).clamp(-448, 448)
            assert bool(((rows.double() - x).abs() <= 2.0**-4 * x.abs() * (1 + 2.0**-10) + 2.0**-10 + 2.0**-16 * x.abs().amax()).all())
        else:
            assert torch.equal(rows, exact[slots >= 0].float()), "the cache does not hold what is returned"


def test_rotation_without_cache_and_weights_in_fp32(cuda_dev):
    g = torch.Generator().manual_seed(3)
    q, k = _randn(g, 11, 4, 128), _randn(g, 11, 2, 128)
    wq = torch.randn(128, generator=g)
    cos, sin = _tables(32, 64)
    pos = torch.arange(11, dtype=torch.int32)
    got, none = ops.qk_norm_rope(q.to(cuda_dev), k.to(cuda_dev), cos.to(cuda_dev), sin.to(cuda_dev), pos.to(cuda_dev), q_weight=wq.to(cuda_dev), want_k=False)
    assert none is None
    _rope_close(got.cpu(), q, wq, 1e-6, cos[:11], sin[:11], torch.bfloat16)


def test_rotation_flags_positions_and_slots_out_of_range(cuda_dev):
    g = torch.Generator().manual_seed(4)
    q, k = _randn(g, 4, 4, 64).to(cuda_dev), _randn(g, 4, 2, 64).to(cuda_dev)
    cos, sin = (t.to(cuda_dev) for t in _tables(16, 64))
    pages = [torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2)]
    run = lambda pos, slots: ops.qk_norm_rope(q, k, cos, sin, torch.tensor(pos, dtype=torch.int32, device=cuda_dev), v=k, k_pages=pages[0], v_pages=pages[1],  # noqa: E731
                                              slots=torch.tensor(slots, device=cuda_dev))  # fmt: skip
    ops.check_status(cuda_dev)
    got, _ = run([0, 16, 1, -1], [0, 1, 2, 3])
    with pytest.raises(RuntimeError, match="status"):
        ops.check_status(cuda_dev)
    bad = got.isnan().flatten(1).all(1).tolist()
    assert bad == [False, True, False, True] and not got[[0, 2]].isnan().any()
    assert pages[1][0, 0].abs().sum(-1).ne(0).tolist() == [True, False, True, False]
    run([0, 1, 2, 3], [0, 1, 2, 8])
    with pytest.raises(RuntimeError, match="status"):
        ops.check_status(cuda_dev)
    empty, _ = ops.qk_norm_rope(q[:0], k[:0], cos, sin, torch.zeros(0, dtype=torch.int32, device=cuda_dev))
    assert empty.shape == (0, 4, 64)


# ---------------------------------------------------------------------------------------------------- attention
def _bound(weighted, size, v, keys, dim, dtype):
    logits = 2 * (dim + 16) * 2.0**-23 * size[:, None] + 2.0**-20
    return (2 * U[dtype] + logits) * weighted + (keys * 2.0**-30 * v + 2.0**-25 if dtype == torch.float16 else 0.0) + 1e-30


def _check_rows(got, q, k, v, pos, window, sinks, scale, dtype, what, weights=None):
    """got, q [heads, d] of the query heads that share k, v [keys, d]."""
    want, weighted, size = OA.attend(q, k, v, pos, window, sinks, scale)
    tol = _bound(weighted, size, float(v.double().abs().max()) if v.numel() else 0.0, k.shape[0], q.shape[1], weights or dtype)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (what, float((err - tol).max()), float(err.max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,hq,hkv,dim,window,sinks", [
    ([(1, 1)], 1, 1, 64, 0, 0), ([(2, 2), (129, 129), (1, 1), (0, 0), (64, 64)], 8, 2, 128, 0, 0), ([(300, 300), (5, 300)], 5, 1, 96, 0, 0),
    ([(260, 400), (7, 7)], 4, 4, 64, 100, 3), ([(513, 513)], 32, 8, 128, 128, 130), ([(200, 200)], 2, 1, 40, 1, 0), ([(40, 7), (3, 0)], 4, 2, 128, 0, 0),
    ([(150, 500)], 12, 12, 64, 33, 1), ([(31, 31), (90, 90)], 24, 1, 128, 0, 0), ([(70, 70)], 128, 1, 64, 20, 5), ([(257, 1025)], 6, 2, 8, 0, 0),
    ([(400, 400), (390, 500)] * 4, 12, 12, 64, 0, 0), ([(280, 600), (3, 600), (290, 290)] * 3, 16, 16, 128, 130, 5), ([(40, 3000)], 8, 1, 128, 0, 0),
    ([(700, 700), (0, 5), (1, 900)], 8, 1, 64, 0, 0), ([(300, 2500)], 4, 1, 96, 1000, 200)])  # fmt: skip
def test_prompt_attention(cuda_dev, dtype, lens, hq, hkv, dim, window, sinks):
    g = torch.Generator().manual_seed(dim + hq)
    nq, nk = sum(n for n, _ in lens), sum(m for _, m in lens)
    q = _randn(g, nq, hq, dim, dtype=dtype, std=1.5)
    kv = _randn(g, nk, 2, hkv, dim, dtype=dtype)
    kv[..., -1] += 2
    dkv = kv.to(cuda_dev)
    cu = [torch.tensor([0] + torch.tensor(x).cumsum(0).tolist(), dtype=torch.int32) for x in ([n for n, _ in lens], [m for _, m in lens])]
    got = ops.prompt_attention(q.to(cuda_dev), dkv[:, 0], dkv[:, 1], cu[0].to(cuda_dev), cu[1].to(cuda_dev), max(n for n, _ in lens), window=window, sinks=sinks).cpu()
    ops.check_status(cuda_dev)
    k, v = kv[:, 0], kv[:, 1]
    for b, (n, m) in enumerate(lens):
        q0, k0 = int(cu[0][b]), int(cu[1][b])
        for i in sorted({0, 1, n // 3, n // 2, 126, 127, 128, 129, n - 2, n - 1}):
            if not 0 <= i < n:
                continue
            for h in range(hkv):
                heads = slice(h * hq // hkv, (h + 1) * hq // hkv)
                _check_rows(got[q0 + i, heads], q[q0 + i, heads], k[k0 : k0 + m, h], v[k0 : k0 + m, h], i + m - n, window, sinks, dim**-0.5, dtype, (b, i, h))


def _paged(g, lens, hkv, dim, page, ct, spare=2):
    per = max(1, max(-(-n // page) for n in lens))
    pages = len(lens) * per + spare
    k, v = (_randn(g, pages, hkv, page, dim, dtype=torch.float32).to(ct) for _ in range(2))
    table = torch.randperm(pages, generator=g)[: len(lens) * per].to(torch.int32).view(len(lens), per)
    return k, v, table


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("lens,hq,hkv,dim,page,window,sinks", [
    ([1], 1, 1, 64, 16, 0, 0), ([0, 1, 15, 16, 17, 129, 4000], 8, 2, 128, 16, 0, 0), ([2049], 32, 8, 128, 64, 0, 0), ([300, 70], 5, 1, 96, 24, 0, 0),
    ([1000, 130, 3], 4, 4, 64, 7, 100, 3), ([513, 5000], 40, 4, 128, 128, 128, 130), ([200], 2, 1, 48, 1, 1, 0), ([777], 24, 1, 128, 48, 0, 0),
    ([640], 9, 1, 64, 33, 50, 4), ([90, 0], 6, 2, 16, 5, 0, 0)])  # fmt: skip
def test_paged_attention(cuda_dev, dtype, f8, lens, hq, hkv, dim, page, window, sinks):
    g = torch.Generator().manual_seed(dim * 3 + hq)
    q = _randn(g, len(lens), hq, dim, dtype=dtype, std=1.5)
    k, v, table = _paged(g, lens, hkv, dim, page, F8 if f8 else dtype)
    ks, vs = (torch.rand(hkv, generator=g) * 0.5 + 0.75 if f8 else None for _ in range(2))
    # what lies in the cache behind the last key is never read into a result
    dk, dv = k.to(cuda_dev), v.to(cuda_dev)
    for b, n in enumerate(lens):
        for j in range(n, table.shape[1] * page):
            dk[int(table[b, j // page]), :, j % page] = math.nan
            dv[int(table[b, j // page]), :, j % page] = math.nan
    dev = lambda t: None if t is None else t.to(cuda_dev)  # noqa: E731
    args = (q.to(cuda_dev), dk, dv, table.to(cuda_dev), torch.tensor(lens, dtype=torch.int32, device=cuda_dev))
    got = ops.paged_attention(*args, window=window, sinks=sinks, k_scale=dev(ks), v_scale=dev(vs))
    ops.check_status(cuda_dev)
    assert torch.equal(got, ops.paged_attention(*args, window=window, sinks=sinks, k_scale=dev(ks), v_scale=dev(vs))), "two runs differ"
    got = got.cpu()
    for b, n in enumerate(lens):
        used = table[b, : -(-n // page)].long()
        for h in range(hkv):
            heads = slice(h * hq // hkv, (h + 1) * hq // hkv)
            kk, vv = (x.float()[used, h].reshape(-1, dim)[:n].double() * (1.0 if s is None else s[h].double()) for x, s in ((k, ks), (v, vs)))
            want, weighted, size = OA.attend(q[b, heads], kk, vv, n - 1, window, sinks, dim**-0.5)
            wt = torch.float16 if f8 else dtype
            tol = _bound(weighted, size, float(vv.abs().max()) if n else 0.0, n, dim, wt) + U[dtype] * want.abs()
            err = (got[b, heads].double() - want).abs()
            assert bool((err <= tol).all()), (b, h, float((err - tol).max()))


@pytest.mark.parametrize("layout", ["tokens first", "interleaved"])
def test_paged_attention_takes_other_cache_layouts(cuda_dev, layout):
    """[pages, page size, kv heads, d] storage, and k and v side by side in one tensor, against the same cache laid out densely."""
    g = torch.Generator().manual_seed(5)
    lens, hq, hkv, dim, page = [100, 31], 8, 2, 64, 16
    q = _randn(g, 2, hq, dim).to(cuda_dev)
    k, v, table = (t.to(cuda_dev) for t in _paged(g, lens, hkv, dim, page, torch.bfloat16))
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    want = ops.paged_attention(q, k, v, table, n)
    if layout == "tokens first":
        k2, v2 = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    else:
        both = torch.stack([k, v], 3).contiguous()
        k2, v2 = both[:, :, :, 0], both[:, :, :, 1]
    assert torch.equal(ops.paged_attention(q, k2, v2, table, n), want)
    wide = torch.zeros(2, hq, 2 * dim, dtype=q.dtype, device=cuda_dev)
    wide[..., :dim] = q
    assert torch.equal(ops.paged_attention(wide[..., :dim], k, v, table, n), want)


def test_paged_attention_passes_32_bits_of_offset(cuda_dev):
    """A cache of more than 2^32 elements; the sequence's pages lie at both ends of it."""
    dim, page, hkv = 128, 64, 8
    per_page = hkv * page * dim
    pages = (1 << 32) // per_page + 40
    g = torch.Generator().manual_seed(6)
    k = torch.zeros(pages, hkv, page, dim, dtype=F8, device=cuda_dev)
    v = torch.zeros(pages, hkv, page, dim, dtype=F8, device=cuda_dev)
    use = [pages - 1, 0, pages - 7, 3]
    sk, sv = (_randn(g, 4, hkv, page, dim, dtype=torch.float32).to(F8) for _ in range(2))
    for i, u in enumerate(use):
        k[u], v[u] = sk[i].to(cuda_dev), sv[i].to(cuda_dev)
    q = _randn(g, 1, 32, dim).to(cuda_dev)
    one = torch.ones(hkv, device=cuda_dev)
    n = torch.tensor([250], dtype=torch.int32, device=cuda_dev)
    got = ops.paged_attention(q, k, v, torch.tensor([use], dtype=torch.int32, device=cuda_dev), n, k_scale=one, v_scale=one)
    small = ops.paged_attention(q, sk.to(cuda_dev), sv.to(cuda_dev), torch.arange(4, dtype=torch.int32, device=cuda_dev)[None], n, k_scale=one, v_scale=one)
    ops.check_status(cuda_dev)
    assert torch.equal(got, small)
    x = _randn(g, 1, hkv, dim).to(cuda_dev)
    cos, sin = (t.to(cuda_dev) for t in _tables(4, dim))
    zero = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    ops.qk_norm_rope(q, x, cos, sin, zero, v=x, k_pages=k, v_pages=v, slots=torch.tensor([pages * page - 1], device=cuda_dev), k_scale=one, v_scale=one)
    assert torch.equal(v[-1, :, -1].float(), x[0].to(F8).float()) and torch.equal(k[-1, :, -1].float(), x[0].to(F8).float())
    assert not v[-2].float().any()


def test_masked_places_may_hold_anything(cuda_dev):
    """NaN and infinities in keys and values that a query does not see leave its output as it is."""
    g = torch.Generator().manual_seed(7)
    n, hq, hkv, dim = 300, 4, 2, 128
    q, k, v = _randn(g, n, hq, dim), _randn(g, n, hkv, dim), _randn(g, n, hkv, dim)
    cu = torch.tensor([0, n], dtype=torch.int32, device=cuda_dev)
    bad = {40: (math.nan, 1.0), 130: (1.0, math.nan), 131: (math.inf, math.inf), 250: (-math.inf, -math.inf), 299: (math.nan, math.nan)}
    k2, v2 = k.clone(), v.clone()
    for j, (a, b) in bad.items():
        k2[j], v2[j] = a, b
    for window, sinks in ((0, 0), (50, 2)):
        want = ops.prompt_attention(*(t.to(cuda_dev) for t in (q, k, v)), cu, cu, n, window=window, sinks=sinks).cpu()
        got = ops.prompt_attention(*(t.to(cuda_dev) for t in (q, k2, v2)), cu, cu, n, window=window, sinks=sinks).cpu()
        for i in range(n):
            seen = OA.visible(i, window, sinks)
            if not any(j in bad for j in seen):
                err = (got[i].double() - want[i].double()).abs()
                assert bool((err <= 4 * U[torch.bfloat16] * v[: i + 1].double().abs().amax()).all()), (window, i, float(err.max()))
            elif 40 in seen or 130 in seen:
                assert bool(got[i].isnan().all()), (window, i)


def test_rows_of_minus_infinity_are_zeros(cuda_dev):
    dim = 64
    q = torch.ones(3, 2, dim, dtype=torch.bfloat16, device=cuda_dev)
    k = torch.full((3, 2, dim), -math.inf, dtype=torch.bfloat16, device=cuda_dev)
    v = torch.ones(3, 2, dim, dtype=torch.bfloat16, device=cuda_dev)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=cuda_dev)
    assert not ops.prompt_attention(q, k, v, cu, cu, 3).any()
    pages = k.transpose(0, 1)[None].contiguous()
    table, n = torch.zeros(1, 1, dtype=torch.int32, device=cuda_dev), torch.tensor([3], dtype=torch.int32, device=cuda_dev)
    assert not ops.paged_attention(q[:1], pages, torch.ones_like(pages), table, n).any()
    # NaN that is visible comes through
    k[1, 0, 0] = math.nan
    got = ops.prompt_attention(q, k, v, cu, cu, 3)
    assert not got[0].any() and got[1, 0].isnan().all() and not got[1, 1].any()


def test_windows_and_first_tokens_beyond_every_sequence(cuda_dev):
    """The largest 32-bit window or number of first tokens is no window, and both attentions refuse a scale that is not positive."""
    g = torch.Generator().manual_seed(12)
    q, k, v = (_randn(g, 300, h, 64).to(cuda_dev) for h in (4, 2, 2))
    cu = torch.tensor([0, 300], dtype=torch.int32, device=cuda_dev)
    pages = [t.transpose(0, 1)[None].contiguous() for t in (k, v)]
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_dev)
    prompt = lambda **kw: ops.prompt_attention(q, k, v, cu, cu, 300, **kw)  # noqa: E731
    token = lambda **kw: ops.paged_attention(q[-1:], *pages, table, cu[1:], **kw)  # noqa: E731
    big = 2**31 - 1
    for run in (prompt, token):
        want = run()
        assert torch.equal(run(window=big), want) and torch.equal(run(window=big, sinks=big), want)
        assert torch.allclose(run(window=7, sinks=big).float(), want.float(), atol=2.0**-6)
        for scale in (0.0, -1.0, math.nan, math.inf):
            with pytest.raises(RuntimeError, match="scale"):
                run(scale=scale)


def test_large_logits_and_scales(cuda_dev):
    """Logits of several thousand: the running maximum has to be followed upwards and the sums must not overflow."""
    g = torch.Generator().manual_seed(8)
    n, dim = 700, 64
    q, k, v = _randn(g, n, 2, dim, std=20.0), _randn(g, n, 1, dim, std=20.0), _randn(g, n, 1, dim)
    k[:, 0, 0] += torch.arange(n).to(torch.bfloat16)  # grows along the keys
    cu = torch.tensor([0, n], dtype=torch.int32, device=cuda_dev)
    got = ops.prompt_attention(*(t.to(cuda_dev) for t in (q, k, v)), cu, cu, n, scale=0.5).cpu()
    for i in (0, 1, 127, 128, 300, 699):
        _check_rows(got[i], q[i], k[:, 0], v[:, 0], i, 0, 0, 0.5, torch.bfloat16, i)
    pages = [t.transpose(0, 1)[None].contiguous().to(cuda_dev) for t in (k, v)]
    out = ops.paged_attention(q[-1:].to(cuda_dev), *pages, torch.zeros(1, 1, dtype=torch.int32, device=cuda_dev), cu[1:], scale=0.5).cpu()
    _check_rows(out[0], q[-1], k[:, 0], v[:, 0], n - 1, 0, 0, 0.5, torch.bfloat16, "token")


def test_queries_of_any_size_meet_an_e4m3_cache(cuda_dev):
    """bf16 queries far outside fp16's range keep their digits."""
    g = torch.Generator().manual_seed(9)
    for std in (1e-30, 1e-6, 1e6, 1e20):
        q = _randn(g, 1, 4, 64, dtype=torch.float32).mul(std).to(torch.bfloat16)
        k, v, table = _paged(g, [200], 1, 64, 16, F8)
        one = torch.ones(1, device=cuda_dev)
        got = ops.paged_attention(q.to(cuda_dev), k.to(cuda_dev), v.to(cuda_dev), table.to(cuda_dev), torch.tensor([200], dtype=torch.int32, device=cuda_dev),
                                  scale=0.1 / std, k_scale=one, v_scale=one).cpu()  # fmt: skip
        kk, vv = (x.float()[table[0].long(), 0].reshape(-1, 64)[:200] for x in (k, v))
        want, weighted, size = OA.attend(q[0], kk, vv, 199, 0, 0, 0.1 / std)
        err = (got[0].double() - want).abs()
        assert bool((err <= _bound(weighted, size, 4.0, 200, 64, torch.float16) + 2.0**-8 * want.abs()).all()), std


def test_lengths_pages_and_offsets_out_of_range_are_reported(cuda_dev):
    g = torch.Generator().manual_seed(10)
    q = _randn(g, 2, 4, 64).to(cuda_dev)
    k, v, table = (t.to(cuda_dev) for t in _paged(g, [64, 64], 2, 64, 16, torch.bfloat16))
    n = torch.tensor([64, 64], dtype=torch.int32, device=cuda_dev)
    ops.check_status(cuda_dev)
    for what in ("length", "negative", "page"):
        t2, n2 = table.clone(), n.clone()
        if what == "page":
            t2[1, 2] = k.shape[0]
        else:
            n2[1] = 65 if what == "length" else -3
        got = ops.paged_attention(q, k, v, t2, n2)
        with pytest.raises(RuntimeError, match="status"):
            ops.check_status(cuda_dev)
        assert torch.equal(got[0], ops.paged_attention(q, k, v, table, n)[0]), what
    x = _randn(g, 10, 4, 64).to(cuda_dev)
    for cu_q, cu_k, most in (([0, 5, 11], [0, 5, 10], 6), ([0, 7, 5], [0, 5, 10], 7), ([0, 5, 10], [0, 5, 10], 4), ([0, 5, 10], [0, 12, 10], 5), ([1, 5, 10], [0, 5, 10], 5)):
        ops.prompt_attention(x, x, x, *(torch.tensor(c, dtype=torch.int32, device=cuda_dev) for c in (cu_q, cu_k)), most)
        with pytest.raises(RuntimeError, match="status"):
            ops.check_status(cuda_dev)


def test_refusals(cuda_dev):
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=cuda_dev)
    i = torch.zeros(2, dtype=torch.int32, device=cuda_dev)
    cos = torch.zeros(4, 32, device=cuda_dev)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16, device=cuda_dev)
    table = torch.zeros(2, 1, dtype=torch.int32, device=cuda_dev)
    f8 = pages.to(F8)
    for bad, match in (
        (lambda: ops.qk_norm_rope(x, x.half(), cos, cos, i), "q and k"),
        (lambda: ops.qk_norm_rope(x, x, cos, cos, i.long()), "positions"),
        (lambda: ops.qk_norm_rope(x, x, cos.half(), cos.half(), i), "cos"),
        (lambda: ops.qk_norm_rope(x, x, cos, cos, i, v=x), "k_pages is missing"),
        (lambda: ops.qk_norm_rope(x, x[:, :2], cos, cos, i, v=x[:, :2], k_pages=f8, v_pages=f8, slots=i.long()), "k_scale"),
        (lambda: ops.qk_norm_rope(x, x[:, :2], cos, cos, i, v=x[:, :2], k_pages=pages, v_pages=pages, slots=i), "slots"),
        (lambda: ops.qk_norm_rope(x, x, torch.zeros(4, 36, device=cuda_dev), torch.zeros(4, 36, device=cuda_dev), i), "rotary"),
        (lambda: ops.qk_norm_rope(x.clone().requires_grad_(), x, cos, cos, i), "gradient"),
        (lambda: ops.paged_attention(x.float(), pages, pages, table, i), "float16"),
        (lambda: ops.paged_attention(x, pages.half(), pages.half(), table, i), "type"),
        (lambda: ops.paged_attention(x, pages, pages.transpose(1, 2).contiguous().transpose(1, 2), table, i), "strides"),
        (lambda: ops.paged_attention(x, f8, f8, table, i), "k_scale"),
        (lambda: ops.paged_attention(x, pages, pages, table.long(), i), "block_table"),
        (lambda: ops.paged_attention(x, pages, pages, table, i, sinks=-1), "sinks"),
        (lambda: ops.paged_attention(x[:, :3], pages, pages, table, i), "multiple"),
        (lambda: ops.paged_attention(x, pages, pages, table, i, out=x.half()), "out"),
        (lambda: ops.prompt_attention(x, x, x.half(), i, i, 1), "q, k and v"),
        (lambda: ops.prompt_attention(x, x, x, i, i[:1], 1), "cu_k"),
        (lambda: ops.prompt_attention(x, x, x, i, i, 3), "max_q"),
        (lambda: ops.prompt_attention(x, x, x.clone().requires_grad_(), i, i, 1), "gradient"),
    ):
        with pytest.raises(RuntimeError, match=match):
            bad()


def test_another_stream_and_graph_capture(cuda_dev):
    g = torch.Generator().manual_seed(11)
    q = _randn(g, 3, 8, 128).to(cuda_dev)
    k, v, table = (t.to(cuda_dev) for t in _paged(g, [900, 50, 333], 2, 128, 32, torch.bfloat16))
    n = torch.tensor([900, 50, 333], dtype=torch.int32, device=cuda_dev)
    x = _randn(g, 333, 8, 128).to(cuda_dev)
    cu = torch.tensor([0, 333], dtype=torch.int32, device=cuda_dev)
    want = ops.paged_attention(q, k, v, table, n), ops.prompt_attention(x, x, x, cu, cu, 333)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_attention(q, k, v, table, n), ops.prompt_attention(x, x, x, cu, cu, 333)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = ops.paged_attention(q, k, v, table, n), ops.prompt_attention(x, x, x, cu, cu, 333)
    n.copy_(torch.tensor([899, 51, 1], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(cap[0], ops.paged_attention(q, k, v, table, n)) and torch.equal(cap[1], want[1])
    ops.check_status(cuda_dev)
