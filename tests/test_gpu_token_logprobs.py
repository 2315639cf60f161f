"""Log probabilities of given tokens, entropy, top alternatives and their gradient, against 64 bits.

Bounds.  A thread adds up one of 256 shares of a row in two halves, so S is a sum of n = vocab / 512 + 64 roundings at most (the pieces' and the joins' among
them), each of its terms an exponential of 2 ulp whose argument is |d| 2^-24 off, d <= 0 the distance from the largest logit: weighted by the terms
themselves that is the mean distance.  So log S is (n + distance) 2^-23 off, a log probability 2^-23 of its size more, and the entropy, whose
second sum has terms d times as large, (n + distance) (1 + distance) 2^-22.  A gradient adds the rounding to the logits' type, half a step there.
"""

import math

import pytest
import torch

from fms_model_optimizer_b200 import ops
from oracle import requests as OR

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(got, x, tokens, top):
    """All four results of rows on the CPU against the oracle's."""
    lp, entropy, top_lp, top_ids = (t.cpu() for t in got)
    want = OR.score(x, tokens, top)
    n, far = x.shape[1] / 512 + 64, want["distance"]
    log_s = (n + far) * 2.0**-23

    def near(a, b, bound):
        assert torch.equal(a.isnan(), b.isnan())
        fine = b.isfinite()
        assert torch.equal(a[~fine & ~b.isnan()], b[~fine & ~b.isnan()].float())
        assert bool(((a.double() - b).abs() <= bound)[fine].all()), float(((a.double() - b).abs() / bound)[fine].max())

    near(lp, want["logprobs"], log_s + 2.0**-23 * want["logprobs"].abs())
    near(entropy, want["entropy"], (n + far) * (1 + far) * 2.0**-22)
    if top:
        assert torch.equal(top_ids, want["top_ids"])
        near(top_lp, want["top_logprobs"], log_s[:, None] + 2.0**-23 * want["top_logprobs"].abs())


def _logits(g, rows, vocab, dtype, std=3.0):
    return (torch.randn((rows, vocab), generator=g) * std).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 7, 7), (3, 33, 5), (2, 1000, 32), (5, 50257, 20), (2, 128256, 5), (300, 2053, 8), (1, 262145, 32), (700, 512, 0),
                                            (9, 4096, 1), (2, 300001, 0), (160, 8191, 31), (1, 1 << 20, 32), (150, 1 << 17, 9)])  # fmt: skip
def test_against_64_bits(cuda_dev, dtype, rows, vocab, top):
    g = torch.Generator().manual_seed(rows * 31 + vocab)
    x = _logits(g, rows, vocab, dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    tokens[rows // 2 :: 3] = -100
    got = ops.token_logprobs(x.to(cuda_dev), tokens.to(cuda_dev), top=top)
    ops.check_status(cuda_dev)
    _check(got, x, tokens, top)
    assert bool((got[0].cpu()[tokens < 0] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,pitch", [(0, 5001), (1, 5008), (3, 4999), (7, 5003), (0, 0)])
def test_rows_of_any_alignment(cuda_dev, dtype, offset, pitch):
    """Rows that start anywhere, with a pitch, shared by all (pitch 0), or with other leading dimensions."""
    g = torch.Generator().manual_seed(offset + pitch)
    flat = _logits(g, 1, 6 * 5100, dtype)[0]
    x = flat.as_strided((6, 4999), (pitch, 1), offset)
    d = flat.to(cuda_dev).as_strided((6, 4999), (pitch, 1), offset)
    tokens = torch.randint(0, 4999, (6,), generator=g)
    _check(ops.token_logprobs(d, tokens.to(cuda_dev), top=9), x, tokens, 9)
    lp, h, tl, ti = ops.token_logprobs(d.unflatten(0, (2, 3)), tokens.to(cuda_dev).view(2, 3), top=9)
    assert lp.shape == h.shape == (2, 3) and tl.shape == ti.shape == (2, 3, 9)
    _check((lp.flatten(), h.flatten(), tl.flatten(0, 1), ti.flatten(0, 1)), x, tokens, 9)


def _orders(vocab, g):
    """Rows whose top elements lie where the search for them has to go its longer ways."""
    i = torch.arange(vocab)
    rows = {
        "equal": torch.zeros(vocab),
        "falling": -i / 8.0,
        "rising": i / 8.0,
        "whole": torch.randint(-3, 4, (vocab,), generator=g).float(),
        "two": (torch.rand(vocab, generator=g) < 0.4).float(),
        "few": torch.where(i % (vocab // 9) == 5, torch.randn(vocab, generator=g), -math.inf),
        "one": torch.where(i == vocab - 1, 2.0, -math.inf),
        "zeros": torch.where(i % 2 == 0, -0.0, 0.0),
        "threads": torch.where(i // 8 % 256 < 31, 9.0 + (i * 7919 % 1021) / 8.0, 1.0),  # thousands in few threads' shares of 16-bit rows
        "narrow": torch.where(i // 4 % 256 < 31, 9.0 + (i * 7919 % 1021) / 8.0, 1.0),  # and of 32-bit ones
        "late": torch.where(i > vocab - 1500, 5.0, 0.0) + torch.where(i == 3, 6.0, 0.0),
    }
    return list(rows), torch.stack([r.float() for r in rows.values()])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,repeat", [(50257, 1), (50257, 40), (300, 1), (16384, 1)])
def test_equal_and_ordered_logits(cuda_dev, dtype, vocab, repeat):
    """Ties go to the lower id whatever the order of the row; few rows (in clusters) and many give the same."""
    _, x = _orders(vocab, torch.Generator().manual_seed(vocab))
    x = x.to(dtype).repeat(repeat, 1)
    tokens = torch.arange(x.shape[0]) * 37 % vocab
    for top in (1, 20, 32):
        _check(ops.token_logprobs(x.to(cuda_dev), tokens.to(cuda_dev), top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan(cuda_dev, dtype):
    vocab, top = 9001, 12
    g = torch.Generator().manual_seed(3)
    x = _logits(g, 9, vocab, dtype)
    x[1] = -math.inf
    x[2, 777] = math.nan
    x[3, 9000] = math.inf
    x[4, ::2] = -math.inf
    x[5, 1:] = -math.inf
    x[6, :5000] = math.nan
    x[7] = math.nan
    x[8, 0] = -math.nan
    tokens = torch.tensor([5, 6, 7, 9000, 10, 0, 1, -1, 4])
    got = ops.token_logprobs(x.to(cuda_dev), tokens.to(cuda_dev), top=top)
    want = OR.score(x, tokens, top)
    assert torch.equal(got[3].cpu(), want["top_ids"])
    for r in (1, 2, 3, 6, 7, 8):
        assert bool(got[1][r].isnan()) and (tokens[r] < 0 or bool(got[0][r].isnan())) and bool(got[2][r].isnan().all())
    assert float(got[0][7]) == 0.0
    for r in (0, 4, 5):
        _check([t[r : r + 1] for t in got], x[r : r + 1], tokens[r : r + 1], top)
    assert float(got[0][5]) == 0.0 and float(got[1][5]) == 0.0


@pytest.mark.parametrize("size", [1e3, 3e4, 1e30, 1e38])
def test_logits_of_any_finite_size(cuda_dev, size):
    dtype = torch.float16 if size == 3e4 else torch.float32
    g = torch.Generator().manual_seed(4)
    x = torch.cat([_logits(g, 2, 3000, torch.float32) + size, _logits(g, 2, 3000, torch.float32) - size, _logits(g, 2, 3000, torch.float32) * size / 16]).to(dtype)
    tokens = torch.randint(0, 3000, (6,), generator=g)
    _check(ops.token_logprobs(x.to(cuda_dev), tokens.to(cuda_dev), top=4), x, tokens, 4)


def test_the_same_every_time(cuda_dev):
    g = torch.Generator().manual_seed(5)
    x, tokens = _logits(g, 37, 50001, torch.bfloat16).to(cuda_dev), torch.randint(0, 50001, (37,), generator=g).to(cuda_dev)
    first = ops.token_logprobs(x, tokens, top=20)
    for _ in range(5):
        for a, b in zip(first, ops.token_logprobs(x, tokens, top=20)):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------- the gradient
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _half_step(want, dtype):
    exponent = torch.frexp(want.abs())[1].clamp(min={torch.float16: -13, torch.bfloat16: -125, torch.float32: -125}[dtype])
    return torch.ldexp(torch.full_like(want, U[dtype]), exponent - 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,offset", [(1, 5, 0), (3, 1000, 0), (7, 50257, 0), (4, 9003, 1), (2, 128256, 0), (1, 1, 0)])
def test_gradient(cuda_dev, dtype, rows, vocab, offset):
    g = torch.Generator().manual_seed(vocab)
    flat = _logits(g, 1, rows * vocab + offset, dtype)[0]
    x = flat[offset:].view(rows, vocab)
    if vocab > 100:
        x[0, ::3] = -math.inf
    tokens = torch.randint(0, vocab // 3 + 1, (rows,), generator=g) * 3 + 1
    tokens = tokens.clamp(max=vocab - 1)
    tokens[rows // 2 :: 3] = -100
    dl, dh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    leaf = flat.to(cuda_dev)[offset:].view(rows, vocab).requires_grad_(True)
    lp, h, top_lp, _ = ops.token_logprobs(leaf, tokens.to(cuda_dev), top=1)
    assert not top_lp.requires_grad
    for use_l, use_h in ((1, 1), (1, 0), (0, 1)):
        outs = [t for t, use in ((lp, use_l), (h, use_h)) if use]
        ins = [t.to(cuda_dev) for t, use in ((dl, use_l), (dh, use_h)) if use]
        (got,) = torch.autograd.grad(outs, leaf, ins, retain_graph=True)
        want, size = OR.score_gradient(x, tokens, dl * use_l, dh * use_h)
        assert got.dtype == dtype and got.shape == x.shape
        # p is as far off as log S and its own exponent, the entropy as above
        s = OR.score(x, tokens, 0)
        n = vocab / 512 + 64 + s["distance"]
        bound = _half_step(want, dtype) * (1 + 2.0**-10) + ((n * (1 + s["distance"]))[:, None] + s["log_p"].abs().clamp(max=200)) * 2.0**-21 * size + 2.0**-126
        err = (got.cpu().double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


def test_gradient_against_differences(cuda_dev):
    g = torch.Generator().manual_seed(11)
    x = _logits(g, 3, 400, torch.float32)
    tokens, dl, dh = torch.tensor([3, -1, 399]), torch.randn(3, generator=g), torch.randn(3, generator=g)
    leaf = x.to(cuda_dev).requires_grad_(True)
    lp, h, _, _ = ops.token_logprobs(leaf, tokens.to(cuda_dev))
    (got,) = torch.autograd.grad((lp, h), leaf, (dl.to(cuda_dev), dh.to(cuda_dev)))
    f = lambda z: (lambda s: (s["logprobs"] * dl + s["entropy"] * dh).sum())(OR.score(z, tokens, 0))  # noqa: E731
    step = 2.0**-12
    for _ in range(4):
        u = torch.randn(x.shape, generator=g, dtype=torch.float64)
        differences = (f(x.double() + step * u) - f(x.double() - step * u)) / (2 * step)
        # the differences' own error is step^2 times third derivatives of order one; the gradient's 2^-17 of a sum of 1200 products
        assert abs(float(differences - (got.cpu().double() * u).sum())) < 100 * step**2 + 2.0**-17 * float((got.cpu().double() * u).abs().sum())


def test_training_through_a_head(cuda_dev):
    """The loss of a head: gradients reach the weights, a step of padding alone gives zeros, and twice differentiating is refused."""
    g = torch.Generator(device=cuda_dev).manual_seed(7)
    w = torch.randn(1003, 64, generator=g, device=cuda_dev).requires_grad_(True)
    hidden = torch.randn(12, 64, generator=g, device=cuda_dev)
    tokens = torch.randint(0, 1003, (12,), generator=g, device=cuda_dev)
    tokens[4] = -100
    lp, _, _, _ = ops.token_logprobs(hidden @ w.t(), tokens)
    (-lp.sum() / 11).backward()
    w2 = w.detach().clone().requires_grad_(True)
    torch.nn.functional.cross_entropy(hidden @ w2.t(), tokens, ignore_index=-100).backward()
    # both are fp32 products of fp32 gradients: sums of 12 and of 64 terms
    assert float((w.grad - w2.grad).abs().max()) <= 2.0**-18 * float(w2.grad.abs().max())
    logits = torch.randn(2, 50, device=cuda_dev, requires_grad=True)
    lp, h, _, _ = ops.token_logprobs(logits, torch.tensor([-1, -7], device=cuda_dev))
    (grad,) = torch.autograd.grad(lp.sum(), logits, retain_graph=True)
    assert int(grad.count_nonzero()) == 0
    (grad,) = torch.autograd.grad(h.sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_large_steps_in_memory(cuda_dev):
    """Rows whose offsets pass 2^31 elements."""
    vocab, pitch = 1000, 1 << 30
    flat = torch.zeros(2 * pitch + vocab, dtype=torch.bfloat16, device=cuda_dev)
    x = flat.as_strided((3, vocab), (pitch, 1))
    g = torch.Generator().manual_seed(8)
    rows = _logits(g, 3, vocab, torch.bfloat16)
    x.copy_(rows)
    tokens = torch.tensor([1, 2, 999])
    _check(ops.token_logprobs(x, tokens.to(cuda_dev), top=5), rows, tokens, 5)


def test_tokens_out_of_range_and_refusals(cuda_dev):
    x = torch.randn(3, 10, device=cuda_dev)
    tokens = torch.tensor([1, 10, 2], device=cuda_dev)
    lp, _, _, _ = ops.token_logprobs(x, tokens)
    assert float(lp[1]) == 0.0
    with pytest.raises(RuntimeError, match="status"):
        ops.check_status(cuda_dev)
    ok = torch.tensor([1, 2, 3], device=cuda_dev)
    for bad in (lambda: ops.token_logprobs(x, ok.int()), lambda: ops.token_logprobs(x, ok[:2]), lambda: ops.token_logprobs(x.double(), ok), lambda: ops.token_logprobs(x, ok, top=11),
                lambda: ops.token_logprobs(x, ok, top=-1), lambda: ops.token_logprobs(x.cpu(), ok), lambda: ops.token_logprobs(x[:, :0], ok),
                lambda: ops.token_logprobs(torch.randn(3, 100, device=cuda_dev), ok, top=33)):  # fmt: skip
        with pytest.raises(RuntimeError):
            bad()
    assert ops.token_logprobs(x[:0], ok[:0], top=3)[2].shape == (0, 3)


def test_streams_and_graphs(cuda_dev):
    g = torch.Generator().manual_seed(9)
    x, tokens = _logits(g, 5, 3001, torch.float16), torch.randint(0, 3001, (5,), generator=g)
    sx, st = x.to(cuda_dev), tokens.to(cuda_dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check(ops.token_logprobs(sx, st, top=7), x, tokens, 7)
    graph = torch.cuda.CUDAGraph()
    leaf = sx.clone().requires_grad_(True)
    ones = torch.ones(5, device=cuda_dev)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.token_logprobs(leaf, st, top=7)
        (grad,) = torch.autograd.grad(out[0], leaf, ones)
    for seed in (1, 2):
        x = _logits(torch.Generator().manual_seed(seed), 5, 3001, torch.float16)
        with torch.no_grad():
            leaf.copy_(x)
        graph.replay()
        _check([t.detach() for t in out], x, tokens, 7)
        want, _ = OR.score_gradient(x, tokens, ones.cpu(), 0 * ones.cpu())
        assert float((grad.cpu().double() - want).abs().max()) < 2.0**-11
