"""Many requests answered together by the decoder: a shared prefix, an adapter each, log probabilities.

A code that flips by one in an int8 row can move a later layer of a random model by any amount, so two ways of one computation are compared call by call, on the inputs that each call
was given, and where their inputs are the same to the bit.  Bounds (u = 2^-8, bf16; 2^-11 with an e4m3 cache, which is read in fp16).  Attention by two kernels: the weights of each
are rounded (u of the largest value), and its output (2^-8): 2 (u + 2^-8) max |v|, and logits that are 2^-12 apart at most here.  Adapters: y is rounded once (2^-9 of it, half a step), v is
kept to 2^-16 and its sums to 2^-12 of the sum of magnitudes.  Log probabilities of 2048 logits: 2^-16.
"""

import pytest
import torch

from fms_model_optimizer_b200 import decoder, ops
from fms_model_optimizer_b200.adapters import LoraAdapters
from fms_model_optimizer_b200.decoder import Generated, W8A8Decoder, linear_shapes
from fms_model_optimizer_b200.kvcache import PagedKVCache
from oracle import requests as OR

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=2048, rope_theta=10000.0, batch=3, seq=256)


@pytest.fixture(scope="module")
def model(cuda_dev):
    return W8A8Decoder(CFG, cuda_dev)


def _ids(dev, *lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, CFG["vocab"], (n,), generator=g).to(dev) for n in lengths]


def _off(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _pool(dev, adapters=3, rank=12, size=0.02, seed=3):
    pool = LoraAdapters({n: s[:2] for n, s in linear_shapes(CFG).items()}, CFG["layers"], adapters, rank, dev)
    g = torch.Generator(device=dev).manual_seed(seed)
    for (li, name), a in pool.a.items():
        for i in range(adapters):
            pool.load(i, li, name, torch.randn(rank, a.shape[2], generator=g, device=dev) * a.shape[2] ** -0.5, torch.randn(pool.b[li, name].shape[1], rank, generator=g, device=dev) * size)
    pool.scale.copy_(torch.tensor([0.5, 1.0, 2.0][:adapters]))
    return pool


class Checked:
    """The three operators, each checked on every call that it gets."""

    def __init__(self, monkeypatch):
        self.calls = dict(prefix=0, lora=0, score=0)
        self.real = ops.prefix_attention, ops.lora_add_, ops.token_logprobs
        for name, fn in (("prefix_attention", self.prefix), ("lora_add_", self.lora), ("token_logprobs", self.score)):
            monkeypatch.setattr(ops, name, fn)

    def prefix(self, q, k_pages, v_pages, prefix_table, prefix_lens, groups, block_table, lens, **kw):
        """Against the attention over pages, on a cache in which every sequence has the prefix to itself."""
        self.calls["prefix"] += 1
        got = self.real[0](q, k_pages, v_pages, prefix_table, prefix_lens, groups, block_table, lens, **kw)
        page, n, longest = k_pages.shape[2], int(prefix_lens[0]), int(lens.max())
        assert groups.tolist() == [0, q.shape[0]] and bool((lens > n).all())
        key = torch.arange(longest, device=q.device)
        column = (key // page).clamp(max=block_table.shape[1] - 1)
        of = torch.where(key < n, prefix_table[0][(key // page).clamp(max=prefix_table.shape[1] - 1)], block_table[:, column]).long()  # [batch, keys]
        raw = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t  # noqa: E731
        dense = [raw(t)[of, :, key % page].transpose(1, 2).contiguous().view(t.dtype) for t in (k_pages, v_pages)]  # a page a sequence
        table = torch.arange(q.shape[0], dtype=torch.int32, device=q.device)[:, None]
        want = ops.paged_attention(q, *dense, table, lens, **{x: y for x, y in kw.items()})
        u = 2.0**-11 if k_pages.dtype == torch.float8_e4m3fn else 2.0**-8
        most = float((dense[1].float() * (1.0 if kw.get("v_scale") is None else kw["v_scale"][:, None, None])).nan_to_num().abs().max())
        assert float((got.float() - want.float()).abs().max()) <= (2 * (u + 2.0**-8) + 2.0**-11) * most
        return got

    def lora(self, y, x, a, b, rows, starts, scale):
        self.calls["lora"] += 1
        before = y.double()
        got = self.real[1](y, x, a, b, rows, starts, scale)
        want, size, at = before.clone(), torch.zeros_like(before), starts.tolist()
        for i in range(a.shape[0]):
            r = rows[at[i] : at[i + 1]].long()
            v = x[r].double() @ a[i].double().t()
            want[r] += scale[i].double() * (v @ b[i].double().t())
            size[r] = scale[i].double() * ((x[r].double().abs() @ a[i].double().abs().t()) @ b[i].double().abs().t())
        assert bool(((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-11 * size + 1e-30).all())
        listed = torch.zeros(y.shape[0], dtype=torch.bool, device=y.device)
        listed[rows[: at[-1]].long()] = True
        assert torch.equal(got[~listed].double(), before[~listed])
        return got

    def score(self, logits, tokens, *, top=0):
        self.calls["score"] += 1
        got = self.real[2](logits, tokens, top=top)
        want = OR.score(logits.cpu(), tokens.cpu(), top)
        assert float((got[0].cpu() - want["logprobs"]).abs().max()) < 2.0**-16 and float((got[1].cpu() - want["entropy"]).abs().max()) < 2.0**-14
        assert torch.equal(got[3].cpu(), want["top_ids"])
        return got


@pytest.mark.parametrize("extra,cache_dtype", [({}, torch.bfloat16), ({}, torch.float8_e4m3fn), (dict(qk_norm=True, window=50, sinks=2), torch.bfloat16)])
@pytest.mark.parametrize("shared", [70, 16, 1])
def test_a_prefix_is_as_if_it_stood_in_every_prompt(cuda_dev, extra, cache_dtype, shared, monkeypatch):
    m = W8A8Decoder(dict(CFG, **extra), cuda_dev)
    prefix, *prompts = _ids(cuda_dev, shared, 37, 1, 90)
    make = lambda: PagedKVCache(2, 3, shared + 95, 2, 128, cuda_dev, cache_dtype, 16)  # noqa: E731
    caches = make(), make()
    out = m.generate(prompts, 6, cache=caches[0], prefix=prefix)
    ops.check_status(cuda_dev)
    assert torch.equal(out, m.generate(prompts, 6, cache_dtype=cache_dtype, page_size=16, prefix=prefix)), "two runs differ"
    checked = Checked(monkeypatch)
    assert torch.equal(out, m.generate(prompts, 6, cache_dtype=cache_dtype, page_size=16, prefix=prefix)) and checked.calls["prefix"] == 2 * 5
    # in the first layer the same keys and values, at the same positions, as where the prefix is written out
    m.generate([torch.cat([prefix, p]) for p in prompts], 6, cache=caches[1])
    for pools in zip(caches[0].k[:1] + caches[0].v[:1], caches[1].k[:1] + caches[1].v[:1]):
        a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in pools)
        for s, p in enumerate(prompts):
            for i in range(shared + p.numel()):
                at = (caches[0].prefix_table[0] if i < shared else caches[0].table[s])[i // 16]
                assert torch.equal(a[at, :, i % 16], b[caches[1].table[s, i // 16], :, i % 16]), (s, i)


def test_adapters_are_each_requests_own(cuda_dev, model):
    prompts = _ids(cuda_dev, 20, 33, 1, 12)
    pool = _pool(cuda_dev)
    base = model.generate(prompts, 4, page_size=8)
    base_hidden = model.last_hidden
    # adapters of nothing but zeros, or none at all, change nothing
    zeros = LoraAdapters({n: s[:2] for n, s in linear_shapes(CFG).items()}, CFG["layers"], 2, 8, cuda_dev)
    assert torch.equal(base, model.generate(prompts, 4, page_size=8, adapters=zeros, which=[0, 1, -1, 0]))
    assert torch.equal(base, model.generate(prompts, 4, page_size=8, adapters=pool, which=[-1] * 4))
    mixed = model.generate(prompts, 4, page_size=8, adapters=pool, which=[2, -1, 0, 2])
    hidden = model.last_hidden
    assert torch.equal(mixed[1], base[1]) and torch.equal(hidden[1], base_hidden[1])
    assert all(_off(hidden[b], base_hidden[b]) > 0.2 for b in (0, 3)), "the adapters do nothing"
    for b, i in ((0, 2), (2, 0), (3, 2)):  # alone, the same
        alone = model.generate([prompts[b]], 4, page_size=8, adapters=pool, which=[i])
        assert torch.equal(alone[0], mixed[b]), b
    ops.check_status(cuda_dev)


def test_adapters_add_the_product_at_every_linear(cuda_dev, model, monkeypatch):
    """Every Linear's adapter is called with that Linear's own input and output, prompts and tokens, and adds what it should."""
    prompts = _ids(cuda_dev, 20, 33, seed=5)
    pool = _pool(cuda_dev)
    out = model.generate(prompts, 3, page_size=8, adapters=pool, which=[1, 2])
    checked, seen = Checked(monkeypatch), []
    inner = ops.lora_add_
    monkeypatch.setattr(ops, "lora_add_", lambda y, x, *rest: (seen.append((tuple(x.shape), tuple(y.shape))), inner(y, x, *rest))[1])
    assert torch.equal(out, model.generate(prompts, 3, page_size=8, adapters=pool, which=[1, 2]))
    shapes = [(n, k) for n, k, _ in linear_shapes(CFG).values()]
    assert checked.calls["lora"] == 3 * 2 * 7 and [(y[1], x[1]) for x, y in seen[:7]] == shapes
    assert [x[0] for x, _ in seen] == [53] * 14 + [2] * 28


@pytest.mark.parametrize("top", [0, 5])
def test_log_probabilities_of_what_is_generated(cuda_dev, model, top):
    prompts = _ids(cuda_dev, 20, 33, 7)
    plain = model.generate(prompts, 4, page_size=8)
    said = model.generate(prompts, 4, page_size=8, logprobs=top)
    assert isinstance(said, Generated) and torch.equal(said.ids, plain)
    assert said.logprobs.shape == said.entropy.shape == (3, 4) and said.top_ids.shape == said.top_logprobs.shape == (3, 4, top)
    logits = (model.last_hidden @ model.lm_head.t()).cpu()
    want = OR.score(logits, plain[:, -1].cpu(), top)
    assert float((said.logprobs[:, -1].cpu() - want["logprobs"]).abs().max()) < 2.0**-16 and float((said.entropy[:, -1].cpu() - want["entropy"]).abs().max()) < 2.0**-14
    if top:
        assert torch.equal(said.top_logprobs[..., 0], said.logprobs)  # what is generated is the most likely
        assert torch.equal(said.top_ids[:, -1].cpu(), want["top_ids"])


def test_scores_of_given_prompts(cuda_dev, model, monkeypatch):
    prompts = _ids(cuda_dev, 20, 2, 33)
    calls = []
    real = ops.token_logprobs

    def noted(logits, tokens, *, top=0):
        calls.append((logits.clone(), tokens.clone()))
        return real(logits, tokens, top=top)

    monkeypatch.setattr(ops, "token_logprobs", noted)
    scores = model.score(prompts, top=3)
    assert [s.logprobs.shape[0] for s in scores] == [19, 1, 32] and scores[0].top_ids.shape == (19, 3)
    logits, tokens = (torch.cat(t) for t in zip(*calls))
    assert torch.equal(tokens, torch.cat([p[1:] for p in prompts]))
    want = OR.score(logits.cpu(), tokens.cpu(), 3)
    assert float((torch.cat([s.logprobs for s in scores]).cpu() - want["logprobs"]).abs().max()) < 2.0**-16
    assert torch.equal(torch.cat([s.top_ids for s in scores]).cpu(), want["top_ids"])
    # the only row of the second prompt sees itself alone, as a prompt of its first token does
    monkeypatch.undo()
    model.generate([prompts[1][:1]], 1)
    one = OR.score((model.last_hidden @ model.lm_head.t()).cpu(), prompts[1][1:].cpu(), 0)
    size = float((model.last_hidden @ model.lm_head.t()).abs().max())
    assert abs(float(scores[1].logprobs[0]) - float(one["logprobs"])) <= 4 * 2.0**-8 * size  # two products, each rounded to bf16, of the token and of the largest
    # alone and in a batch the same
    for p, s in zip(prompts, scores):
        assert abs(float((model.score([p])[0].logprobs - s.logprobs).abs().max())) <= 4 * 2.0**-8 * float(logits.abs().max())
    # in parts, the same
    whole = torch.cat([s.logprobs for s in scores])
    model.lm_head, kept = model.lm_head[:1500], model.lm_head
    low = [p % 1500 for p in prompts]
    short = torch.cat([s.logprobs for s in model.score(low)])
    model.lm_head = kept
    assert short.shape == whole.shape and bool((whole < 0).all())


def test_all_together(cuda_dev, model, monkeypatch):
    """A prefix, an adapter each, an e4m3 cache and log probabilities in one run."""
    prefix, *prompts = _ids(cuda_dev, 50, 20, 33, 1, 9, seed=6)
    pool = _pool(cuda_dev)
    run = lambda: model.generate(prompts, 5, page_size=16, cache_dtype=torch.float8_e4m3fn, prefix=prefix, adapters=pool, which=[2, -1, 0, 2], logprobs=4)  # noqa: E731
    said = run()
    ops.check_status(cuda_dev)
    checked = Checked(monkeypatch)
    assert all(torch.equal(a, b) for a, b in zip(said, run())), "two runs differ"
    assert checked.calls == dict(prefix=2 * 4, lora=5 * 2 * 7, score=5)
    assert said.ids.shape == (4, 5) and said.top_ids.shape == (4, 5, 4) and torch.equal(said.top_logprobs[..., 0], said.logprobs)


def test_refusals(cuda_dev, model):
    prefix, *prompts = _ids(cuda_dev, 10, 4, 6)
    pool = _pool(cuda_dev)
    cache = PagedKVCache(2, 2, 20, 2, 128, cuda_dev, page_size=4, pages=8)
    used = PagedKVCache(2, 2, 20, 2, 128, cuda_dev, page_size=4)
    used.share(3)
    for bad, match in ((dict(prefix=prefix[:0]), "prefix"), (dict(adapters=pool), "belong together"), (dict(which=[0, 1]), "belong together"),
                       (dict(adapters=pool, which=[0]), "every prompt"), (dict(adapters=pool, which=[0, 3]), "every prompt"), (dict(logprobs=33), "top"),
                       (dict(prefix=torch.cat([prefix] * 25)), "positions"), (dict(prefix=prefix, cache=cache), "out of pages"), (dict(cache=used), "empty cache")):  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            model.generate(prompts, 5, **bad)
    assert model.generate(prompts, 2, prefix=prefix, cache=cache).shape == (2, 2)
    for bad in (lambda: model.score([]), lambda: model.score([prefix[:1]]), lambda: model.score([prefix], adapters=pool), lambda: model.score([torch.cat([prefix] * 26)])):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("rows", [1, 7, 32])
def test_scores_in_parts(cuda_dev, model, monkeypatch, rows):
    """The head's logits a few rows at a time, whose bounds fall inside prompts: each part with its own tokens, and the answers in one piece."""
    prompts = _ids(cuda_dev, 20, 2, 33)
    whole, calls, real = model.score(prompts, top=3), [], ops.token_logprobs

    def noted(logits, tokens, *, top=0):
        calls.append((logits.clone(), tokens.clone()))
        return real(logits, tokens, top=top)

    monkeypatch.setattr(ops, "token_logprobs", noted)
    monkeypatch.setattr(decoder, "SCORE_LOGITS", rows * CFG["vocab"] + 5)
    parts = model.score(prompts, top=3)
    assert [c[0].shape[0] for c in calls] == [min(rows, 52 - i) for i in range(0, 52, rows)]
    logits, tokens = (torch.cat(t) for t in zip(*calls))
    assert torch.equal(tokens, torch.cat([p[1:] for p in prompts]))
    want = OR.score(logits.cpu(), tokens.cpu(), 3)
    at = 0
    for p, s, w in zip(prompts, parts, whole):
        here = slice(at, at := at + p.numel() - 1)
        assert all(x.shape == y.shape for x, y in zip(s, w))
        assert float((s.logprobs.cpu() - want["logprobs"][here]).abs().max()) < 2.0**-16 and float((s.entropy.cpu() - want["entropy"][here]).abs().max()) < 2.0**-14
        assert torch.equal(s.top_ids.cpu(), want["top_ids"][here]) and float((s.top_logprobs.cpu() - want["top_logprobs"][here]).abs().max()) < 2.0**-16
        # two products of one row, each rounded to bf16, of the token and of the largest
        assert float((s.logprobs - w.logprobs).abs().max()) <= 4 * 2.0**-8 * float(logits.abs().max())
