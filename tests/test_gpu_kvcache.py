"""The paged cache in a running batch: the kernels on what ``PagedKVCache`` hands out, against every sequence's own history."""

import pytest
import torch

from fms_model_optimizer_b200 import ops
from fms_model_optimizer_b200.kvcache import PagedKVCache
from oracle import attention as OA

pytestmark = pytest.mark.gpu

HQ, HKV, DIM = 4, 2, 64


class _Batch:
    """A cache and, on the host, the keys and values of each of its sequences."""

    def __init__(self, dev, batch, pages):
        self.dev, self.g = dev, torch.Generator().manual_seed(21)
        self.cache = PagedKVCache(1, batch, 64, HKV, DIM, dev, page_size=8, pages=pages)
        self.k, self.v = ([torch.zeros(0, HKV, DIM, dtype=torch.bfloat16) for _ in range(batch)] for _ in range(2))
        self.cos, self.sin = torch.ones(64, DIM // 2, device=dev), torch.zeros(64, DIM // 2, device=dev)  # keys reach the cache as they are

    def write(self, step, of):
        """Random queries, keys and values into the step's slots; ``of[t]``: the sequence of row t, None where it does not run."""
        q, k, v = (torch.randn(len(of), h, DIM, generator=self.g).bfloat16() for h in (HQ, HKV, HKV))
        for t, b in enumerate(of):
            if b is not None:
                self.k[b], self.v[b] = torch.cat([self.k[b], k[t : t + 1]]), torch.cat([self.v[b], v[t : t + 1]])
        ops.qk_norm_rope(*(x.to(self.dev) for x in (q, k)), self.cos, self.sin, step.positions, v=v.to(self.dev), slots=step.slots, want_k=False, **self.cache.layer(0))
        return q

    def token(self):
        q = self.write(self.cache.token(), [b if self.k[b].shape[0] else None for b in range(self.cache.batch)])
        got = ops.paged_attention(q.to(self.dev), block_table=self.cache.table, lens=self.cache.lens, **self.cache.layer(0)).cpu()
        ops.check_status(self.dev)
        for b in range(self.cache.batch):
            for h in range(HKV):
                heads = slice(h * HQ // HKV, (h + 1) * HQ // HKV)
                # weights rounded to 16 bits, then the output; logits off by a few fp32 roundings
                want, weighted, size = OA.attend(q[b, heads], self.k[b][:, h], self.v[b][:, h], self.k[b].shape[0] - 1, 0, 0, DIM**-0.5)
                tol = (2 * 2.0**-8 + 2 * (DIM + 16) * 2.0**-23 * size[:, None] + 2.0**-20) * weighted + 1e-30
                assert bool(((got[b, heads].double() - want).abs() <= tol).all()), (b, h)

    def prompts(self, lengths, which):
        self.write(self.cache.prompts(lengths, which), [b for b, n in zip(which, lengths) for _ in range(n)])

    def release(self, b):
        self.cache.release(b)
        self.k[b], self.v[b] = self.k[b][:0], self.v[b][:0]


def test_sequences_end_and_others_take_their_place(cuda_dev):
    batch = _Batch(cuda_dev, 3, 9)
    batch.prompts([5, 17, 1], [0, 1, 2])
    for _ in range(4):
        batch.token()
    batch.release(1)
    for _ in range(3):
        batch.token()  # the released row gives zeros
    batch.prompts([20], [1])
    for _ in range(5):
        batch.token()
    batch.release(0)
    batch.release(2)
    with pytest.raises(RuntimeError, match="out of pages"):
        batch.cache.prompts([9, 30], [2, 0])  # four pages are held, six would be wanted
    batch.prompts([9, 12], [2, 0])
    for _ in range(3):
        batch.token()


def test_a_step_waits_for_nothing(cuda_dev):
    """Handing out pages, prompts and releases included, never blocks the host on the device's work."""
    cache = PagedKVCache(1, 3, 64, HKV, DIM, cuda_dev, page_size=4)
    cache.token()  # a first use of each operation may load its code
    torch.cuda.synchronize()
    for b in range(3):
        cache.release(b)
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        cache.prompts([3, 9, 4])
        for _ in range(6):  # a page starts in most of the steps, in two sequences at once in some
            step = cache.token()
        cache.release(1)
        cache.prompts([6], [1])
        cache.token()
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    assert cache.lens.tolist() == cache.host_lens == [10, 7, 11] and step.positions.tolist() == [8, 14, 9]
    for b, n in enumerate(cache.host_lens):
        assert cache.table[b, : -(-n // 4)].tolist() == cache._owned[b][: -(-n // 4)]


def test_what_is_sent_without_waiting_is_not_overwritten(cuda_dev):
    """Steps queued behind a long kernel: each one's pages and lengths arrive as they were when it was made."""
    cache = PagedKVCache(1, 4, 256, HKV, DIM, cuda_dev, page_size=1)
    cache.prompts([1, 2, 3, 4])
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    steps = [cache.token() for _ in range(100)]
    for i, step in enumerate(steps):
        assert step.positions.tolist() == [1 + i, 2 + i, 3 + i, 4 + i]
        assert step.slots.tolist() == [cache._owned[b][1 + b + i] for b in range(4)]


def test_generate_looks_at_a_given_cache_before_it_runs(cuda_dev):
    """A cache that cannot take the whole generation is refused before the prompts are computed, and left as it was."""
    from fms_model_optimizer_b200.decoder import W8A8Decoder

    cfg = dict(layers=1, hidden=256, q_heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=512, rope_theta=10000.0, batch=2, seq=64)
    model = W8A8Decoder(cfg, cuda_dev)
    prompts = [torch.arange(n, device=cuda_dev) for n in (5, 9)]
    make = lambda **kw: PagedKVCache(**{**dict(layers=1, batch=2, max_len=20, kv_heads=2, head_dim=64, dev=cuda_dev, page_size=8), **kw})  # noqa: E731
    ran = []
    model._forward_steps, steps = lambda *a: ran.append(1) or steps(*a), model._forward_steps
    busy = make()
    busy.prompts([3, 4])
    for cache, match in ((make(max_len=18), "20"), (make(pages=4), "pages"), (make(kv_heads=4), "heads"), (make(head_dim=128), "heads"), (make(dtype=torch.float16), "bfloat16"),
                         (make(layers=2), "another number"), (busy, "release")):  # fmt: skip
        before = list(cache.host_lens), len(cache._free)
        with pytest.raises(RuntimeError, match=match):
            model.generate(prompts, 12, cache=cache)
        assert not ran and (list(cache.host_lens), len(cache._free)) == before
    cache = make(pages=5)
    out = model.generate(prompts, 12, cache=cache)
    assert cache.host_lens == [16, 20] and torch.equal(out, model.generate(prompts, 12))
    for b in range(2):  # and once more in the same cache
        cache.release(b)
    assert torch.equal(out, model.generate(prompts, 12, cache=cache))


def test_a_prompt_alone_and_in_a_batch(cuda_dev):
    """The last hidden state behind a prompt, and behind five tokens that both runs read: what differs is the order of sums in the
    attention, split by the number of sequences, and the int8 codes that flip by one with it (two layers under two roundings differ by 4.4 %)."""
    from fms_model_optimizer_b200.decoder import W8A8Decoder

    cfg = dict(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=2048, rope_theta=10000.0, batch=3, seq=256)
    model = W8A8Decoder(cfg, cuda_dev)
    g = torch.Generator().manual_seed(22)
    prompts = [torch.randint(0, 2048, (n,), generator=g).to(cuda_dev) for n in (37, 1, 130)]

    def hidden(prompts, tail):
        cache = PagedKVCache(2, len(prompts), 256, 2, 128, cuda_dev, page_size=16)
        ids, step = torch.cat(prompts), cache.prompts([p.numel() for p in prompts])
        out = []
        for t in [*tail, None]:
            _, h = model._drive([model._forward_steps(ids, model._attend_cached(cache, step), step.last)])
            out.append(h.float())
            if t is not None:
                ids, step = t.to(cuda_dev), cache.token()
        return torch.stack(out)

    tail = [torch.randint(0, 2048, (3,), generator=g) for _ in range(5)]
    batch = hidden(prompts, tail)
    for b, p in enumerate(prompts):
        alone = hidden([p], [t[b : b + 1] for t in tail])[:, 0]
        assert bool(((alone - batch[:, b]).norm(dim=-1) < 0.09 * alone.norm(dim=-1)).all()), b


def test_generation_can_be_traced(cuda_dev):
    from fms_model_optimizer_b200.decoder import W8A8Decoder

    cfg = dict(layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=512, rope_theta=10000.0, batch=2, seq=64)
    model = W8A8Decoder(cfg, cuda_dev)
    prompts = [torch.arange(n, device=cuda_dev) for n in (5, 9)]
    want = model.generate(prompts, 3)
    model.trace = []
    assert torch.equal(model.generate(prompts, 3), want)
    rows = [t.shape[0] for tag, li, t in model.trace if tag == "attn" and li == 1]
    assert rows == [14, 2, 2] and len([1 for tag, li, _ in model.trace if tag == "k_rope" and li == 0]) == 1  # single tokens' keys go to the cache alone
