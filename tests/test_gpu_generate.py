"""Generation: the decoder over its paged cache against the same decoder run over the whole sequence at every step.

Both compute the same model; what differs is the attention's rounding (one token over pages against the library's attention of the
whole sequence) and, behind it, int8 codes that flip by one.  One part in 127 of a row's maximum for a few codes of a row leaves
the hidden state within a few per cent: two layers of the same model under two roundings differ by 4.4 %, and the bound is twice
that.  An e4m3 cache moves every key and value by up to 2^-4, which the weights average down: 0.25.
"""

import pytest
import torch

from fms_model_optimizer_b200 import ops
from fms_model_optimizer_b200.decoder import W8A8Decoder
from fms_model_optimizer_b200.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=2048, rope_theta=10000.0, batch=3, seq=256)


def _prompts(dev, lengths=(37, 1, 130)):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, CFG["vocab"], (n,), generator=g).to(dev) for n in lengths]


def _off(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("extra,cache_dtype,bound", [({}, torch.bfloat16, 0.09), ({}, torch.float8_e4m3fn, 0.25),
                                                     (dict(qk_norm=True, window=50, sinks=2), torch.bfloat16, 0.09)])  # fmt: skip
def test_generation_follows_the_whole_sequence(cuda_dev, extra, cache_dtype, bound):
    model = W8A8Decoder(dict(CFG, **extra), cuda_dev)
    prompts = _prompts(cuda_dev)
    out = model.generate(prompts, 6, cache_dtype=cache_dtype, page_size=16)
    hidden = model.last_hidden
    ops.check_status(cuda_dev)
    assert out.shape == (3, 6)
    for b, p in enumerate(prompts):
        whole = torch.cat([p, out[b, :-1]])[None]
        model.forward(whole)
        assert _off(hidden[b], model.last_hidden[0]) < bound, b
    # the same calls give the same ids
    assert torch.equal(out, model.generate(prompts, 6, cache_dtype=cache_dtype, page_size=16))


def test_sequences_of_a_batch_do_not_touch_each_other(cuda_dev):
    """With kernels whose results do not depend on the neighbours' rows, a prompt's ids are the same alone and in a batch."""
    model = W8A8Decoder(CFG, cuda_dev)
    prompts = _prompts(cuda_dev, (20, 33))
    both = model.generate(prompts, 4, page_size=8)
    again = model.generate(prompts[::-1], 4, page_size=8)
    assert torch.equal(both, again.flip(0))


def test_cache_hands_out_pages_and_takes_them_back(cuda_dev):
    cache = PagedKVCache(1, 2, 40, 2, 64, cuda_dev, page_size=8, pages=7)
    step = cache.prompts([9, 17])
    assert step.max_q == 17 and step.cu.tolist() == [0, 9, 26] and step.last.tolist() == [8, 25]
    assert step.positions.tolist() == list(range(9)) + list(range(17))
    assert len(set(step.slots.tolist())) == 26
    for b, first in ((0, 0), (1, 9)):
        for i in range(9):
            assert int(step.slots[first + i]) == int(cache.table[b, i // 8]) * 8 + i % 8
    with pytest.raises(RuntimeError, match="release"):
        cache.prompts([1, 1])
    for _ in range(7):
        step = cache.token()
    assert cache.lens.tolist() == [16, 24] == cache.host_lens and step.single
    before = cache.table.clone()
    cache.token()  # both start a page: all seven are in use
    assert cache.host_lens == [17, 25] and not torch.equal(before, cache.table)
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.reserve([25, 25])
    with pytest.raises(RuntimeError, match="does not fit"):
        cache.reserve([41, 1])
    cache.release(1)
    cache.reserve([32, 24])
    assert cache.lens.tolist() == [17, 0]
    with pytest.raises(RuntimeError, match="float8"):
        PagedKVCache(1, 1, 1, 1, 64, cuda_dev, dtype=torch.float32)


def test_refusals(cuda_dev):
    with pytest.raises(RuntimeError, match="fused surface"):
        W8A8Decoder(dict(CFG, qk_norm=True), cuda_dev, surface="modules")
    model = W8A8Decoder(CFG, cuda_dev, layers=1)
    p = _prompts(cuda_dev, (4,))
    for bad, match in ((lambda: model.generate([], 1), "at least one"), (lambda: model.generate(p, 0), "at least one"), (lambda: model.generate(p, 300), "positions"),
                       (lambda: model.generate(p, 2, cache=PagedKVCache(2, 1, 8, 2, 128, cuda_dev)), "another number")):  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            bad()
