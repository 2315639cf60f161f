"""The paged cache's book-keeping on the CPU: pages, lengths and slots of sequences that end while others go on."""

import pytest
import torch

from fms_model_optimizer_b200.kvcache import PagedKVCache


def _cache(batch=2, max_len=40, page_size=8, pages=None, dev="cpu"):
    return PagedKVCache(1, batch, max_len, 2, 64, torch.device(dev), page_size=page_size, pages=pages)


def test_a_released_sequence_stays_out_of_the_steps():
    cache = _cache(batch=3, pages=6)
    cache.prompts([4, 9, 1])
    cache.release(1)
    for i in range(5):
        step = cache.token()
        assert cache.host_lens == [5 + i, 0, 2 + i] == cache.lens.tolist()
        assert step.positions.tolist() == [4 + i, 0, 1 + i] and int(step.slots[1]) == -1
        assert step.slots.tolist()[::2] == [int(cache.table[b, n // 8]) * 8 + n % 8 for b, n in ((0, 4 + i), (2, 1 + i))]
    # its pages are there for the others: 6 pages, of which sequence 2 holds one
    cache.reserve([40, 0, 6])
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.reserve([40, 1, 6])


def test_a_released_place_takes_another_prompt_while_the_others_go_on():
    cache = _cache(batch=3, pages=6)
    cache.prompts([4, 20, 1])
    cache.token()
    cache.release(1)
    cache.token()
    step = cache.prompts([11], [1])
    assert cache.host_lens == [6, 11, 3] == cache.lens.tolist()
    assert step.positions.tolist() == list(range(11)) and step.cu.tolist() == [0, 11] and step.last.tolist() == [10] and step.max_q == 11 and not step.single
    assert step.slots.tolist() == [int(cache.table[1, i // 8]) * 8 + i % 8 for i in range(11)]
    others = {int(cache.table[0, 0]), int(cache.table[2, 0])}
    assert not others & {s // 8 for s in step.slots.tolist()}
    cache.token()
    assert cache.host_lens == [7, 12, 4] == cache.lens.tolist()
    for bad, match in (([5], [0]), "release"), (([5], [3]), "sequences"), (([5, 5], [1, 1]), "sequences"), (([5], [1, 2]), "one prompt"):
        with pytest.raises(RuntimeError, match=match):
            cache.prompts(*bad)
    assert cache.host_lens == [7, 12, 4]


def test_places_that_never_had_a_prompt_wait_for_one():
    cache = _cache(batch=3)
    step = cache.prompts([3, 2], [2, 0])
    assert step.positions.tolist() == [0, 1, 2, 0, 1] and step.cu.tolist() == [0, 3, 5]
    assert [s // 8 for s in step.slots.tolist()] == [int(cache.table[2, 0])] * 3 + [int(cache.table[0, 0])] * 2
    step = cache.token()
    assert cache.host_lens == [3, 0, 4] == cache.lens.tolist() and int(step.slots[1]) == -1
    # a whole empty cache can start from its first token, as before
    cache = _cache()
    assert cache.token().positions.tolist() == [0, 0] and cache.lens.tolist() == [1, 1]
