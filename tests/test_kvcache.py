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


def test_a_shared_prefix_has_pages_of_its_own():
    cache = _cache(batch=3, max_len=40, page_size=8, pages=9)
    first = cache.share(19)  # three pages, the last one with room that nobody else's keys go into
    assert first.positions.tolist() == list(range(19)) and first.cu.tolist() == [0, 19] and first.last.tolist() == [18] and first.max_q == 19 and not first.single
    assert first.slots.tolist() == [int(cache.prefix_table[0, i // 8]) * 8 + i % 8 for i in range(19)]
    assert cache.prefix_lens.tolist() == [19] and cache.groups.tolist() == [0, 3]
    step = cache.prompts([4, 9, 1])
    assert cache.host_lens == [23, 28, 20] == cache.lens.tolist()
    assert step.positions.tolist() == [*range(19, 23), *range(19, 28), 19]
    assert step.slots.tolist() == [int(cache.table[b, i // 8]) * 8 + i % 8 for b, n in ((0, 4), (1, 9), (2, 1)) for i in range(19, 19 + n)]
    used = {s // 8 for s in first.slots.tolist()}
    assert len(used) == 3 and not used & {s // 8 for s in step.slots.tolist()} and len(set(step.slots.tolist())) == 14
    both = cache.behind(first, step)
    assert both.positions.tolist() == [*range(19), *range(19, 23), *range(19, 28), 19] and both.cu.tolist() == [0, 19, 23, 32, 33]
    assert both.cu_k.tolist() == [0, 19, 42, 70, 90] and both.last.tolist() == [22, 31, 32] and both.max_q == 19
    assert both.keys.tolist() == [*range(19), *range(19), *range(19, 23), *range(19), *range(23, 32), *range(19), 32]
    assert both.slots.tolist() == first.slots.tolist() + step.slots.tolist()
    one = cache.token()
    assert one.positions.tolist() == [23, 28, 20] and cache.lens.tolist() == [24, 29, 21]
    # 3 + 1 + 2 + 1 pages of nine: two are left, and the lengths count the prefix
    cache.reserve([32, 29, 32])
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.reserve([33, 29, 32])
    with pytest.raises(RuntimeError, match="does not fit"):
        cache.check([41, 1, 1])
    with pytest.raises(RuntimeError, match="release"):
        cache.unshare()
    with pytest.raises(RuntimeError, match="empty cache"):
        cache.share(1)
    cache.release(1)
    step = cache.prompts([2], [1])
    assert step.positions.tolist() == [19, 20] and cache.host_lens == [24, 21, 21]
    for b in range(3):
        cache.release(b)
    cache.unshare()
    assert cache.prefix == 0 and len(cache._free) == 9 and cache.prompts([40, 1, 8]).positions.tolist()[:2] == [0, 1]


def test_a_shared_prefix_that_does_not_fit_is_refused():
    cache = _cache(batch=2, max_len=40, page_size=8, pages=4)
    for bad in (0, 41, 33):
        with pytest.raises(RuntimeError, match="fit|out of pages"):
            cache.share(bad)
    assert cache.prefix == 0 and len(cache._free) == 4
    cache.check([20, 20], 16)  # two pages together, one each
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.check([20, 20], 17)
    cache.prompts([1, 1])
    with pytest.raises(RuntimeError, match="empty cache"):
        cache.share(4)


def test_places_wait_for_a_prompt_behind_the_shared_tokens():
    """Nobody runs between `share` and `prompts`: a step then writes nothing, and least of all over the shared keys."""
    cache = _cache(batch=2, max_len=40, page_size=4)
    first = cache.share(10)
    for _ in range(2):
        step = cache.token()
        assert step.slots.tolist() == [-1, -1] and cache.host_lens == [0, 0] == cache.lens.tolist() and cache._owned == [[], []]
    step = cache.prompts([2], [1])
    assert step.positions.tolist() == [10, 11] and cache.host_lens == [0, 12] == cache.lens.tolist()
    assert not {s // 4 for s in first.slots.tolist()} & {s // 4 for s in step.slots.tolist()}
    step = cache.token()
    assert step.positions.tolist() == [0, 12] and int(step.slots[0]) == -1 and int(step.slots[1]) == int(cache.table[1, 3]) * 4
    assert cache.host_lens == [0, 13] == cache.lens.tolist()
    cache.release(1)
    cache.unshare()
    # as after `release`: places wait for a prompt without shared tokens too
    assert cache.token().slots.tolist() == [-1, -1] and cache.prompts([3, 1]).positions.tolist() == [0, 1, 2, 0]


def test_pages_handed_out_ahead_are_where_they_were_meant():
    """`reserve` before `share`, or between `share` and `unshare`, hands out pages for other columns of the table than those that the tokens would then be looked for in."""
    cache = _cache(batch=2, max_len=40, page_size=8)
    cache.reserve([16, 9])
    with pytest.raises(RuntimeError, match="empty cache"):
        cache.share(19)
    for b in range(2):
        cache.release(b)
    cache.share(19)
    cache.reserve([30, 0])
    assert cache.prompts([11, 5]).slots.tolist() == [int(cache.table[b, i // 8]) * 8 + i % 8 for b, n in ((0, 11), (1, 5)) for i in range(19, 19 + n)]
    for b in range(2):
        cache.release(b)
    cache.reserve([30, 30])
    with pytest.raises(RuntimeError, match="release"):
        cache.unshare()
    for b in range(2):
        cache.release(b)
    cache.unshare()
    assert len(cache._free) == 10
