"""A paged key-value cache for a decoder that generates: the pool of pages, the page table and the lengths that
``ops.qk_norm_rope`` writes with and ``ops.paged_attention`` reads with.

Every layer has its own pool ``[pages, kv heads, page size, head_dim]`` of keys and of values; all layers share one page table
``[batch, pages of a sequence]`` and one length for each sequence.  Pages are handed out as sequences grow and come back with
``release``; a released place stays out of the steps until ``prompts`` fills it again.  Tables, lengths, positions and slots live on
the device; the host keeps a copy of the lengths to hand out pages by, and what it sends goes through pinned memory, so that a step
waits for nothing.  No counterpart in the reference, which leaves generation to a serving stack.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch


@dataclass
class Step:
    """The tokens of one forward pass, packed sequence behind sequence."""

    positions: torch.Tensor  # int32 [tokens]
    slots: torch.Tensor  # int64 [tokens]; -1: the row of a sequence that does not run, which is not written
    last: torch.Tensor  # int64 [sequences]: row of every sequence's last token
    single: bool  # a row for every sequence of the cache, one new token for those that run
    cu: Optional[torch.Tensor] = None  # int32 [sequences + 1], prompts only
    max_q: int = 1


class PagedKVCache:
    def __init__(self, layers: int, batch: int, max_len: int, kv_heads: int, head_dim: int, dev, dtype: torch.dtype = torch.bfloat16, page_size: int = 64,
                 pages: Optional[int] = None):  # fmt: skip
        """``max_len``: the most tokens of a sequence.  ``pages``: size of the pool, by default enough for all sequences at full
        length.  ``dtype`` float8_e4m3fn holds codes with one fp32 scale per layer and kv head: ``k_scale[layer]`` and ``v_scale[layer]`` are ones until the caller sets them
        (largest magnitude / 448), before the first token is written."""
        if min(layers, batch, max_len, page_size) < 1:
            raise RuntimeError("layers, batch, max_len and page_size must be positive")
        if dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
            raise RuntimeError("the cache holds bfloat16, float16 or float8_e4m3fn")
        per = -(-max_len // page_size)
        pages = batch * per if pages is None else pages
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        f8 = dtype == torch.float8_e4m3fn
        self.k_scale = [torch.ones(kv_heads, device=dev) for _ in range(layers)] if f8 else [None] * layers
        self.v_scale = [torch.ones(kv_heads, device=dev) for _ in range(layers)] if f8 else [None] * layers
        self.dev, self.batch, self.max_len, self.page_size = torch.device(dev), batch, max_len, page_size
        self.table = torch.zeros(batch, per, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.host_lens = [0] * batch
        self._runs = [True] * batch
        self._runs_dev = torch.ones(batch, dtype=torch.int32, device=dev)
        self._owned: List[List[int]] = [[] for _ in range(batch)]
        self._free = list(range(pages - 1, -1, -1))

    def layer(self, i: int) -> dict:
        """The keyword arguments of layer ``i`` for ``ops.qk_norm_rope`` (and, without the slots, ``ops.paged_attention``)."""
        return dict(k_pages=self.k[i], v_pages=self.v[i], k_scale=self.k_scale[i], v_scale=self.v_scale[i])

    def check(self, lengths: Sequence[int]) -> List[int]:
        """Refuses lengths that the cache cannot hold; otherwise the pages that every sequence still needs for them."""
        need = [max(0, -(-int(n) // self.page_size) - len(own)) for n, own in zip(lengths, self._owned)]
        if any(n > self.max_len for n in lengths):
            raise RuntimeError(f"a sequence of {max(lengths)} tokens does not fit a cache of {self.max_len}")
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache is out of pages: {sum(need)} wanted, {len(self._free)} free")
        return need

    def reserve(self, lengths: Sequence[int]) -> None:
        """Hands out the pages for sequences of these lengths.  Refused as a whole where the pool does not hold them."""
        need = self.check(lengths)
        rows, columns, pages = [], [], []
        for b, n in enumerate(need):
            rows += [b] * n
            columns += range(len(self._owned[b]), len(self._owned[b]) + n)
            self._owned[b] += [self._free.pop() for _ in range(n)]
            pages += self._owned[b][len(self._owned[b]) - n :]
        if rows:
            rows, columns, pages = self._send(rows, columns, pages)
            self.table[rows, columns] = pages.to(torch.int32)

    def _send(self, *parts) -> List[torch.Tensor]:
        """Integers to the device as int64 tensors, in one copy that the host does not wait for.  PyTorch keeps the pinned memory until
        the copy has run."""
        parts = [torch.as_tensor(p, dtype=torch.int64) for p in parts]
        whole = torch.cat(parts)
        if self.dev.type == "cuda":
            whole = whole.pin_memory().to(self.dev, non_blocking=True)
        return list(whole.split([p.numel() for p in parts]))

    def release(self, b: int) -> None:
        """Sequence ``b`` is over: its pages go back to the pool, its length to 0, and ``token`` passes it over."""
        self._free += reversed(self._owned[b])
        self._owned[b] = []
        self.host_lens[b] = 0
        self.lens[b].zero_()
        self._runs[b] = False
        self._runs_dev[b].zero_()

    def _slots(self, which: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        page = self.table[which, positions // self.page_size].long()
        return page * self.page_size + positions % self.page_size

    def prompts(self, lengths: Sequence[int], which: Optional[Sequence[int]] = None) -> Step:
        """Room for prompts of ``lengths[i]`` >= 1 tokens in the empty sequences ``which[i]``, by default in all of them.  From then on
        ``token`` goes on with these and with those that have tokens already; other empty ones wait for a prompt of their own."""
        which = list(range(self.batch)) if which is None else [int(b) for b in which]
        if len(lengths) != len(which) or not which or min(lengths) < 1:
            raise RuntimeError("one prompt of at least one token for every sequence is wanted")
        if len(set(which)) != len(which) or min(which) < 0 or max(which) >= self.batch:
            raise RuntimeError(f"prompts go to different sequences of the {self.batch}")
        if any(self.host_lens[b] for b in which):
            raise RuntimeError("prompts start empty sequences: release them first")
        new = dict(zip(which, (int(n) for n in lengths)))
        self.reserve([new.get(b, 0) for b in range(self.batch)])
        n, rows = torch.tensor(lengths), torch.tensor(which)
        cu = torch.zeros(len(which) + 1, dtype=torch.int64)
        cu[1:] = n.cumsum(0)
        of = torch.repeat_interleave(torch.arange(len(which)), n)
        self.host_lens = [new.get(b, have) for b, have in enumerate(self.host_lens)]
        self._runs = [have > 0 for have in self.host_lens]
        positions, of, last, cu, lens, runs = self._send(torch.arange(int(cu[-1])) - cu[of], rows[of], cu[1:] - 1, cu, self.host_lens, self._runs)
        self.lens.copy_(lens)
        self._runs_dev.copy_(runs)
        return Step(positions.to(torch.int32), self._slots(of, positions), last, False, cu.to(torch.int32), int(n.max()))

    def token(self) -> Step:
        """Room for one more token of every sequence that runs."""
        grown = [n + 1 if runs else n for n, runs in zip(self.host_lens, self._runs)]
        self.reserve(grown)
        positions = self.lens.clone()
        every = torch.arange(self.batch, device=self.dev)
        slots = torch.where(self._runs_dev > 0, self._slots(every, positions.long()), -1)
        self.lens += self._runs_dev
        self.host_lens = grown
        return Step(positions, slots, every, True)
