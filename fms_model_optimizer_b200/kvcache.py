"""A paged key-value cache for a decoder that generates: the pool of pages, the page table and the lengths that
``ops.qk_norm_rope`` writes with and ``ops.paged_attention`` reads with.

Sequences may share their first tokens (``share``): these have pages of their own, which ``ops.prefix_attention`` reads once for all sequences.

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
    keys: Optional[torch.Tensor] = None  # int64: the rows whose keys every sequence sees, one sequence behind the other; None: its own
    cu_k: Optional[torch.Tensor] = None  # int32 [sequences + 1], of `keys`


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
        self.prefix = 0  # tokens that all sequences share
        self._prefix_pages: List[int] = []
        self.prefix_table = self.prefix_lens = self.groups = None

    def layer(self, i: int) -> dict:
        """The keyword arguments of layer ``i`` for ``ops.qk_norm_rope`` (and, without the slots, ``ops.paged_attention``)."""
        return dict(k_pages=self.k[i], v_pages=self.v[i], k_scale=self.k_scale[i], v_scale=self.v_scale[i])

    def shared(self) -> dict:
        """The arguments of the shared prefix for ``ops.prefix_attention``."""
        return dict(prefix_table=self.prefix_table, prefix_lens=self.prefix_lens, groups=self.groups)

    def check(self, lengths: Sequence[int], prefix: Optional[int] = None) -> List[int]:
        """Refuses lengths that the cache cannot hold; otherwise the pages that every sequence still needs for them.  ``prefix``: as if so many tokens were still
        to be shared."""
        common = -(-prefix // self.page_size) if prefix is not None else 0
        first = (self.prefix if prefix is None else prefix) // self.page_size  # the page that a sequence's own tokens begin in
        need = [max(0, -(-int(n) // self.page_size) - first - len(own)) for n, own in zip(lengths, self._owned)]
        if any(n > self.max_len for n in lengths):
            raise RuntimeError(f"a sequence of {max(lengths)} tokens does not fit a cache of {self.max_len}")
        if sum(need) + common > len(self._free):
            raise RuntimeError(f"the cache is out of pages: {sum(need) + common} wanted, {len(self._free)} free")
        return need

    def share(self, tokens: int) -> Step:
        """Room for ``tokens`` >= 1 first tokens that all sequences have in common, in an empty cache: the step that writes them.  From then on ``prompts`` places a sequence's
        tokens behind them and its length counts them in; until then a sequence has length 0, and ``token`` passes it over."""
        if self.prefix or any(self.host_lens) or any(self._owned):
            raise RuntimeError("a prefix goes into an empty cache: release its sequences, and unshare, first")
        if not 1 <= tokens <= self.max_len:
            raise RuntimeError(f"a prefix of {tokens} tokens does not fit a cache of {self.max_len}")
        self.check([0] * self.batch, tokens)
        self.prefix = tokens
        self._runs = [False] * self.batch
        self._runs_dev.zero_()
        self._prefix_pages = [self._free.pop() for _ in range(-(-tokens // self.page_size))]
        positions, pages, lens, groups, last = self._send(range(tokens), self._prefix_pages, [tokens], [0, self.batch], [tokens - 1])
        self.prefix_table, self.prefix_lens, self.groups = pages.to(torch.int32)[None], lens.to(torch.int32), groups.to(torch.int32)
        slots = pages[positions // self.page_size] * self.page_size + positions % self.page_size
        cu = torch.cat([positions[:1], lens]).to(torch.int32)
        return Step(positions.to(torch.int32), slots, last, False, cu, tokens)

    def unshare(self) -> None:
        """The shared tokens are over: their pages go back to the pool.  All sequences have been released, and wait for prompts."""
        if any(self.host_lens) or any(self._owned):
            raise RuntimeError("sequences still have the shared tokens, or pages behind them: release them first")
        self._free += reversed(self._prefix_pages)
        self.prefix, self._prefix_pages = 0, []
        self.prefix_table = self.prefix_lens = self.groups = None

    def behind(self, shared: Step, step: Step) -> Step:
        """The step of ``share`` and that of the prompts behind it as one: the shared tokens, then the prompts, whose queries see the former's keys and their own."""
        n = self.prefix
        own = step.cu.diff().long()
        cu_k = torch.cat([step.cu[:1], (step.cu[1:] + n * torch.arange(1, own.numel() + 1, device=self.dev, dtype=torch.int32))])
        key = torch.arange(step.positions.numel() + n * own.numel(), device=self.dev)
        of = torch.searchsorted(cu_k[1:].contiguous(), key.to(torch.int32), right=True)  # the sequence of each key
        within = key - cu_k[of]
        keys = torch.where(within < n, within, n + step.cu[of] + within - n)
        first = torch.arange(n, device=self.dev)
        return Step(torch.cat([shared.positions, step.positions]), torch.cat([shared.slots, step.slots]), step.last + n, False, torch.cat([shared.cu, step.cu[1:] + n]),
                    max(shared.max_q, step.max_q), torch.cat([first, keys]), torch.cat([shared.cu, cu_k[1:] + n]))  # fmt: skip

    def reserve(self, lengths: Sequence[int]) -> None:
        """Hands out the pages for sequences of these lengths.  Refused as a whole where the pool does not hold them."""
        need = self.check(lengths)
        first = self.prefix // self.page_size
        rows, columns, pages = [], [], []
        for b, n in enumerate(need):
            rows += [b] * n
            columns += range(first + len(self._owned[b]), first + len(self._owned[b]) + n)
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
        """Room for prompts of ``lengths[i]`` >= 1 tokens (behind the shared ones, if there are any) in the empty sequences ``which[i]``, by default in all of them.  From then on
        ``token`` goes on with these and with those that have tokens already; other empty ones wait for a prompt of their own."""
        which = list(range(self.batch)) if which is None else [int(b) for b in which]
        if len(lengths) != len(which) or not which or min(lengths) < 1:
            raise RuntimeError("one prompt of at least one token for every sequence is wanted")
        if len(set(which)) != len(which) or min(which) < 0 or max(which) >= self.batch:
            raise RuntimeError(f"prompts go to different sequences of the {self.batch}")
        if any(self.host_lens[b] for b in which):
            raise RuntimeError("prompts start empty sequences: release them first")
        new = dict(zip(which, (self.prefix + int(n) for n in lengths)))
        self.reserve([new.get(b, 0) for b in range(self.batch)])
        n, rows = torch.tensor(lengths), torch.tensor(which)
        cu = torch.zeros(len(which) + 1, dtype=torch.int64)
        cu[1:] = n.cumsum(0)
        of = torch.repeat_interleave(torch.arange(len(which)), n)
        self.host_lens = [new.get(b, have) for b, have in enumerate(self.host_lens)]
        self._runs = [have > 0 for have in self.host_lens]
        positions, of, last, cu, lens, runs = self._send(torch.arange(int(cu[-1])) - cu[of] + self.prefix, rows[of], cu[1:] - 1, cu, self.host_lens, self._runs)
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
