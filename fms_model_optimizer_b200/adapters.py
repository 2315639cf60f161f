"""Low-rank adapters of a decoder whose Linears are quantized: a pool of them for every Linear of every layer, and the rows that each has in a step.

An adapter i adds ``scale[i] * (x a[i]^T) b[i]^T`` to the output of a Linear whose quantized weights all requests share; requests with different adapters, or none, run in one batch
(``ops.lora_add_``).  Which rows belong to which adapter is worked out once a step, for all Linears of all layers.  No counterpart in the reference, which leaves
adapters to the stack around it.
"""

from __future__ import annotations

from typing import Dict, Iterable, Optional, Sequence, Tuple

import torch

from . import ops


class LoraAdapters:
    def __init__(self, shapes: Dict[str, Tuple[int, int]], layers: int, adapters: int, rank: int, dev, dtype: torch.dtype = torch.bfloat16, names: Optional[Iterable[str]] = None):
        """``shapes``: name -> (out features, in features) of a layer's Linears; ``names``: those that have adapters, by default all.  ``rank`` is the largest rank of an adapter, up to 128;
        lower ones leave the rest zero, as all of them are at first.  ``scale`` (fp32 ``[adapters]``, ones at first) is the factor alpha / rank."""
        if not 1 <= rank <= 128 or adapters < 1 or layers < 1:
            raise RuntimeError("adapters have a rank of 1 to 128, and there is at least one, in at least one layer")
        if dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError("adapters are bfloat16 or float16")
        padded = -(-rank // 8) * 8
        self.adapters, self.rank, self.layers = adapters, rank, layers
        self.scale = torch.ones(adapters, device=dev)
        self.a, self.b = {}, {}
        for name in shapes if names is None else names:
            out, width = shapes[name]
            for li in range(layers):
                self.a[li, name] = torch.zeros(adapters, padded, width, dtype=dtype, device=dev)
                self.b[li, name] = torch.zeros(adapters, out, padded, dtype=dtype, device=dev)

    @torch.no_grad()
    def load(self, adapter: int, layer: int, name: str, a: torch.Tensor, b: torch.Tensor) -> None:
        """The weights of one adapter for one Linear: ``a [r, in]``, ``b [out, r]`` with ``r`` up to the pool's rank."""
        if not 0 <= adapter < self.adapters or (layer, name) not in self.a:
            raise RuntimeError(f"there is no adapter {adapter} for {name} in layer {layer}")
        pool_a, pool_b = self.a[layer, name][adapter], self.b[layer, name][adapter]
        r = a.shape[0] if a.dim() == 2 else 0
        if a.dim() != 2 or b.dim() != 2 or r > self.rank or a.shape[1] != pool_a.shape[1] or tuple(b.shape) != (pool_b.shape[0], r):
            raise RuntimeError(f"an adapter of {name} has weights [r, {pool_a.shape[1]}] and [{pool_b.shape[0]}, r], r up to {self.rank}")
        for pool, new in ((pool_a[:r], a), (pool_b[:, :r], b)):
            pool.copy_(new)
        pool_a[r:].zero_()
        pool_b[:, r:].zero_()

    def step(self, which: torch.Tensor) -> "LoraStep":
        """The rows of a step: ``which [rows]``, the adapter of each, negative for none."""
        return LoraStep(self, *ops.lora_groups(which, self.adapters))

    def which(self, of: Sequence[int], lengths: Sequence[int], dev, without: int = 0) -> torch.Tensor:
        """The adapter of each row of packed prompts, behind ``without`` rows that have none."""
        if len(of) != len(lengths) or any(not -1 <= int(i) < self.adapters for i in of):
            raise RuntimeError(f"every prompt has an adapter from 0 to {self.adapters - 1}, or -1 for none")
        rows = torch.repeat_interleave(torch.tensor([-1, *(int(i) for i in of)]), torch.tensor([without, *(int(n) for n in lengths)]))
        return rows.pin_memory().to(dev, non_blocking=True) if torch.device(dev).type == "cuda" else rows.to(dev)


class LoraStep:
    def __init__(self, adapters: LoraAdapters, rows: torch.Tensor, starts: torch.Tensor):
        self.adapters, self.rows, self.starts = adapters, rows, starts

    def add_(self, layer: int, name: str, y: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """Adds to ``y``, the output of this layer's Linear for ``x``, where it has adapters."""
        pool = self.adapters
        if (layer, name) not in pool.a:
            return y
        return ops.lora_add_(y, x, pool.a[layer, name], pool.b[layer, name], self.rows, self.starts, pool.scale)
