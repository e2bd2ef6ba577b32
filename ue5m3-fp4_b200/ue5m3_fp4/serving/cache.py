"""A paged key/value cache: the pages of every attention layer, and which of them belong to which
sequence.

The bookkeeping is on the host: a sequence's pages are taken from a free list as it grows and given
back when it is released.  What the kernels read of it (page table, lengths, row offsets) lies in
device tensors of fixed addresses that ``begin_step`` overwrites, so that a captured step can be
replayed with new contents.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor

from ue5m3_fp4.serving.operators import paged_attention


class PagedKVCache:
    """``pages`` pages of ``page_size`` keys and values per layer (bf16, uninitialised), shared by
    ``sequences`` slots of up to ``max_length`` keys each."""

    def __init__(self, *, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, sequences: int,
                 max_length: int, device: torch.device | str = "cuda") -> None:
        for name, value in (("layers", layers), ("pages", pages), ("kv_heads", kv_heads), ("sequences", sequences),
                            ("max_length", max_length)):
            if type(value) is not int or value <= 0:
                raise ValueError(f"{name} must be a positive integer")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64, 128 or 256")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        self.device = torch.device(device)
        self.page_size, self.sequences, self.max_length = page_size, sequences, max_length
        shape = (layers, pages, page_size, kv_heads, head_dim)
        self.k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        self.v = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        self._width = (max_length + page_size - 1) // page_size
        self._free = list(range(pages - 1, -1, -1))
        self._pages: list[list[int]] = [[] for _ in range(sequences)]
        self._lengths = [0] * sequences
        counts = (sequences * self._width, sequences, sequences + 1, sequences)
        self._words = torch.zeros(sum(counts), dtype=torch.int32, device=self.device)
        table, self.kv_lengths, self.query_starts, self.last_rows = self._words.split(counts)
        self.page_table = table.view(sequences, self._width)
        self.max_query_length = self.max_kv_length = 0
        self.step_tokens = 0  # of all slots, in the step that was begun last

    @property
    def lengths(self) -> tuple[int, ...]:
        """Keys per slot, those of the step that was begun last included."""

        return tuple(self._lengths)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def begin_step(self, new_tokens: Sequence[int]) -> None:
        """Make room for ``new_tokens[b]`` tokens of every slot b (0: none in this step), whose rows lie
        one slot behind the other in the step's tensors.  Raises without any change when a slot would
        pass ``max_length`` or the pages do not suffice."""

        new = [int(count) for count in new_tokens]
        if len(new) != self.sequences or any(count < 0 for count in new) or not any(new):
            raise ValueError("new_tokens must have one count per slot, none negative, at least one positive")
        lengths = [old + count for old, count in zip(self._lengths, new)]
        if max(lengths) > self.max_length:
            raise RuntimeError(f"a sequence would pass max_length = {self.max_length}")
        wanted = [(length + self.page_size - 1) // self.page_size - len(held) for length, held in zip(lengths, self._pages)]
        if sum(wanted) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, the step needs {sum(wanted)}")
        for held, count in zip(self._pages, wanted):
            held.extend(self._free.pop() for _ in range(count))
        self._lengths = lengths
        starts = [0]
        for count in new:
            starts.append(starts[-1] + count)
        self.max_query_length, self.max_kv_length, self.step_tokens = max(new), max(lengths), starts[-1]
        words = [page for held in self._pages for page in held + [-1] * (self._width - len(held))]
        # the last row of a slot without new tokens is immaterial, but a row
        words += lengths + starts + [max(stop - 1, 0) for stop in starts[1:]]
        host = torch.tensor(words, dtype=torch.int32)
        if self.device.type == "cuda":
            host = host.pin_memory()
        self._words.copy_(host, non_blocking=True)

    def release(self, slot: int) -> None:
        """End a slot's sequence and give its pages back."""

        if not 0 <= slot < self.sequences:
            raise IndexError("no such slot")
        self._free.extend(reversed(self._pages[slot]))
        self._pages[slot] = []
        self._lengths[slot] = 0

    def attend(self, layer: int, q: Tensor, k: Tensor, v: Tensor, *, scale: float | None = None) -> Tensor:
        """Write the step's keys and values [tokens, kv_heads, head_dim] of one layer and attend with its
        queries [tokens, heads, head_dim] (:func:`paged_attention`).  At least the tokens of the step, which come
        first; rows behind them are padding."""

        if self.max_query_length == 0:
            raise RuntimeError("begin_step has not been called")
        if q.shape[0] < self.step_tokens:
            raise ValueError(f"the step has {self.step_tokens} tokens, q has rows for {q.shape[0]}")
        return paged_attention(q, self.k[layer], self.v[layer], self.page_table, self.kv_lengths, self.query_starts,
                               max_query_length=self.max_query_length, max_kv_length=self.max_kv_length, scale=scale,
                               new_k=k, new_v=v)


__all__ = ["PagedKVCache"]
