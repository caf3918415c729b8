"""A paged key-value cache for the layers of a stack, and the bookkeeping of the sequences in it.

The pages of all layers are one tensor; every layer uses the same page numbers, so there is one page table.  Lengths and pages
are kept on the host, where sequences come and go, and copied to the device when they change: the attention operators read
them there.
"""
from __future__ import annotations

import torch


class PagedCache:
    """``num_pages`` pages of ``page_size`` tokens, shared by up to ``max_seqs`` sequences of up to ``max_pages`` pages.

    ``k(layer)`` and ``v(layer)`` are [num_pages, kv_heads, page_size, head_dim], ``page_table`` int32 [max_seqs, max_pages] and
    ``seq_lens`` int32 [max_seqs] what :mod:`attention` takes.  :meth:`extend` makes room for new tokens, :meth:`release`
    gives a sequence's pages back."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, num_pages: int, *, page_size: int = 64, max_seqs: int = 1,
                 max_pages: int | None = None, dtype: torch.dtype = torch.float16, device="cuda"):
        if dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError("dtype must be torch.float16 or torch.bfloat16")
        if head_dim not in (64, 128):
            raise RuntimeError("head_dim must be 64 or 128")
        if page_size < 16 or page_size & (page_size - 1):
            raise RuntimeError("page_size must be a power of two, 16 or more")
        if min(layers, kv_heads, num_pages, max_seqs) < 1:
            raise RuntimeError("layers, kv_heads, num_pages and max_seqs must be positive")
        self.layers, self.kv_heads, self.head_dim, self.page_size = layers, kv_heads, head_dim, page_size
        self.max_seqs, self.max_pages = max_seqs, num_pages if max_pages is None else max_pages
        if self.max_pages < 1:
            raise RuntimeError("max_pages must be positive")
        self.pages = torch.zeros((layers, 2, num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.device = self.pages.device  # ("cuda" alone is whichever device is current when it is used)
        self.page_table = torch.zeros((max_seqs, self.max_pages), dtype=torch.int32, device=self.device)
        self.seq_lens = torch.zeros((max_seqs,), dtype=torch.int32, device=self.device)
        self.lengths = [0] * max_seqs
        self._owned: list[list[int]] = [[] for _ in range(max_seqs)]
        self._free = list(range(num_pages - 1, -1, -1))

    def k(self, layer: int) -> torch.Tensor:
        return self.pages[layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.pages[layer, 1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, new, *, idle: bool = False) -> torch.Tensor | None:
        """Makes room for ``new[b]`` tokens at the end of every sequence and counts them in.  Returns the ``cu_seqlens`` of
        their rows, packed in the order of the sequences, or None when every sequence has one.  Raises without having
        changed anything when pages run out.

        ``idle``: sequences that have no tokens, such as those that :meth:`release` has ended, sit out a step of one token for each of the
        others (``new[b]`` is 0 for them, 1 for the others).  Returns None: every sequence has a row, which counts for nothing where
        the sequence is empty.  A captured step of single tokens so goes on while sequences come and go."""
        new = [int(n) for n in new]
        if len(new) != self.max_seqs or min(new) < 0:
            raise RuntimeError(f"new must be {self.max_seqs} numbers of tokens")
        if idle and any(n > 1 or (n == 0 and length > 0) for n, length in zip(new, self.lengths)):
            raise RuntimeError("with idle, new must be 1, or 0 for sequences without tokens")
        want = [-(-(length + n) // self.page_size) - len(own) for length, n, own in zip(self.lengths, new, self._owned)]
        if any(len(own) + w > self.max_pages for own, w in zip(self._owned, want)):
            raise RuntimeError(f"a sequence is longer than {self.max_pages} pages of {self.page_size} tokens")
        if sum(want) > len(self._free):
            raise RuntimeError(f"{sum(want)} pages are needed, {len(self._free)} are free")
        for b, w in enumerate(want):
            if w:
                at = len(self._owned[b])
                self._owned[b] += [self._free.pop() for _ in range(w)]
                self.page_table[b, at:at + w] = torch.tensor(self._owned[b][at:], dtype=torch.int32)
        self.lengths = [length + n for length, n in zip(self.lengths, new)]
        if all(n == 1 for n in new):
            self.seq_lens += 1
            return None
        self.seq_lens.copy_(torch.tensor(self.lengths, dtype=torch.int32))
        if idle:
            return None
        ends = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        return ends.to(self.device)

    def release(self, seq: int) -> None:
        """Ends sequence ``seq``: its pages are free, its length is 0."""
        if not 0 <= seq < self.max_seqs:
            raise RuntimeError(f"there is no sequence {seq}")
        self._free += reversed(self._owned[seq])
        self._owned[seq] = []
        self.lengths[seq] = 0
        self.seq_lens[seq] = 0
