"""A paged cache of keys and values in 8 bits: its memory, which sequence has which pages, and the calls of a serving step.

`Pages` keeps the books on the host (no GPU): pages are handed out, shared by forked sequences, copied when one of
them writes, taken back and moved together. `PagedCache` has the memory of all layers and makes the launches: `ops.cache_store`,
`ops.cache_attention` and `ops.copy_pages`, on torch's current stream. The reference has no cache; its models run whole
sequences (tests/python/test_models.py:64-67).

    cache = PagedCache(layers=12, kv_heads=12, width=64, pages=4096)
    a = cache.start()
    prompt = cache.extend([a], 37)                      # room for 37 tokens more, and where they go
    cache.store(prompt, layer, k, v)                    # k, v [1, kv_heads, 37, width], in every layer
    b = cache.fork(a)                                   # shares a's pages until either writes
    step = cache.extend([a, b], 1)
    cache.store(step, layer, k, v)
    out = cache.attention(step, layer, q, window=1024, sinks=4)
    cache.truncate(b, 30); cache.free(a); cache.compact()

Not for several host threads at once.
"""

from __future__ import annotations

import heapq
from dataclasses import dataclass, field
from typing import Sequence

import torch

from . import ops


class Pages:
    """Which sequence has which pages. A page is free, or belongs to as many sequences as `references` says; only a sequence's last page
    is ever written again, and only while it belongs to that sequence alone."""

    def __init__(self, pages: int, page_tokens: int):
        if pages < 0 or page_tokens < 1:
            raise ValueError(f"{pages} pages of {page_tokens} tokens")
        self.page_tokens = page_tokens
        self.references = [0] * pages
        self._free = list(range(pages))      # a heap: the lowest is handed out first
        self._sequences: dict[int, tuple[list[int], int]] = {}
        self._next = 0
        self.changes = 0                     # of all sequences together
        self._changes: dict[int, list[int]] = {}      # sequence -> [how often what was named as its own is not any more, ... was copied]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def sequences(self) -> list[int]:
        return list(self._sequences)

    def _of(self, sequence: int) -> tuple[list[int], int]:
        try:
            return self._sequences[sequence]
        except KeyError:
            raise KeyError(f"no sequence {sequence}") from None

    def length(self, sequence: int) -> int:
        return self._of(sequence)[1]

    def pages_of(self, sequence: int) -> list[int]:
        return list(self._of(sequence)[0])

    def _add(self, pages: list[int], length: int) -> int:
        sequence, self._next = self._next, self._next + 1
        self._sequences[sequence] = (pages, length)
        self._changes[sequence] = [0, 0]
        return sequence

    def _changed(self, sequence: int, which: int) -> None:
        self._changes[sequence][which] += 1
        self.changes += 1

    def changes_of(self, sequence: int) -> tuple[int, int]:
        """How often pages or tokens that were the sequence's stopped being its own (truncated, moved, its last page exchanged for a copy), and how often a
        copy was taken of a page it has."""
        self._of(sequence)
        moved, copied = self._changes[sequence]
        return moved, copied

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self.references[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self.references[page] -= 1
        if self.references[page] == 0:
            heapq.heappush(self._free, page)

    def start(self) -> int:
        return self._add([], 0)

    def fork(self, sequence: int) -> int:
        """A sequence with the same tokens, on the same pages."""
        pages, length = self._of(sequence)
        for page in pages:
            self.references[page] += 1
        return self._add(list(pages), length)

    def free(self, sequence: int) -> None:
        pages, _ = self._of(sequence)
        del self._sequences[sequence], self._changes[sequence]
        self.changes += 1
        for page in pages:
            self._drop(page)

    def truncate(self, sequence: int, length: int) -> None:
        """Forgets the tokens from `length` on (rejected drafts)."""
        pages, now = self._of(sequence)
        if not 0 <= length <= now:
            raise ValueError(f"sequence {sequence} has {now} tokens, not {length}")
        keep = -(-length // self.page_tokens)
        for page in pages[keep:]:
            self._drop(page)
        self._sequences[sequence] = (pages[:keep], length)
        if length < now:
            self._changed(sequence, 0)

    def extend(self, sequences: Sequence[int], counts: Sequence[int]) -> tuple[list[int], list[int]]:
        """Room for `counts` tokens more in each of `sequences`. Returns the pages to copy, (from, to): last pages that are shared and will be
        written. MemoryError, and nothing has changed, where the pages do not suffice."""
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence is extended twice in one call")
        if len(sequences) != len(counts) or any(count < 0 for count in counts):
            raise ValueError(f"{len(sequences)} sequences by {list(counts)} tokens")
        left = {}                            # references of shared last pages as the call goes on
        needed, copied = 0, []
        for sequence, count in zip(sequences, counts):
            pages, length = self._of(sequence)
            needed += -(-(length + count) // self.page_tokens) - len(pages)
            copies = False
            if count and length % self.page_tokens:
                shared = left.setdefault(pages[-1], self.references[pages[-1]])
                copies = shared > 1
                left[pages[-1]] = shared - 1 if copies else shared
            copied.append(copies)
        if needed + sum(copied) > len(self._free):
            raise MemoryError(f"{needed + sum(copied)} pages are needed and {len(self._free)} are free")
        sources, targets = [], []
        for sequence, count, copies in zip(sequences, counts, copied):
            pages, length = self._of(sequence)
            if copies:
                block = len(pages) - 1           # (forks have a page they share at the same place)
                for other, (theirs, _) in self._sequences.items():
                    if len(theirs) > block and theirs[block] == pages[block]:
                        self._changed(other, 0 if other == sequence else 1)
                sources.append(pages[-1])
                self._drop(pages[-1])
                pages[-1] = self._take()
                targets.append(pages[-1])
            length += count
            while len(pages) * self.page_tokens < length:
                pages.append(self._take())
            self._sequences[sequence] = (pages, length)
        return sources, targets

    def compact(self) -> tuple[list[int], list[int]]:
        """Gives the pages in use the lowest numbers. Returns the pages to copy, (from, to)."""
        used = len(self.references) - len(self._free)
        holes = sorted(page for page in self._free if page < used)
        high = [page for page in range(used, len(self.references)) if self.references[page]]
        moved = dict(zip(high, holes))
        for source, target in moved.items():
            self.references[target], self.references[source] = self.references[source], 0
        for sequence, (pages, length) in self._sequences.items():
            if any(page in moved for page in pages):
                self._sequences[sequence] = ([moved.get(page, page) for page in pages], length)
                self._changed(sequence, 0)
        self._free = list(range(used, len(self.references)))
        return list(moved), list(moved.values())


@dataclass
class Step:
    """Where the new tokens of some sequences go, on the device: what `ops.cache_store` and `ops.cache_attention` take. Good until pages move (`compact`),
    one of its sequences is truncated or freed, or its last page, shared with a fork, is exchanged for a copy as it is extended again; to store also until a
    fork takes such a copy, which would miss what is stored then. `PagedCache` refuses a step beyond that. Steps of a sequence are stored in the
    order they were made: tokens in a page behind those that are stored are not encoded again."""

    table: torch.Tensor      # int32 [batch, blocks]
    starts: torch.Tensor     # int32 [batch]
    counts: torch.Tensor
    lengths: torch.Tensor    # starts + counts
    tokens: int              # the largest count
    changes: int = 0         # the books' counts as the step was made (Pages.changes, Pages.changes_of each sequence)
    sequences: dict[int, tuple[int, int]] = field(default_factory=dict)


class PagedCache:
    """Keys and values of `layers` layers in e4m3, `pages` pages of `page_tokens` tokens each, with an f32 scale a page and head."""

    def __init__(self, layers: int, kv_heads: int, width: int, pages: int, page_tokens: int = 64, device="cuda"):
        if page_tokens not in (16, 32, 64, 128, 256, 512, 1024) or width not in range(16, 129, 16) or layers < 1 or kv_heads < 1 or pages < 1:
            raise ValueError(f"no cache of {layers} layers, {kv_heads} heads of {width}, {pages} pages of {page_tokens} tokens: a page has a power of two of tokens "
                             "from 16 to 1024, a head a multiple of 16 elements up to 128")
        shape = (layers, pages, kv_heads, page_tokens, width)
        self.k_pages, self.v_pages = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        self.k_scales, self.v_scales = (torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
        self.layers = layers
        self.books = Pages(pages, page_tokens)

    @property
    def tensors(self) -> list[torch.Tensor]:
        """[layers, pages, ...] each: codes of keys and values, their scales."""
        return [self.k_pages, self.v_pages, self.k_scales, self.v_scales]

    def layer(self, layer: int) -> tuple[torch.Tensor, ...]:
        """One layer's codes of keys and values and their scales, as the operators take them."""
        return self.k_pages[layer], self.v_pages[layer], self.k_scales[layer], self.v_scales[layer]

    def start(self) -> int:
        return self.books.start()

    def fork(self, sequence: int) -> int:
        return self.books.fork(sequence)

    def free(self, sequence: int) -> None:
        self.books.free(sequence)

    def truncate(self, sequence: int, length: int) -> None:
        self.books.truncate(sequence, length)

    def length(self, sequence: int) -> int:
        return self.books.length(sequence)

    def _not_in_a_graph(self, what: str) -> None:
        if self.k_scales.is_cuda and (torch.cuda.is_current_stream_capturing() or ops.lib.tq_is_recording()):
            raise RuntimeError(f"{what} keeps its books on the host and cannot go into a graph or a recording; storing and attention of a step can")

    def extend(self, sequences: Sequence[int], tokens) -> Step:
        """Room for `tokens` (one number, or one for each) tokens more in each of `sequences`; last pages that forks share are copied first."""
        self._not_in_a_graph("extend")
        sequences = list(sequences)
        counts = [int(tokens)] * len(sequences) if isinstance(tokens, int) else [int(count) for count in tokens]
        starts = [self.books.length(sequence) for sequence in sequences]
        sources, targets = self.books.extend(sequences, counts)
        if sources:
            ops.copy_pages(self.tensors, sources, targets, page_axis=1)
        rows = [self.books.pages_of(sequence) for sequence in sequences]
        blocks = max([len(row) for row in rows], default=0)
        numbers = [page for row in rows for page in row + [0] * (blocks - len(row))]
        batch = len(sequences)
        host = torch.tensor([*numbers, *starts, *counts, *[s + c for s, c in zip(starts, counts)]], dtype=torch.int32)
        if self.k_scales.is_cuda:
            host = host.pin_memory()
        there = host.to(self.k_scales.device, non_blocking=True)
        table, starts, counts_there, lengths = there.split([batch * blocks, batch, batch, batch])
        return Step(table.reshape(batch, blocks), starts, counts_there, lengths, max(counts, default=0), self.books.changes,
                    {sequence: self.books.changes_of(sequence) for sequence in sequences})

    def _good(self, step: Step, stores: bool) -> None:
        if step.changes == self.books.changes:
            return
        for sequence, (moved, copied) in step.sequences.items():
            if sequence not in self.books._sequences:
                raise ValueError(f"sequence {sequence} of the step has been freed")
            moved_now, copied_now = self.books.changes_of(sequence)
            if moved != moved_now:
                raise ValueError(f"the step is from before pages of sequence {sequence} were moved, truncated or exchanged for a copy")
            if stores and copied != copied_now:
                raise ValueError(f"a fork of sequence {sequence} has copied the page the step writes: what is stored now would be missing there")

    def store(self, step: Step, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Writes [batch, kv_heads, tokens, width] new keys and values of one layer; of a sequence that got fewer than `tokens`, the first ones."""
        self._good(step, True)
        if k.dim() == 4 and k.shape[2] < step.tokens:
            raise ValueError(f"the step has room for {step.tokens} tokens and was given {k.shape[2]}: attention would read what nobody wrote")
        ops.cache_store(k, v, *self.layer(layer), step.table, step.starts, step.counts)

    def attention(self, step: Step, layer: int, q: torch.Tensor, window=None, sinks=0, scale=None, token_major=True) -> torch.Tensor:
        """q [batch, heads, q_tokens, width] are the last `q_tokens` tokens of each sequence (a query before its first token gives zeros)."""
        self._good(step, False)
        return ops.cache_attention(q, *self.layer(layer), step.table, step.lengths, window, sinks, scale, token_major)

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers; how many moved. Steps from before must not be used again."""
        self._not_in_a_graph("compact")
        sources, targets = self.books.compact()
        if sources:
            ops.copy_pages(self.tensors, sources, targets, page_axis=1)
        return len(sources)
