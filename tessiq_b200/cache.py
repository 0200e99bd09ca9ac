"""A paged cache of keys and values in 8 bits: its memory, which sequence has which pages, and the calls of a serving step.

`Pages` keeps the books on the host (no GPU): pages are handed out, shared by forked sequences, copied when one of
them writes, taken back and moved together. `PagedCache` has the memory of all layers and makes the launches: `ops.cache_store`,
`ops.cache_attention` or `ops.prefix_attention`, and `ops.copy_pages`, on torch's current stream. `Beams` are rows whose books are on the device
(`ops.cache_advance`), for a search that goes on without the host. The reference has no cache; its models run whole
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

    search = cache.beams([a], 4, 64)                    # four rows that go on from a, up to 64 tokens each
    step = search.step(parents)                         # row r goes on from row parents[r] (None: each from itself), with one token more
    cache.store(step, layer, k, v); out = cache.attention(step, layer, q)       # all of it can be captured into a graph
    scores, parents, tokens = ops.beam_select(logits, scores, 4)
    best = search.keep(0); search.free()                # row 0 becomes a sequence like others

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

    def reserve(self, count: int) -> list[int]:
        """`count` pages that belong to no sequence yet; `drop` gives them back, and `compact` has to wait for that."""
        if count > len(self._free):
            raise MemoryError(f"{count} pages are needed and {len(self._free)} are free")
        return [self._take() for _ in range(count)]

    def drop(self, pages: Sequence[int]) -> None:
        for page in pages:
            self._drop(page)

    def adopt(self, pages: Sequence[int], length: int) -> int:
        """A sequence of `length` tokens on pages that others have (`reserve`, sequences), who keep their hold on them."""
        for page in pages:
            self.references[page] += 1
        return self._add(list(pages), length)

    def shared_tokens(self, sequences: Sequence[int]) -> int:
        """How many first tokens of all of `sequences` lie on the same pages."""
        rows = [self._of(sequence) for sequence in sequences]
        common = 0
        for pages in zip(*[pages for pages, _ in rows]):
            if len(set(pages)) > 1:
                break
            common += 1
        return min([common * self.page_tokens, *[length for _, length in rows]])

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
    shared: torch.Tensor | None = None      # int32 [runs]: how many first tokens the sequences of each of as many equal runs have in common
    together: bool = False   # whether these are enough to be worth reading once (see `worth_reading_once`)
    search: Beams | None = None      # whose step it is, and its number
    number: int = 0


def worth_reading_once(shared: Sequence[int], longest: int) -> bool:
    """Whether attention reads what runs of sequences share (tokens, of each run) once for all of a run, or with each sequence: it takes a launch or two more,
    and how the work is split is decided by the table's width, so that sequences with much of their own behind little that they share are slower. Measured
    (us, each alone / once, from cold caches, one run of 64 x 32/8 heads of 128, of 32 x 12 of 64, sixteen of 4 x 12 of 64): 512 tokens shared and 2048
    of their own 57 / 72, 33 / 33, 45 / 51; 2048 and 8192 176 / 182, 76 / 121, 131 / 119; 2048 and 2048 82 / 74, 39 / 47, 62 / 55; 8192 and 2048 176 / 84, 72 /
    55, 131 / 72."""
    return bool(shared) and max(shared) >= 128 and 3 * sum(shared) >= longest * len(shared)


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
        self._searches = 0       # `Beams` that have not been freed

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

    def extend(self, sequences: Sequence[int], tokens, runs: int | None = None) -> Step:
        """Room for `tokens` (one number, or one for each) tokens more in each of `sequences`; last pages that forks share are copied first. `runs`:
        the sequences are as many equal runs of neighbours that go back to a common beginning (forks of one prompt), whose attention reads
        what is still common to all of a run once, where that is a third of the sequences or more; None: each reads its own."""
        self._not_in_a_graph("extend")
        sequences = list(sequences)
        if runs is not None and (runs < 1 or len(sequences) % runs):
            raise ValueError(f"{len(sequences)} sequences are not {runs} equal runs")
        counts = [int(tokens)] * len(sequences) if isinstance(tokens, int) else [int(count) for count in tokens]
        starts = [self.books.length(sequence) for sequence in sequences]
        sources, targets = self.books.extend(sequences, counts)
        if sources:
            ops.copy_pages(self.tensors, sources, targets, page_axis=1)
        rows = [self.books.pages_of(sequence) for sequence in sequences]
        blocks = max([len(row) for row in rows], default=0)
        numbers = [page for row in rows for page in row + [0] * (blocks - len(row))]
        batch = len(sequences)
        each = len(sequences) // runs if runs else 0
        shared = [self.books.shared_tokens(sequences[r * each : (r + 1) * each]) for r in range(runs or 0)] if each else []
        together = worth_reading_once(shared, max([s + c for s, c in zip(starts, counts)], default=0))
        host = torch.tensor([*numbers, *starts, *counts, *[s + c for s, c in zip(starts, counts)], *shared], dtype=torch.int32)
        if self.k_scales.is_cuda:
            host = host.pin_memory()
        there = host.to(self.k_scales.device, non_blocking=True)
        table, starts, counts_there, lengths, shared = there.split([batch * blocks, batch, batch, batch, len(shared)])
        return Step(table.reshape(batch, blocks), starts, counts_there, lengths, max(counts, default=0), self.books.changes,
                    {sequence: self.books.changes_of(sequence) for sequence in sequences}, shared if each else None, together)

    def _good(self, step: Step, stores: bool) -> None:
        if step.search is not None and (step.search.cache is not self or step.search.steps != step.number):
            raise ValueError("the step of the beams is over: another one has been made since, or they have been freed")
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
        if step.shared is not None and step.together and window is None:
            return ops.prefix_attention(q, *self.layer(layer), step.table, step.lengths, step.shared, scale, token_major)
        return ops.cache_attention(q, *self.layer(layer), step.table, step.lengths, window, sinks, scale, token_major)

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers; how many moved. Steps from before must not be used again."""
        self._not_in_a_graph("compact")
        if self._searches:
            raise RuntimeError("beams have pages that only the device's books know: free them before compact")
        sources, targets = self.books.compact()
        if sources:
            ops.copy_pages(self.tensors, sources, targets, page_axis=1)
        return len(sources)

    def beams(self, sequences: Sequence[int], beams: int, tokens: int) -> Beams:
        """`beams` rows for each of `sequences`, which go on from it; see `Beams`."""
        return Beams(self, sequences, beams, tokens)


class Beams:
    """Rows that go on from some sequences, `beams` of them each, by up to `tokens` tokens, as a search's beams do: which pages each has is known to the device
    alone, and a step needs nothing of the host. A sequence's whole pages are all its rows' together; behind them the rows have pages that are set aside for
    them here, as many as they can ever need at once. The sequences may be extended, truncated or freed meanwhile; `compact` has to wait for `free`.

    `rows` of the batch: sequence s's beams are rows s * beams to (s + 1) * beams - 1. A step is good until the next one is made: its tensors are the
    search's own."""

    def __init__(self, cache: PagedCache, sequences: Sequence[int], beams: int, tokens: int):
        cache._not_in_a_graph("beams")
        sequences = list(sequences)
        if beams < 1 or tokens < 0 or not sequences:
            raise ValueError(f"no search of {beams} beams of {tokens} tokens for {len(sequences)} sequences")
        books, page = cache.books, cache.books.page_tokens
        lengths = [books.length(sequence) for sequence in sequences]
        blocks = max(1, *[-(-(length + tokens) // page) for length in lengths])
        self.reserved = books.reserve(sum(beams * (-(-(length + tokens) // page) - length // page) for length in lengths))
        self.held: list[int] = []                                         # (the rows' hold on the sequences' pages)
        try:
            self._begin(cache, sequences, beams, blocks, lengths)
        except BaseException:
            self._give_back(books)
            raise
        self.cache, self.beams, self.rows, self.tokens = cache, beams, beams * len(sequences), tokens
        self.steps = 0
        cache._searches += 1

    def _begin(self, cache: PagedCache, sequences: list[int], beams: int, blocks: int, lengths: list[int]) -> None:
        books, page = cache.books, cache.books.page_tokens
        for sequence in sequences:
            self.held.append(books.fork(sequence))
        references = [1] * len(books.references)                          # whatever is others' is never free, nor a row's alone
        for reserved in self.reserved:
            references[reserved] = 0
        table = []
        for sequence in self.held:
            pages = books.pages_of(sequence)
            for number in pages:
                references[number] += beams
            table += (pages + [0] * (blocks - len(pages))) * beams
        shared = [length // page * page for length in lengths]
        host = torch.tensor([*table, *[length for length in lengths for _ in range(beams)], *shared, *references], dtype=torch.int32)
        there = host.to(cache.k_scales.device)
        rows = beams * len(sequences)
        sizes = [rows * blocks, rows, len(sequences), len(references)]
        self.table, self.lengths, self.shared, self.references = (part.clone() for part in there.split(sizes))
        self.table = self.table.reshape(rows, blocks)
        self.together = worth_reading_once(shared, blocks * page)         # (the rows' own tokens as they may come to be)
        self._counts: dict[int, torch.Tensor] = {}

    def _give_back(self, books: Pages) -> None:
        for sequence in self.held:
            books.free(sequence)
        books.drop(self.reserved)

    def _alive(self) -> None:
        if self.cache is None:
            raise ValueError("the beams have been freed")

    def step(self, parents: torch.Tensor | None = None, count: int = 1) -> Step:
        """Row r goes on from row parents[r] (int32, any shape of `rows` elements, as `ops.beam_select` gives them; None: from itself) and gets room for `count`
        tokens more. parents[r] is one of the rows of r's own sequence: `attention` reads what these have in common once. Beyond `tokens` tokens (and what
        their last page has room for), or where kept sequences have taken the pages, the step is not made (`kernel.check_status` raises) and its stores
        write nothing."""
        self._alive()
        if count < 0:
            raise ValueError(f"a step of {count} tokens")
        if count not in self._counts:
            self.cache._not_in_a_graph("a count that no step before had")
            self._counts[count] = torch.full((self.rows,), count, dtype=torch.int32, device=self.lengths.device)
        if parents is not None:
            parents = parents.reshape(-1)
        cache = self.cache
        _, _, _, starts = ops.cache_advance(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, self.table, self.lengths, self.references,
                                            self._counts[count], parents, in_place=True)
        self.steps += 1
        return Step(self.table, starts, self._counts[count], self.lengths, count, cache.books.changes, {}, self.shared, self.together, self, self.steps)

    def keep(self, row: int) -> int:
        """Row `row` as a sequence of the cache, which `free` leaves. Waits for the device. The rows may go on: the sequence's pages are its own then, and
        not among those set aside for them any more."""
        self._alive()
        self.cache._not_in_a_graph("keep")
        if not 0 <= row < self.rows:
            raise ValueError(f"there is no row {row} among {self.rows}")
        length = int(self.lengths[row])
        pages = self.table[row, : -(-length // self.cache.books.page_tokens)].long()
        self.references[pages] += 1                                       # (rows that go on neither write into them nor hand them out again)
        return self.cache.books.adopt(pages.tolist(), length)

    def free(self) -> None:
        """Gives back what no kept sequence has."""
        self._alive()
        self._give_back(self.cache.books)
        self.cache._searches -= 1
        self.cache = None
