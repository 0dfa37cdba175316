"""Generation of many sequences over one paged key-value cache on the device.

``PagedDecoder`` pairs a ``Decoder``, which consumes prompts, with a step program of ``export_paged``, which
consumes one token of every sequence at a time. The cache lies in the step program's input staging; a
sequence is a list of its pages (``PagePool``). Rows move on the device (``chroma_hip_cache_move``): a prompt's
from the decoder's cache, a step's new rows into their pages, the last page of a forked sequence when it is
first written to, live pages to the front of the cache. A step commits only after its program returned and its moves are
queued, in a section that defers SIGINT, so an interrupt or an error leaves the last committed state.

(No counterpart in the reference, whose decoder holds one sequence, chroma/_src/decoder.py:44-152.)
"""

from __future__ import annotations

import contextlib
import heapq
import threading
from typing import Any, Dict, Iterable, Iterator, List, Mapping, Optional, Sequence, Tuple

import numpy as np

from chroma_amd._src import host, native
from chroma_amd._src.decoder import SELECT_MAX_K, Decoder, _interrupts_deferred, _staging_mirror
from chroma_amd._src.dtypes import numpy_dtype
from chroma_amd._src.program import Program
from chroma_amd._src.rules import TokenRules, unread


class PagePool:
    """Which pages of a cache are used, and by how many sequences. The lowest free page is taken first."""

    def __init__(self, pages: int) -> None:
        self.references = np.zeros(pages, dtype=np.int64)
        self._free = list(range(pages))  # a heap

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self) -> int:
        if not self._free:
            raise RuntimeError("no free page in the cache")
        page = heapq.heappop(self._free)
        self.references[page] = 1
        return page

    def share(self, pages: Iterable[int]) -> None:
        for page in pages:
            self.references[page] += 1

    def release(self, pages: Iterable[int]) -> None:
        for page in pages:
            self.references[page] -= 1
            if self.references[page] == 0:
                heapq.heappush(self._free, page)

    def compaction(self) -> Dict[int, int]:
        """Where each live page above the number of live pages goes, among the free ones below it."""
        live = int((self.references > 0).sum())
        holes = sorted(page for page in self._free if page < live)
        return dict(zip((int(page) for page in np.flatnonzero(self.references) if page >= live), holes))

    def move(self, moves: Mapping[int, int]) -> None:
        for source, target in moves.items():
            self.references[target], self.references[source] = self.references[source], 0
        self._free = [int(page) for page in np.flatnonzero(self.references == 0)]


class PagedDecoder:
    """Sequences are named by integers that ``add`` and ``fork`` return. Calls are serialized by one lock."""

    def __init__(self, decoder: Decoder, step: Program) -> None:
        """``decoder`` (a ``Decoder`` of hip programs, made with the model's own sliding window, which the step program
        holds) consumes the prompts, at most its context long, and is reset by each; ``step`` is a compiled
        ``export_paged`` of the same model. Both are closed with the paged decoder."""
        if len(step.inputs) != 6 or len(step.outputs) != 3:
            raise ValueError(f"PagedDecoder step wants six inputs and three outputs, not {len(step.inputs)} and {len(step.outputs)}")
        cache, table = step.inputs[2], step.inputs[4]
        layers, pages, rows, heads, dim = cache["shape"] if len(cache["shape"]) == 5 else (0,) * 5
        slots, span = table["shape"] if len(table["shape"]) == 2 else (0, 0)
        prompts = decoder._models[1].inputs[2]
        # rows move by these extents, so every input and output must have them
        fresh = ([layers, slots, heads, dim], prompts["dtype"])
        wanted = [([slots], "int64"), ([slots], "float32"), *[([layers, pages, rows, heads, dim], prompts["dtype"])] * 2, ([slots, span], "int64"),
                  ([slots], "int64"), ([slots, decoder.vocab_size], step.outputs[0]["dtype"]), fresh, fresh]
        if [layers, heads, dim] != [prompts["shape"][0], *prompts["shape"][2:]] or \
                [(list(spec["shape"]), spec["dtype"]) for spec in (*step.inputs, *step.outputs)] != wanted:
            raise ValueError("PagedDecoder decoder and step were not exported from the same model")
        if not decoder.stats["cache_on_device"] or decoder.device != step.device:
            raise ValueError("PagedDecoder wants a decoder of hip programs on the step's device")
        self._decoder, self._step = decoder, step
        self._layers, self._page_rows = layers, rows
        self._row_bytes = heads * dim * numpy_dtype(cache["dtype"]).itemsize
        self._slots, self._span = slots, span
        self.vocab_size = decoder.vocab_size
        self._logit_dtype = numpy_dtype(step.outputs[0]["dtype"])
        self._pool = PagePool(pages)
        self._slot_of: Dict[int, int] = {}  # sequence -> its row of the step program
        self._pages: Dict[int, List[int]] = {}
        self._lengths: Dict[int, int] = {}
        self._next = 0
        self._args = _staging_mirror(step)
        self._lock = threading.RLock()
        self._closed = False
        for value in (value for value in self._args if value is not None):
            value.fill(0)
        self._args[4].fill(-1)
        with self._lock:
            step.native.clear_input(2)
            step.native.clear_input(3)

    # ------------------------------------------------------------------------------------ what there is
    @property
    def sequences(self) -> List[int]:
        return list(self._slot_of)

    @property
    def page_rows(self) -> int:
        return self._page_rows

    @property
    def free_pages(self) -> int:
        return self._pool.free

    def position(self, sequence: int) -> int:
        return self._lengths[self._known(sequence)]

    def pages(self, sequence: int) -> List[int]:
        """The pages that hold the sequence's rows, in order."""
        return list(self._pages[self._known(sequence)])

    def _known(self, sequence: int) -> int:
        if self._closed:
            raise RuntimeError("PagedDecoder is closed")
        if sequence not in self._slot_of:
            raise KeyError(f"no sequence {sequence}")
        return sequence

    # ------------------------------------------------------------------------------------ rows on the device
    def _cache(self) -> native.CacheRows:
        model = self._step.native
        rows = len(self._pool.references) * self._page_rows
        return native.CacheRows(keys=model.input_pointer(2), values=model.input_pointer(3), rows=rows, layer_pitch=rows * self._row_bytes)

    def _move(self, source: native.CacheRows, moves: Sequence[Tuple[int, int, int]]) -> None:
        if moves:
            self._step.native.cache_move(self._cache(), source, self._layers, self._row_bytes, np.array(moves, dtype=np.int64))

    @contextlib.contextmanager
    def _taking(self, count: int) -> Iterator[List[int]]:
        """``count`` pages from the pool, which go back to it if the block fails."""
        pages = [self._pool.take() for _ in range(count)]
        try:
            yield pages
        except BaseException:
            self._pool.release(pages)
            raise

    def _new_slot(self) -> int:
        used = set(self._slot_of.values())
        slot = next((slot for slot in range(self._slots) if slot not in used), None)
        if slot is None:
            raise RuntimeError(f"the step program holds {self._slots} sequences")
        return slot

    def _enter(self, slot: int, pages: List[int], length: int) -> int:
        sequence, self._next = self._next, self._next + 1
        self._slot_of[sequence], self._pages[sequence], self._lengths[sequence] = slot, pages, length
        self._set_row(sequence)
        return sequence

    def _set_row(self, sequence: int) -> None:
        row = self._args[4][self._slot_of[sequence]]
        row.fill(-1)
        row[: len(self._pages[sequence])] = self._pages[sequence]

    # ------------------------------------------------------------------------------------ sequences
    def add(self, tokens: Any) -> Tuple[int, np.ndarray]:
        """Consume a prompt; returns the new sequence and the logits [1, vocab] after the prompt's last token."""
        with self._lock, self._decoder._lock:  # the decoder's cache stays this prompt's until its rows have been taken
            if self._closed:
                raise RuntimeError("PagedDecoder is closed")
            count = len(tokens)
            if count > self._decoder.context or count > self._span * self._page_rows:
                raise ValueError(f"a prompt of {count} tokens; the decoder holds {self._decoder.context}, a sequence {self._span * self._page_rows}")
            slot, needed = self._new_slot(), -(-count // self._page_rows)
            if needed > self._pool.free:
                raise RuntimeError(f"a prompt of {count} tokens needs {needed} pages, {self._pool.free} are free")
            self._decoder.reset()
            logits = self._decoder.append(tokens)
            with _interrupts_deferred():
                # the prompt starts a fresh cache, so row i holds position i
                owner = self._decoder._models[self._decoder._state.owner].native
                owner.synchronize()  # its queued commits have landed
                rows = self._decoder.context
                source = native.CacheRows(keys=owner.input_pointer(2), values=owner.input_pointer(3), rows=rows, layer_pitch=rows * self._row_bytes)
                size = self._page_rows
                with self._taking(needed) as pages:
                    self._move(source, [(i * size, page * size, min(size, count - i * size)) for i, page in enumerate(pages)])
                    self._step.native.synchronize()  # before the decoder's next prompt overwrites the rows
                return self._enter(slot, pages, count), logits

    def fork(self, sequence: int) -> int:
        """A new sequence with the same rows: the pages are shared, and the last one is copied when either of
        the two first writes to it."""
        with self._lock:
            pages = list(self._pages[self._known(sequence)])
            slot = self._new_slot()
            with _interrupts_deferred():
                self._pool.share(pages)
                return self._enter(slot, pages, self._lengths[sequence])

    def free(self, sequence: int) -> None:
        """End a sequence; its pages that no other sequence shares are free again."""
        with self._lock:
            self._known(sequence)
            with _interrupts_deferred():
                self._pool.release(self._pages.pop(sequence))
                slot = self._slot_of.pop(sequence)
                del self._lengths[sequence]
                self._args[4][slot].fill(-1)

    def compact(self) -> int:
        """Bring the live pages to the front of the cache; returns how many moved."""
        with self._lock:
            if self._closed:
                raise RuntimeError("PagedDecoder is closed")
            moves = self._pool.compaction()
            with _interrupts_deferred():
                size = self._page_rows
                self._move(self._cache(), [(source * size, target * size, size) for source, target in moves.items()])
                self._pool.move(moves)
                for sequence, pages in self._pages.items():
                    self._pages[sequence] = [moves.get(page, page) for page in pages]
                    self._set_row(sequence)
            return len(moves)

    # ------------------------------------------------------------------------------------ steps
    def step(self, tokens: Mapping[int, int]) -> np.ndarray:
        """Consume one token of each named sequence ({sequence: token}); returns the logits [n, vocab] after
        them, in the mapping's order."""
        logits = host.empty((self._slots, self.vocab_size), self._logit_dtype)
        with self._lock:
            slots, _ = self._run(tokens, [logits, None, None], None, None)
            adjacent = slots == list(range(slots[0], slots[0] + len(slots)))
            return logits[slots[0] : slots[0] + len(slots)] if adjacent else logits[slots]

    def step_top(self, tokens: Mapping[int, int], k: int = 1, *, rules: Optional[Mapping[int, TokenRules]] = None) -> Tuple[np.ndarray, np.ndarray]:
        """``step`` that returns the ``k`` largest logits after each token and their ids (both [n, k]), chosen on
        the device by the rule of ``Decoder.append_top``; ``rules`` ({sequence: rules}) adjust a sequence's logits
        first."""
        if not isinstance(k, (int, np.integer)) or not 1 <= k <= min(self.vocab_size, SELECT_MAX_K):
            raise ValueError(f"k must be an integer from 1 to {min(self.vocab_size, SELECT_MAX_K)}, got {k!r}")
        with self._lock:
            slots, (values, ids) = self._run(tokens, [None, None, None], int(k), rules)
            return values[slots], ids[slots]

    def _run(self, tokens: Mapping[int, int], outputs: List[Optional[np.ndarray]], k: Optional[int],
             rules: Optional[Mapping[int, TokenRules]]) -> Tuple[List[int], Any]:
        if self._closed:
            raise RuntimeError("PagedDecoder is closed")
        if not tokens:
            raise ValueError("a step wants a token of at least one sequence")
        for sequence, token in tokens.items():
            self._known(sequence)
            if not isinstance(token, (int, np.integer)):
                raise TypeError(f"token ids must be integers, got {token!r}")
            if self._lengths[sequence] >= self._span * self._page_rows:
                raise ValueError(f"sequence {sequence} holds {self._lengths[sequence]} rows, all that the step program has pages for")
        for sequence in rules or ():
            if sequence not in tokens:
                raise KeyError(f"rules for sequence {sequence}, which has no token in this step")
        # a page for a row that begins one, or for a copy of a last page that other sequences share
        size = self._page_rows
        starts = [s for s in tokens if self._lengths[s] % size == 0]
        leaving: Dict[int, int] = {}
        copies = []
        for s in tokens:
            if self._lengths[s] % size:
                page = self._pages[s][-1]
                if self._pool.references[page] - leaving.get(page, 0) > 1:  # the last of its owners keeps it
                    leaving[page] = leaving.get(page, 0) + 1
                    copies.append(s)
        if len(starts) + len(copies) > self._pool.free:
            raise RuntimeError(f"the step needs {len(starts) + len(copies)} pages, {self._pool.free} are free")
        ids, positions, _, _, _, lengths = self._args
        ids.fill(0)
        positions.fill(0)
        lengths.fill(0)
        for sequence, token in tokens.items():
            slot = self._slot_of[sequence]
            ids[slot], positions[slot], lengths[slot] = token, self._lengths[sequence], self._lengths[sequence]
        selection = None
        if k is None:
            self._step.run_resident(self._args, outputs)
        elif rules:
            plain = TokenRules()
            by_slot = {self._slot_of[sequence]: rules.get(sequence, plain) for sequence in tokens}
            idle = unread(list(by_slot.values()))
            selection = self._step.run_top_resident(self._args, outputs, 0, k, [by_slot.get(slot, idle) for slot in range(self._slots)])
        else:
            selection = self._step.run_top_resident(self._args, outputs, 0, k)
        with _interrupts_deferred():
            with self._taking(len(copies) + len(starts)) as taken:
                pages = {s: self._pages[s][-1] for s in tokens} | dict(zip((*copies, *starts), taken))
                self._move(self._cache(), [(self._pages[s][-1] * size, pages[s] * size, self._lengths[s] % size) for s in copies])
                model = self._step.native
                fresh = native.CacheRows(keys=model.output_pointer(1), values=model.output_pointer(2), rows=self._slots,
                                         layer_pitch=self._slots * self._row_bytes)
                self._move(fresh, [(self._slot_of[s], pages[s] * size + self._lengths[s] % size, 1) for s in tokens])
            for sequence in copies:
                self._pool.release(self._pages[sequence][-1:])
                self._pages[sequence][-1] = pages[sequence]
            for sequence in starts:
                self._pages[sequence].append(pages[sequence])
            for sequence in tokens:
                self._lengths[sequence] += 1
                self._set_row(sequence)
        return [self._slot_of[s] for s in tokens], selection

    def close(self) -> None:
        with self._lock:
            self._closed = True
            self._decoder.close()
            self._step.close()

    def __enter__(self) -> "PagedDecoder":
        return self

    def __exit__(self, *exc: Any) -> None:
        self.close()
