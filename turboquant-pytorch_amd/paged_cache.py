"""
Compressed KV cache in pages, for sequences of different lengths that are served together.

`V3Cache` holds one batch whose sequences are equally long.  `PagedV3Cache` holds any number of sequences in two pools: whole pages of packed
tokens, bit for bit what `V3Cache` packs, and uncompressed pages for the most recent `residual_window` tokens of a sequence and what fills up its next page.  A page is the
same page of every layer, so that a sequence has one table of pages, and copying or sharing a page is one copy or none.

A step gives sequences new tokens, one each (decoding) or many (chunks of prompts), mixed as they come:

    step = cache.step(seqs, counts)
    for layer in ...:
        step.append(keys, values, layer)            # [new tokens, kv heads, D], sequence after sequence
        out = step.attend(queries, layer)           # [new tokens, query heads, D], causal
    step.commit()                                   # pages that have become old enough are packed (or step.cancel(): the tokens are taken back)

The step's own tokens are attended to as they are; what is packed, and with which codec, is as in `V3Cache` (the reference's generation-time cache,
turboquant/generation_test_v2.py:48-165), but a page at a time.  Lengths and tables live on the host.
"""
from __future__ import annotations

import ctypes
import heapq
from array import array
from collections import Counter
from itertools import chain, groupby
from typing import Dict, Iterable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native
from .beams import beam_select
from .compressors_v3 import TurboQuantV3

_JOB = np.dtype([("states", np.uint64), ("idx_bytes", np.uint64), ("vec_norms", np.uint64), ("table", np.uint64), ("rows", np.int64), ("tokens", np.int64), ("row_stride", np.int64),
                 ("token_stride", np.int64), ("bits", np.int32), ("dtype", np.int32), ("packed_row_stride", np.int64)])
assert _JOB.itemsize == ctypes.sizeof(_native.TqJob)
MAX_JOBS = 4096                     # TQ_MAX_JOBS of include/tqamd.h


class _Pages:
    """Numbers of the pages of a pool: which are free, and how many sequences hold each of the others.  The lowest free one goes first.  A page keeps its number when it is moved into
    another pool: `places` has where it lies there (None: every page lies at its number)."""

    def __init__(self, count: int):
        self.free = list(range(count))
        self.held = array("i", bytes(4 * count))
        self.places: Optional[np.ndarray] = None

    def numbers(self) -> np.ndarray:
        """Of the pages that are held."""
        return np.flatnonzero(np.frombuffer(self.held, dtype=np.int32))

    def lie(self, pages: np.ndarray) -> np.ndarray:
        """Where pages lie."""
        return pages if self.places is None else self.places[pages]

    def gathered(self, numbers: np.ndarray, size: int) -> "_Pages":
        """What becomes of these pages in a pool of `size` that has the held ones (`numbers`) at its beginning."""
        new, n, known = _Pages(0), len(numbers), len(self.held)
        free = np.flatnonzero(np.frombuffer(self.held, dtype=np.int32) == 0)[:size - n]
        if len(free) < size - n:
            free = np.concatenate((free, np.arange(known, known + size - n - len(free))))
        new.free = free.tolist()
        new.held = self.held[:]
        new.held.extend([0] * (1 + max(numbers[-1] if n else 0, free[-1] if len(free) else 0) - known))
        if n and numbers[-1] != n - 1:
            new.places = np.zeros(len(new.held), dtype=np.int32)
            new.places[numbers] = np.arange(n, dtype=np.int32)
            new.places[free] = np.arange(n, size, dtype=np.int32)
        return new

    def take(self) -> int:
        page = heapq.heappop(self.free)
        self.held[page] = 1
        return page

    def drop(self, page: int) -> bool:
        self.held[page] -= 1
        if self.held[page]:
            return False
        heapq.heappush(self.free, page)
        return True

    def drop_all(self, pages: Iterable[int]) -> None:
        held, free = self.held, self.free
        for p in pages:
            n = held[p] - 1
            held[p] = n
            if not n:
                heapq.heappush(free, p)

    def hold_again(self, pages: Iterable[int]) -> None:
        """The reverse of drop_all, of pages that nobody has taken meanwhile."""
        held = self.held
        for p in pages:
            held[p] += 1
        self.free = [p for p in self.free if not held[p]]
        heapq.heapify(self.free)


class _Sequence:
    """Its pages, as int32 (a step joins the tables of all its sequences), and tokens."""
    __slots__ = ("pages", "plain", "total")

    def __init__(self, pages: array, plain: array, total: int):
        self.pages, self.plain, self.total = pages, plain, total


def _up(n: int) -> int:
    return -(-n // 256) * 256


class PagedV3Cache:
    """head_dim 64, 128, 256, or a multiple of 8 from 72 to 96 whose packed vectors are whole words; 2 to 8 bits.  pages, plain_pages: how many packed and uncompressed pages of
    page_tokens tokens (a power of two, 32 to 1024) the pools have, over all layers at once; a sequence needs a packed page for every page_tokens tokens
    and uncompressed ones for its window, a page that is being filled and the tokens of a step."""

    def __init__(self, head_dim: int, kv_heads: int, key_bits: int = 4, value_bits: int = 2, residual_window: int = 128, protected_layers: int = 0, n_layers: int = 36, *,
                 pages: int, plain_pages: int, page_tokens: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        for name, n, least in (("kv_heads", kv_heads, 1), ("n_layers", n_layers, 1), ("residual_window", residual_window, 0), ("pages", pages, 1), ("plain_pages", plain_pages, 1)):
            if isinstance(n, bool) or int(n) != n or n < least:
                raise ValueError(f"{name} must be a whole number, {least} or more; got {n!r}")
        if page_tokens not in (32, 64, 128, 256, 512, 1024):
            raise ValueError(f"page_tokens must be a power of two from 32 to 1024; got {page_tokens!r}")
        code = _native.dtype_code(dtype)
        self.head_dim, self.kv_heads, self.n_layers, self.residual_window, self.page_tokens = int(head_dim), int(kv_heads), int(n_layers), int(residual_window), page_tokens
        self.dtype = dtype
        dev = torch.device(device)
        if dev.type != "cuda":
            raise _native.TqError(f"a paged cache lives on a HIP device (got {dev}); this package has no CPU path")
        self._codecs = [TurboQuantV3(head_dim=head_dim, key_bits=key_bits, value_bits=value_bits, residual_window=0, layer_idx=i, n_layers=n_layers,
                                     protected_layers=protected_layers, seed=42, device="cpu") for i in range(n_layers)]
        for c in self._codecs:
            if not _native.lib().tq_paged_supported(head_dim, code, c.key_bits, c.value_bits):
                raise ValueError(f"no paged attention for head_dim {head_dim} at {c.key_bits} and {c.value_bits} bits: head_dim 64, 128, 256, or a multiple of 8 from 72 to 96 whose "
                                 "packed vectors are whole words, and 2 to 8 bits")
        self.device = dev if dev.index is not None else torch.device("cuda", torch.cuda.current_device())
        # a packed page: of every layer key codes, key norms, value codes, value norms
        H, P, at = self.kv_heads, page_tokens, 0
        self._parts = []
        for c in self._codecs:
            widths = [-(-head_dim // (8 // b)) for b in (c.key_bits, c.value_bits)]
            offsets = []
            for size in (H * P * widths[0], 2 * H * P, H * P * widths[1], 2 * H * P):
                offsets.append(at)
                at += _up(size)
            self._parts.append((*offsets, *widths))
        self._page_bytes, self._plain_shape = at, (self.n_layers, 2, H, P, self.head_dim)
        self._pool, self._plain = self._pools(pages, plain_pages)
        self._views = None
        self._layers: List[Optional[tuple]] = [None] * self.n_layers
        self._packed_pages, self._plain_pages = _Pages(pages), _Pages(plain_pages)
        self._packed_of: Dict[int, int] = {}         # uncompressed pages still held by others -> the packed page one of their sequences made of them
        self._seqs: Dict[int, _Sequence] = {}
        self._next = 0
        self._open: Optional[PagedStep] = None
        self._recorded: List[PagedStep] = []         # into graphs, and not over yet
        self._kept: List[torch.Tensor] = []          # tables of recorded steps that are over, which replays read

    def _pools(self, pages: int, plain_pages: int) -> Tuple[torch.Tensor, torch.Tensor]:
        return (torch.empty((pages, self._page_bytes), dtype=torch.uint8, device=self.device),
                torch.empty((plain_pages,) + self._plain_shape, dtype=self.dtype, device=self.device))

    # ---- what is there --------------------------------------------------------------------------------------------------------
    def codec(self, layer_idx: int) -> TurboQuantV3:
        """The layer's codec (the one `V3Cache` has for the same widths and layers)."""
        return self._codecs[layer_idx]

    def packed_pages(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """The layer's part of every packed page, views of the pool: key codes [pages, H, page_tokens, width], key norms [pages, H, page_tokens], and the same of values."""
        if self._views is None:              # (of this pool: `resize` makes another)
            H, P, n, row = self.kv_heads, self.page_tokens, self._pool.shape[0], self._page_bytes
            halves, views = self._pool.view(torch.float16), []
            # layers of equal widths follow one another at the same distance
            for (wk, wv), group in groupby(self._parts, key=lambda part: part[4:]):
                group = list(group)
                (k, kn, v, vn), many = group[0][:4], len(group)
                apart = group[1][0] - k if many > 1 else 0
                codes = lambda at, w: self._pool.as_strided((many, n, H, P, w), (apart, row, P * w, w, 1), at).unbind(0)  # noqa: E731
                norms = lambda at: halves.as_strided((many, n, H, P), (apart // 2, row // 2, P, 1), at // 2).unbind(0)  # noqa: E731
                views += zip(codes(k, wk), norms(kn), codes(v, wv), norms(vn))
            self._views = views
        return self._views[layer_idx]

    def plain_pages(self) -> torch.Tensor:
        """The uncompressed pool, [pages, layers, keys and values, H, page_tokens, D]."""
        return self._plain

    def tables(self, seq: int) -> Tuple[List[int], List[int]]:
        """Numbers of a sequence's packed and uncompressed pages, in the order of its tokens."""
        s = self._sequence(seq)
        return tuple(pool.lie(np.array(of, dtype=np.int32)).tolist() for pool, of in ((self._packed_pages, s.pages), (self._plain_pages, s.plain)))

    def lengths(self, seqs: Sequence[int]) -> List[int]:
        """Tokens of sequences, those of an open step among them."""
        return [self._sequence(s).total for s in seqs]

    def free_pages(self) -> Tuple[int, int]:
        """How many packed and uncompressed pages no sequence holds."""
        return len(self._packed_pages.free), len(self._plain_pages.free)

    def stored_bytes(self) -> int:
        """Bytes of the pages that are held, packed and uncompressed."""
        used = [sum(map(bool, p.held)) for p in (self._packed_pages, self._plain_pages)]
        return used[0] * self._page_bytes + used[1] * int(np.prod(self._plain_shape)) * self._plain.element_size()

    def _layer(self, layer: int) -> tuple:
        """What an attention call needs of a layer, whatever the step: (address of a request with it, the codec's compressors, the request, their tables)."""
        kept, codec = self._layers[layer], self._codecs[layer]
        kc, vc = codec.key_compressor, codec.val_compressor
        if kept is not None and kept[1] is kc and kept[2] is vc:
            return kept
        tables = kc.table(self.device), vc.table(self.device)
        for t, comp in zip(tables, (kc, vc)):
            _native.check_table(t, self.head_dim, comp.bits)
        (k, kn, v, vn, _, _), plain, es = self._parts[layer], self._plain, self._plain.element_size()
        r = _native.TqPagedRequest(packed_pool=self._pool.data_ptr() + k, plain_pool=plain.data_ptr() + layer * plain.stride(1) * es, table_k=tables[0].data_ptr(), table_v=tables[1].data_ptr(),
                                   packed_page_stride=self._page_bytes, k_norms=kn - k, v_idx=v - k, v_norms=vn - k, plain_page_stride=plain.stride(0) * es, plain_values=plain.stride(2) * es,
                                   bits_k=kc.bits, bits_v=vc.bits)
        kept = self._layers[layer] = (ctypes.addressof(r), kc, vc, r, tables)
        return kept

    def _sequence(self, seq: int) -> _Sequence:
        s = self._seqs.get(seq)
        if s is None:
            raise ValueError(f"no sequence {seq!r} in this cache")
        return s

    def _states(self, seqs: Iterable[int]) -> List[_Sequence]:
        known = self._seqs
        try:
            return [known[s] for s in seqs]
        except (KeyError, TypeError):
            return [self._sequence(s) for s in seqs]         # (which says what is wrong)

    def _eager(self, what: str) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} reads and changes tables on the host: it cannot be recorded into a graph (`append` and `attend` of a step made before can)")

    # ---- sequences come, continue more than once, and go --------------------------------------------------------------------------
    def add(self, count: int = 1) -> List[int]:
        """New, empty sequences."""
        if isinstance(count, bool) or int(count) != count or count < 0:
            raise ValueError(f"count must be a whole number, 0 or more; got {count!r}")
        new = list(range(self._next, self._next + int(count)))
        self._next += int(count)
        for s in new:
            self._seqs[s] = _Sequence(array("i"), array("i"), 0)
        return new

    def place(self, seqs: Sequence[int], packed: Sequence[int], plain: Sequence[int]) -> None:
        """Pages for sequences that are empty so far, `packed` (whole pages) and `plain` tokens, whose contents the caller writes (`packed_pages`, `plain_pages`, `tables`): stores
        that come from elsewhere."""
        self._settle()
        states = self._states(seqs)
        if not len(states) == len(packed) == len(plain) or len(set(seqs)) != len(states):
            raise ValueError("place: one number of packed and one of plain tokens for each of different sequences")
        if any(s.total for s in states) or any(p < 0 or p % self.page_tokens for p in packed) or any(n < 0 for n in plain):
            raise ValueError(f"place: sequences must be empty, packed tokens a multiple of {self.page_tokens}")
        self._room("place", sum(p // self.page_tokens for p in packed), sum(-(-n // self.page_tokens) for n in plain))
        for s, p, n in zip(states, packed, plain):
            s.pages.extend(self._packed_pages.take() for _ in range(p // self.page_tokens))
            s.plain.extend(self._plain_pages.take() for _ in range(-(-n // self.page_tokens)))
            s.total = int(p) + int(n)

    def _room(self, what: str, packed: int, plain: int) -> None:
        free = self.free_pages()
        if packed > free[0] or plain > free[1]:
            raise _native.TqError(f"{what} needs {packed} packed and {plain} uncompressed pages, {free[0]} and {free[1]} are free (free sequences, or `resize`)")

    def _drop(self, gone: Sequence[_Sequence]) -> None:
        """Sequences' pages are theirs no longer."""
        self._packed_pages.drop_all(chain.from_iterable([s.pages for s in gone]))
        self._plain_pages.drop_all(chain.from_iterable([s.plain for s in gone]))

    def _undrop(self, states: Sequence[_Sequence]) -> None:
        self._packed_pages.hold_again(chain.from_iterable([s.pages for s in states]))
        self._plain_pages.hold_again(chain.from_iterable([s.plain for s in states]))

    def _forget(self) -> None:
        """Of which pages it is known what they were packed into: those that are still held, as what they became is."""
        if self._packed_of:
            plain, packed = self._plain_pages.held, self._packed_pages.held
            self._packed_of = {p: q for p, q in self._packed_of.items() if plain[p] and packed[q]}

    def _settle(self) -> None:
        """An open step is committed before tables change, and what graphs have recorded of steps works on the pages no longer."""
        if self._open is not None:
            self._open.commit()
        if self._recorded:
            self._eager("a call that changes tables")
            for step in self._recorded:
                step._end()
            self._recorded.clear()

    def free(self, seqs: Sequence[int]) -> None:
        """Sequences end; pages that no other one holds are free."""
        self._settle()
        if len(set(seqs)) != len(seqs):
            raise ValueError("free: a sequence ends once")
        gone = self._states(seqs)
        for seq in seqs:
            del self._seqs[seq]
        self._drop(gone)
        self._forget()

    def _share(self, states: Sequence[_Sequence]) -> List[_Sequence]:
        """Sequences that continue as `states` are, with the same pages."""
        for pool, lists in ((self._packed_pages, [s.pages for s in states]), (self._plain_pages, [s.plain for s in states])):
            held = pool.held
            for p in chain.from_iterable(lists):
                held[p] += 1
        return [_Sequence(s.pages[:], s.plain[:], s.total) for s in states]

    def _copy_last(self, sharing: Sequence[_Sequence]) -> None:
        """The page that is being filled becomes a sequence's own, where it has been shared so far."""
        P, vector, pool = self.page_tokens, self.head_dim * self._plain.element_size(), self._plain_pages
        sources: List[int] = []
        targets: List[int] = []
        sizes: List[int] = []
        held, free, take = pool.held, pool.free, heapq.heappop
        for s in sharing:
            filled = s.total % P
            if filled:
                page = s.plain[-1]
                s.plain[-1] = target = take(free)
                held[target] = 1
                held[page] -= 1                  # (its owner still holds it)
                sources.append(page)
                targets.append(target)
                sizes.append(filled * vector)
        if sources:
            if pool.places is not None:
                sources, targets = (pool.places[pages].tolist() for pages in (sources, targets))
            _native.copy_pages(self._plain, self._plain, self.n_layers * 2 * self.kv_heads, P * vector, sources, targets, sizes)

    def fork(self, seqs: Sequence[int]) -> List[int]:
        """For each of `seqs` (one may be there more than once) a new sequence that begins as it is: whole pages are shared, one that is being filled is copied."""
        self._eager("fork")
        self._settle()
        states, P = self._states(seqs), self.page_tokens
        self._room("fork", 0, len([s for s in states if s.total % P]))
        fresh = self._share(states)
        try:
            self._copy_last(fresh)
        except BaseException:                # (tables stay as they were)
            self._drop(fresh)
            raise
        new = list(range(self._next, self._next + len(fresh)))
        self._next += len(fresh)
        self._seqs.update(zip(new, fresh))
        return new

    def reorder(self, seqs: Sequence[int], parents) -> None:
        """Sequence seqs[i] goes on from what seqs[parents[i]] is (beams that were chosen).  parents: whole numbers, a list or a tensor (which is waited for).
        Pages are shared; of several that go on from one, all but one get a copy of the page that is being filled."""
        self._eager("reorder")
        self._settle()
        states = self._states(seqs)
        if isinstance(parents, torch.Tensor):
            if parents.dtype.is_floating_point or parents.dtype == torch.bool:
                raise ValueError(f"reorder: parents must be whole numbers, got {parents.dtype}")
            parents = parents.flatten().tolist()
        parents = list(parents)
        if len(parents) != len(states) or len(set(seqs)) != len(states) or any(isinstance(p, bool) or int(p) != p or not 0 <= p < len(states) for p in parents):
            raise ValueError(f"reorder: for each of {len(states)} different sequences the place of one among them")
        # who takes over the page that is being filled: the sequence itself if it goes on, otherwise the first that goes on from it
        heir: Dict[int, int] = {}
        for i, p in enumerate(parents):
            if p not in heir or i == p:
                heir[p] = i
        twice = sum(1 for i, p in enumerate(parents) if heir[p] != i and states[p].total % self.page_tokens)
        if twice > len(self._plain_pages.free):
            # (pages that only sequences hold that end become free first)
            held = self._plain_pages.held
            ending = Counter(chain.from_iterable(s.plain for p, s in enumerate(states) if p not in heir))
            self._room("reorder", 0, twice - sum(1 for page, n in ending.items() if n == held[page]))
        fresh, known = self._share([states[p] for p in parents]), self._packed_of
        self._drop(states)
        self._forget()               # (before a page that has become free is taken again)
        try:
            self._copy_last([f for i, (f, p) in enumerate(zip(fresh, parents)) if heir[p] != i])
        except BaseException:                # (tables stay as they were; a copy that is refused has written nothing)
            self._drop(fresh)
            self._undrop(states)
            self._packed_of = known
            raise
        self._seqs.update(zip(seqs, fresh))

    def beam_step(self, seqs: Sequence[int], logits: torch.Tensor, scores: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """One step of beam search: of every group of beams (logits [groups, beams, vocabulary], scores [groups, beams]; seqs group after group) the `beams` best continuations,
        (scores, tokens, parents) [groups, beams] of `beam_select`, and the sequences reordered by them.  Waits for the parents."""
        if logits.dim() != 3 or len(seqs) != logits.shape[0] * logits.shape[1]:
            raise ValueError(f"beam_step: logits [groups, beams, vocabulary] for {len(seqs)} sequences, got {tuple(logits.shape)}")
        chosen = beam_select(logits, scores, logits.shape[1])
        first = torch.arange(logits.shape[0], device=chosen[2].device).unsqueeze(1) * logits.shape[1]
        self.reorder(seqs, chosen[2] + first)
        return chosen

    def resize(self, pages: Optional[int] = None, plain_pages: Optional[int] = None) -> None:
        """Pools of other sizes (default: just what is held, one page at least), into which the pages that are held are gathered (`tables` says where they lie then)."""
        self._eager("resize")
        self._settle()
        # (sequences' tables have numbers, which stay: what a gather costs the host does not depend on how many sequences there are)
        kept = self._packed_pages.numbers(), self._plain_pages.numbers()
        sizes = []
        for name, asked, n in zip(("pages", "plain_pages"), (pages, plain_pages), map(len, kept)):
            size = max(1, n) if asked is None else asked
            if isinstance(size, bool) or int(size) != size or size < max(1, n):
                raise ValueError(f"resize: {name} must be a whole number, {max(1, n)} or more (as many are held); got {size!r}")
            sizes.append(int(size))
        pool, plain = self._pools(*sizes)
        stream, vector = torch.cuda.current_stream(self.device), self.head_dim * self._plain.element_size()
        for source, target, of, numbers, rows, row_bytes in ((self._pool, pool, self._packed_pages, kept[0], 1, self._page_bytes),
                                                             (self._plain, plain, self._plain_pages, kept[1], self.n_layers * 2 * self.kv_heads, self.page_tokens * vector)):
            if len(numbers):
                _native.copy_pages(source, target, rows, row_bytes, of.lie(numbers).astype(np.int32))
            source.record_stream(stream)         # (what it was allocated on may be another one)
        self._pool, self._plain, self._views, self._layers = pool, plain, None, [None] * self.n_layers
        self._packed_pages, self._plain_pages = (of.gathered(numbers, size) for of, numbers, size in zip((self._packed_pages, self._plain_pages), kept, sizes))

    # ---- steps ----------------------------------------------------------------------------------------------------------------
    def step(self, seqs: Sequence[int], counts) -> "PagedStep":
        """Room for counts[i] new tokens (or `counts` each) of sequence seqs[i].  An open step is committed first."""
        self._eager("step")
        self._settle()
        seqs = list(seqs)
        states = self._states(seqs)
        counts = [counts] * len(seqs) if isinstance(counts, int) else list(counts)
        if len(counts) != len(seqs) or len(set(seqs)) != len(seqs) or any(isinstance(c, bool) or int(c) != c or c < 0 for c in counts):
            raise ValueError("step: for each of different sequences a whole number of new tokens, 0 or more")
        counts = [int(c) for c in counts]
        P = self.page_tokens
        need = [max(0, -(-(s.total - len(s.pages) * P + c) // P) - len(s.plain)) for s, c in zip(states, counts)]
        if any(s.total + c > 0x7fffffff - 65536 for s, c in zip(states, counts)):
            raise ValueError("step: a sequence of more than 2^31 tokens")
        self._room("step", 0, sum(need))
        self._open = PagedStep(self, seqs, states, counts, need)
        return self._open


class PagedStep:
    """New tokens of some sequences of a `PagedV3Cache`: `append` for every layer, `attend` where it is wanted, then `commit` (the next step or any other call that changes tables commits
    what is open).  Where a graph is recorded, the step has to be made before, and `attend` called once with the same window before the recording.  Replays work on the step's tokens until the step is taken
    back, or is committed and the cache's tables then change (the next step, place, fork, reorder, free, resize): from then on a replay does nothing, as the step's pages may be others'.  The tables
    that a graph reads, some numbers a page, are kept as long as the cache."""

    def __init__(self, cache: PagedV3Cache, seqs, states, counts, need):
        self.cache, self.seqs, self.counts = cache, seqs, counts
        self._states, self._pages_taken, self._begun = states, need, 0
        self.tokens = sum(counts)
        try:
            self._begin()
        except BaseException:                # (no memory for the tables: the sequences stay as they were)
            self._take_back()
            raise
        self._plans: Dict[Tuple[int, int], tuple] = {}
        self._ready: Dict[tuple, tuple] = {}
        self._quick: Dict[Optional[int], tuple] = {}         # window as it is asked for -> what the one-step call takes
        self._appended: set = set()
        self._done = False

    def _begin(self) -> None:
        """Pages for the new tokens, and the tables of all sequences onto the card."""
        cache, P = self.cache, self.cache.page_tokens
        records, packed, plain, singles, slots, at, packed_at, plain_at = [], [], [], [], [], 0, 0, 0
        rest = (0,) * (_native.PAGED_SEQ - 6)
        for s, c, n in zip(self._states, self.counts, self._pages_taken):
            held = len(s.pages)
            first = s.total - held * P
            if n:
                s.plain.extend([cache._plain_pages.take() for _ in range(n)])
            s.total += c
            self._begun += 1
            if c == 1:
                singles.append(s.plain[first // P] * P + first % P)
            elif c:
                places = np.arange(first, first + c)
                slots += [np.array(singles, dtype=np.int64), np.array(s.plain, dtype=np.int64)[places // P] * P + places % P]
                singles = []
            records += (at, c, s.total, held * P, packed_at, plain_at, *rest)
            packed.append(s.pages)
            plain.append(s.plain)
            packed_at += held
            plain_at += len(s.plain)
            at += c
        slots.append(np.array(singles, dtype=np.int64))
        self._records = np.array(records, dtype=np.int32).reshape(len(self.seqs), _native.PAGED_SEQ)
        self._records[:, 5] += packed_at     # (plain pages' numbers lie behind those of all packed ones)
        tables, slots = np.frombuffer(b"".join(packed + plain), dtype=np.int32), np.concatenate(slots)
        if cache._packed_pages.places is not None or cache._plain_pages.places is not None:
            tables = np.concatenate((cache._packed_pages.lie(tables[:packed_at]), cache._plain_pages.lie(tables[packed_at:])))
            slots = cache._plain_pages.lie(slots // P) * np.int64(P) + slots % P
        self._sections = [self._records.ravel(), tables, slots.astype(np.int32)]
        self._blob, (self._seq_at, self._table_at, self._slot_at) = self._upload(self._sections)

    def _take_back(self) -> None:
        for s, count, pages in zip(self._states[:self._begun], self.counts, self._pages_taken):
            s.total -= count
            if pages:
                self.cache._plain_pages.drop_all(s.plain[-pages:])
                del s.plain[-pages:]

    def _upload(self, sections: Sequence[np.ndarray]) -> Tuple[torch.Tensor, List[int]]:
        """Whole numbers onto the card, in one copy; addresses of the sections."""
        at, starts = 0, []
        for s in sections:
            starts.append(at)
            at += -(-max(s.size, 1) // 4) * 4
        host = torch.empty(at, dtype=torch.int32, pin_memory=True)
        flat = host.numpy()
        for s, lo in zip(sections, starts):
            flat[lo:lo + s.size] = s
        blob = host.to(self.cache.device, non_blocking=True)
        event = torch.cuda.Event()
        with torch.cuda.device(self.cache.device):
            event.record()
        stream = _native._stream_handle(self.cache.device)
        return (blob, event, stream), [blob.data_ptr() + 4 * lo for lo in starts]

    def _await(self, uploaded) -> None:
        """The upload is done before this stream goes on, and its memory stays while the stream reads it."""
        blob, event, stream = uploaded
        if torch.cuda.is_current_stream_capturing():
            if self not in self.cache._recorded:
                self.cache._recorded.append(self)        # (replays read its tables, whether the caller keeps it or not)
            return
        if _native._stream_handle(self.cache.device) != stream:
            current = torch.cuda.current_stream(self.cache.device)
            current.wait_event(event)
            blob.record_stream(current)

    def _end(self) -> None:
        """Replays of what was recorded of this step do nothing from here on: no token has a place, no item a sequence."""
        with _native._on(self.cache.device):
            for uploaded in (self._blob, *(plan[4] for plan in self._plans.values())):
                self._await(uploaded)
                uploaded[0].fill_(-1)
                self.cache._kept.append(uploaded[0])

    def _live(self, what: str) -> None:
        if self._done:
            raise RuntimeError(f"{what}: the step is committed")

    def _layer(self, layer_idx: int) -> int:
        if isinstance(layer_idx, bool) or int(layer_idx) != layer_idx or not 0 <= layer_idx < self.cache.n_layers:
            raise ValueError(f"layer_idx must be a whole number from 0 to {self.cache.n_layers - 1}, got {layer_idx!r}")
        return int(layer_idx)

    def append(self, keys: torch.Tensor, values: torch.Tensor, layer_idx: int) -> None:
        """The new tokens' keys and values of a layer, [new tokens, kv heads, D], sequence after sequence in the step's order."""
        if not self._done and type(layer_idx) is int and self.tokens and not torch.compiler.is_compiling():
            status = _native.fast().put_tokens(keys, values, self.cache._plain, layer_idx, self._slot_at, self.tokens, self._blob[2])
            if status is not None:
                _native.check(status, "tq_put_tokens")
                self._appended.add(layer_idx)
                return
        self._append(keys, values, layer_idx)

    @torch.compiler.disable
    @torch.no_grad()
    def _append(self, keys: torch.Tensor, values: torch.Tensor, layer_idx: int) -> None:
        """`append` with every check."""
        self._live("append")
        c, layer = self.cache, self._layer(layer_idx)
        shape = (self.tokens, c.kv_heads, c.head_dim)
        for name, t in (("keys", keys), ("values", values)):
            if tuple(t.shape) != shape or t.dtype != c.dtype:
                raise ValueError(f"append: {name} must be {list(shape)} {c.dtype}, got {tuple(t.shape)} {t.dtype}")
            if t.device != c.device:
                raise _native.TqError(f"append: {name} on {t.device}, the cache on {c.device}")
        if not self.tokens:
            self._appended.add(layer)
            return
        keys, values = (t if t.stride(2) == 1 and min(t.stride()) >= 0 else t.contiguous() for t in (keys, values))
        es = keys.element_size()
        with _native._on(c.device):
            self._await(self._blob)
            pool = c._plain[:, layer]
            _native.check(_native.lib().tq_put_tokens(keys.data_ptr(), values.data_ptr(), keys.stride(0) * es, keys.stride(1) * es, values.stride(0) * es, values.stride(1) * es,
                                                      pool.data_ptr(), pool.stride(0) * es, pool.stride(1) * es, self._slot_at, self.tokens, c.kv_heads, c.head_dim * es, c.page_tokens,
                                                      _native._stream_handle(c.device)), "tq_put_tokens")
        self._appended.add(layer)

    def _plan(self, group: int, window: int) -> tuple:
        """How the blocks of the attention share the step's work, on the card: (counts, items, merges, scratch)."""
        key = (group, window)
        plan = self._plans.get(key)
        if plan is None:
            self.cache._eager("the first attend of a step with this window")
            c, counts = self.cache, _native.TqPagedCounts()
            if None in c._layers:            # (all tables are on the card before a graph may be recorded)
                for i in range(c.n_layers):
                    c._layer(i)
            call = lambda items, merges: _native.lib().tq_paged_plan(  # noqa: E731
                self._records.ctypes.data, len(self.seqs), c.kv_heads, group, window, c.head_dim, _native.dtype_code(c.dtype), c.page_tokens, items.ctypes.data, len(items), merges.ctypes.data,
                len(merges), ctypes.byref(counts))
            items, merges = np.empty((1024, _native.PAGED_ITEM), np.int32), np.empty((256, _native.PAGED_MERGE), np.int32)
            with _native._on(c.device):
                rc = call(items, merges)
                if rc == _native.ERR_CAPACITY:
                    items = np.empty((counts.items + counts.blocks // _native.PAGED_ITEM + 1, _native.PAGED_ITEM), np.int32)
                    merges = np.empty((max(1, counts.merges), _native.PAGED_MERGE), np.int32)
                    rc = call(items, merges)
            _native.check(rc, "tq_paged_plan")
            floats = int(_native.lib().tq_paged_scratch(ctypes.byref(counts), c.kv_heads, c.head_dim))
            uploaded, (items_at, merges_at) = self._upload([items.ravel()[:counts.items * _native.PAGED_ITEM + (counts.blocks + 1 if counts.few else 0)], merges[:counts.merges].ravel()])
            plan = self._plans[key] = (counts, items_at, merges_at, floats, uploaded)
        return plan

    def _request(self, group: int, window: int) -> tuple:
        """What is the same in all layers: (request, scratch values, what its plan was uploaded as)."""
        ready = self._ready.get((group, window))
        if ready is None:
            counts, items_at, merges_at, floats, uploaded = self._plan(group, window)
            c = self.cache
            r = _native.TqPagedRequest(sequences=self._seq_at, tables=self._table_at, items=items_at, merges=merges_at, counts=counts, heads=c.kv_heads, group=group, sliding_window=window,
                                       page_tokens=c.page_tokens, head_dim=c.head_dim, dtype=_native.dtype_code(c.dtype))
            ready = self._ready[group, window] = (r, floats, uploaded)
        return ready

    def attend(self, queries: torch.Tensor, layer_idx: int, scale: Optional[float] = None, softcap: Optional[float] = None, slopes: Optional[torch.Tensor] = None,
               sliding_window: Optional[int] = None) -> torch.Tensor:
        """softmax(z) V of the new tokens' queries, [new tokens, query heads, D] -> the same shape and type: a new token sees everything its sequence holds before it and itself.
        Query head j uses kv head j // (query heads / kv heads).  z = scale * q . k (scale: D ** -0.5 by default), as softcap * tanh(z / softcap) if softcap (up to 1024 for 16-bit elements) is given, less
        slopes[query head] * distance if slopes (float [query heads]) are; sliding_window: only the last so many tokens, the new one among them, are seen.
        The layer has to be appended to before (the step's own tokens are read from its pages); of a step that no layer has been appended to, it is what the caller has written there itself.
        Not differentiable."""
        ready, appended = self._quick.get(sliding_window), self._appended
        if ready is not None and not self._done and type(layer_idx) is int and 0 <= layer_idx < self.cache.n_layers and (layer_idx in appended or not appended) and not torch.compiler.is_compiling():
            # as the call before with this window, if the queries are laid out for it
            out = _native.fast().paged_attend(ready[0], self.cache._layer(layer_idx)[0], queries, self.tokens, self.cache.head_dim ** -0.5 if scale is None else scale, softcap, slopes, ready[1], ready[2], ready[3])
            if out is not None:
                if type(out) is int:
                    _native.check(out, "tq_paged_attend")
                return out
        return self._attend(queries, layer_idx, scale, softcap, slopes, sliding_window)

    @torch.compiler.disable
    @torch.no_grad()
    def _attend(self, queries, layer_idx, scale, softcap, slopes, sliding_window) -> torch.Tensor:
        """`attend` with every check."""
        self._live("attend")
        c, layer = self.cache, self._layer(layer_idx)
        if self._appended and layer not in self._appended and self.tokens:
            raise RuntimeError(f"attend: layer {layer} has not been appended to in this step")
        if queries.dim() != 3 or queries.shape[0] != self.tokens or queries.shape[2] != c.head_dim or queries.shape[1] == 0 or queries.shape[1] % c.kv_heads or queries.dtype != c.dtype:
            raise ValueError(f"attend: queries must be [{self.tokens}, k * {c.kv_heads}, {c.head_dim}] {c.dtype}, got {tuple(queries.shape)} {queries.dtype}")
        if queries.device != c.device:
            raise _native.TqError(f"attend: queries on {queries.device}, the cache on {c.device}")
        heads, cap, window = queries.shape[1], 0.0, 0
        if softcap is not None:
            cap = float(softcap)
            if not 2.0 ** -100 <= cap <= (2.0 ** 100 if c.dtype == torch.float32 else 1024.0):         # (what a cap far above the logits leaves of them has too few bits there)
                raise ValueError(f"attend: softcap must be a number above zero, up to 1024 for 16-bit elements; got {softcap!r}")
        if sliding_window is not None:
            if isinstance(sliding_window, bool) or int(sliding_window) != sliding_window or sliding_window < 1:
                raise ValueError(f"attend: sliding_window must be a whole number, 1 or more; got {sliding_window!r}")
            window = min(int(sliding_window), 0x7fffffff)
        if slopes is not None:
            if tuple(slopes.shape) != (heads,) or not slopes.dtype.is_floating_point:
                raise ValueError(f"attend: slopes must be one float per query head, [{heads}]; got {tuple(slopes.shape)} {slopes.dtype}")
            if slopes.device != c.device:
                raise _native.TqError(f"attend: slopes on {slopes.device}, the cache on {c.device}")
            slopes = slopes.float().contiguous()
        with _native._on(c.device):
            out = torch.empty(queries.shape, dtype=c.dtype, device=c.device)
            if not self.tokens:
                return out
            # (16 bytes at a time: with other loads other kernels would do some of the work, and results differ in their last bits)
            es = queries.element_size()
            if queries.stride(2) != 1 or queries.data_ptr() % 16 or queries.stride(0) * es % 16 or queries.stride(1) * es % 16:
                queries = queries.clone(memory_format=torch.contiguous_format)
            request, floats, uploaded = self._request(heads // c.kv_heads, window)
            if uploaded[2] == self._blob[2]:
                self._quick[sliding_window] = (ctypes.addressof(request), floats, self._blob[0], uploaded[2])
            self._await(self._blob)
            self._await(uploaded)
            r, own = _native.TqPagedRequest.from_buffer_copy(request), c._layer(layer)[3]
            for name in ("packed_pool", "plain_pool", "table_k", "table_v", "packed_page_stride", "k_norms", "v_idx", "v_norms", "plain_page_stride", "plain_values", "bits_k", "bits_v"):
                setattr(r, name, getattr(own, name))
            r.queries, r.out = queries.data_ptr(), out.data_ptr()
            r.q_token, r.q_head = queries.stride(0), queries.stride(1)
            r.scale, r.softcap = c.head_dim ** -0.5 if scale is None else float(scale), cap
            r.slopes = None if slopes is None else slopes.data_ptr()
            # the call's own: its launches hand their sums on through it, and those of another thread on the stream may come in between
            scratch = torch.empty(floats, dtype=torch.float32, device=c.device) if floats else None
            _native.check(_native.lib().tq_paged_attend(ctypes.byref(r), None if scratch is None else scratch.data_ptr(), floats, _native._stream_handle(c.device)), "tq_paged_attend")
        return out

    @torch.no_grad()
    def commit(self) -> None:
        """The step is over: whole pages that lie before the last `residual_window` tokens are packed, all layers at once, and their uncompressed pages are free again.  Where packed pages
        run out, pages stay uncompressed until a later commit of their sequences finds some."""
        if self._done:
            return
        c = self.cache
        c._eager("commit")
        if self.tokens and len(self._appended) != c.n_layers:
            missing = sorted(set(range(c.n_layers)) - self._appended)
            raise RuntimeError(f"commit: layers {missing[:8]} have not been appended to in this step")
        becomes: Dict[int, int] = {}         # uncompressed page -> packed page, of those that are packed now
        moves: List[Tuple[_Sequence, List[int]]] = []
        for s in self._states:
            pages: List[int] = []
            for plain in s.plain[:max(0, (s.total - c.residual_window) // c.page_tokens - len(s.pages))]:
                packed = becomes.get(plain, c._packed_of.get(plain))
                if packed is None:
                    if not c._packed_pages.free:
                        break
                    packed = becomes[plain] = c._packed_pages.take()
                else:
                    c._packed_pages.held[packed] += 1
                pages.append(packed)
            if pages:
                moves.append((s, pages))
        try:
            if becomes:
                made = np.array(list(becomes.items()))
                self._pack(np.stack((c._plain_pages.lie(made[:, 0]), c._packed_pages.lie(made[:, 1])), 1).astype(np.uint64))
        except BaseException:                # (tables stay as they were)
            for _, pages in moves:
                c._packed_pages.drop_all(pages)
            raise
        c._packed_of.update(becomes)
        for s, pages in moves:
            c._plain_pages.drop_all(s.plain[:len(pages)])
            del s.plain[:len(pages)]
            s.pages.extend(pages)
        c._forget()
        self._done = True
        if c._open is self:
            c._open = None

    def cancel(self) -> None:
        """The step has not been: its tokens are taken back (what came in between, an error in a forward pass, leaves the sequences as they were)."""
        if self._done:
            return
        c = self.cache
        c._eager("cancel")
        self._take_back()
        self._done = True
        if c._open is self:
            c._open = None
        if self in c._recorded:
            c._recorded.remove(self)
            self._end()

    def _pack(self, made: np.ndarray) -> None:
        """Uncompressed pages into packed ones, of all layers: a job a page, layer and side; a launch a code width."""
        c = self.cache
        H, P, D, es, code = c.kv_heads, c.page_tokens, c.head_dim, c._plain.element_size(), _native.dtype_code(c.dtype)
        source = c._plain.data_ptr() + made[:, 0] * np.uint64(c._plain.stride(0) * es)
        target = c._pool.data_ptr() + made[:, 1] * np.uint64(c._page_bytes)
        by_bits: Dict[int, list] = {}
        for layer, (codec, parts) in enumerate(zip(c._codecs, c._parts)):
            for side, comp in enumerate((codec.key_compressor, codec.val_compressor)):
                jobs = np.zeros(len(made), dtype=_JOB)
                jobs["states"] = source + np.uint64((layer * 2 + side) * H * P * D * es)
                jobs["idx_bytes"], jobs["vec_norms"] = target + np.uint64(parts[2 * side]), target + np.uint64(parts[2 * side + 1])
                jobs["table"] = comp.table(c.device).data_ptr()
                jobs["rows"], jobs["tokens"], jobs["row_stride"], jobs["token_stride"] = 1, H * P, 0, D          # (a page's vectors follow one another)
                jobs["bits"], jobs["dtype"] = comp.bits, code
                by_bits.setdefault(comp.bits, []).append(jobs)
        with _native._on(c.device):
            for jobs in by_bits.values():
                jobs = np.concatenate(jobs)
                for lo in range(0, len(jobs), MAX_JOBS):
                    part = np.ascontiguousarray(jobs[lo:lo + MAX_JOBS])
                    host = torch.empty(part.nbytes, dtype=torch.uint8, pin_memory=True)
                    host.numpy()[:] = part.view(np.uint8)
                    dev = host.to(c.device, non_blocking=True)
                    _native.check(_native.lib().tq_compress_batched(part.ctypes.data, dev.data_ptr(), len(part), D, 0, _native._stream_handle(c.device)), "tq_compress_batched")
