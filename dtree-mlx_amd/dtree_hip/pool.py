"""Caches of several sequences over one pool of pages: forked, shared, freed.

``PagedKVPool`` holds the pages of a bf16 or an 8-bit cache and, for ``num_seqs``
sequences, their page tables and lengths. ``fork`` makes sequence i continue sequence
parents[i]: whole pages are shared by reference count, the page that is about to be
written is copied where others hold it too, pages that nobody holds are free again
(dtree_pages_fork, dtree_pages_copy). ``sequence(i)`` is one of them as the verify
engines take a cache.

``HypothesisCache`` is the decoding state of a batch of hypotheses that an engine
steps one token at a time (``beam.py``): an 8-bit pool and, for a hybrid, the
convolution windows and recurrent states of every sequence, held twice, since a step
reads those of the sequences that it continues and writes its own.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _native as N
from ._native import PAGE
from .cache import PagedKVCache, PagedKVCacheQ8


def _pages(positions: int) -> int:
    return (positions + PAGE - 1) // PAGE


class PagedKVPool:
    """k_pages, v_pages (and, in 8 bits, k_scales, v_scales) as PagedKVCache's and
    PagedKVCacheQ8's, ``num_pages`` of them, for ``num_seqs`` sequences of up to
    ``capacity`` positions. A bf16 pool keeps one more page, which stands behind every
    sequence's end in its table (its kernels read table entries there); an 8-bit
    pool's entries are -1 there.

    tables   two [num_seqs, pages] int32: a fork reads one and writes the other
    refs     [pages] int32: sequences that hold a page, 0 is free
    copies   [num_seqs, 3] int32, status [2] int32: dtree_pages_fork's
    lengths  the sequences' positions on the host, as the last fork left them or
             ``sequence(i).offset`` has moved them since

    A sequence may be written where its pages are its own (``sequence(i).room``, (first,
    end) positions): behind ``start`` on its first lengths[i], behind a fork on the rows
    asked for, from the page of the fork's length on. The engines refuse steps elsewhere.
    """

    def __init__(self, layers: int, kv_heads: int, head_dim: int, capacity: int, num_seqs: int,
                 num_pages: int | None = None, kv_bits: int = 16, device="cuda"):
        if kv_bits not in (8, 16):
            raise ValueError("kv_bits is 16 (bf16 cache) or 8 (int8 rows with one fp32 scale each)")
        if capacity < 1 or not 1 <= num_seqs <= 1024:
            raise ValueError("capacity must be positive, num_seqs in [1, 1024]")
        if head_dim not in (64, 128, 256) if kv_bits == 8 else head_dim % 32:
            raise ValueError("head_dim must be 64, 128 or 256 (8-bit), a multiple of 32 (bf16)")
        self.layers, self.kv_heads, self.head_dim, self.num_seqs, self.kv_bits = layers, kv_heads, head_dim, num_seqs, kv_bits
        per = _pages(capacity)
        self.capacity = per * PAGE
        spare = 1 if kv_bits == 16 else 0
        self.n_pages = (per * num_seqs if num_pages is None else int(num_pages)) + spare
        if self.n_pages < 1 + spare:
            raise ValueError("a pool needs a page")
        self.absent = 0 if spare else -1
        dev = self.device = torch.device(device)
        shape = (layers, self.n_pages, kv_heads, PAGE * head_dim)
        self.k_pages = torch.zeros(shape, dtype=torch.int8 if kv_bits == 8 else torch.bfloat16, device=dev)
        self.v_pages = torch.zeros_like(self.k_pages)
        self.pools = [self.k_pages, self.v_pages]
        if kv_bits == 8:
            self.k_scales = torch.zeros(layers, self.n_pages, kv_heads, PAGE, dtype=torch.float32, device=dev)
            self.v_scales = torch.zeros_like(self.k_scales)
            self.pools += [self.k_scales, self.v_scales]
        i32 = dict(dtype=torch.int32, device=dev)
        self.tables = [torch.full((num_seqs, per), self.absent, **i32) for _ in range(2)]
        self.refs = torch.zeros(self.n_pages, **i32)
        self.copies = torch.full((num_seqs, 3), -1, **i32)
        self.status = torch.zeros(2, **i32)
        self.turn = 0
        self._lengths = [0] * num_seqs
        self._rooms = [(0, 0)] * num_seqs
        self._sequences: dict[int, PagedKVCache | PagedKVCacheQ8] = {}

    @property
    def table(self) -> torch.Tensor:
        """The page tables as the last fork left them."""
        return self.tables[self.turn]

    @property
    def lengths(self) -> list[int]:
        return [self._sequences[i].offset if i in self._sequences else n for i, n in enumerate(self._lengths)]

    # ---- launches ----------------------------------------------------------------
    def launch_fork(self, turn: int, lengths: int, lengths_out: int, parents: int | None, rows: int, advance: int,
                    st: int) -> None:
        """dtree_pages_fork from tables[turn] into the other, or, without parents, in
        place, and the copies it asks for. The arguments are device addresses."""
        a = N.PagesFork()
        a.refs = self.refs.data_ptr(); a.num_pages = self.n_pages
        a.num_seqs = self.num_seqs; a.ld_tables = self.tables[0].shape[1]
        a.tables = self.tables[turn].data_ptr()
        a.tables_out = self.tables[turn if parents is None else 1 - turn].data_ptr()
        a.lengths = lengths; a.lengths_out = lengths_out; a.parents = parents
        a.advance = advance; a.rows = rows; a.absent = self.absent
        a.copies = self.copies.data_ptr(); a.status = self.status.data_ptr()
        lib = N.lib()
        N.check(lib.dtree_pages_fork(C.byref(a), st), "pages fork")
        c = N.PagesCopy()
        c.copies = self.copies.data_ptr(); c.max_copies = self.num_seqs
        c.num_pages = self.n_pages; c.num_heads = self.kv_heads; c.layers = self.layers
        for i, t in enumerate(self.pools):
            c.pools[i] = t.data_ptr(); c.block_bytes[i] = t.shape[3] * t.element_size()
        N.check(lib.dtree_pages_copy(C.byref(c), st), "pages copy")

    def fork(self, parents=None, rows: int = 0) -> None:
        """Sequence i continues sequence parents[i] (-1: empty; None: itself), with room
        for ``rows`` more positions. Raises if the pool has no pages left for that; the
        sequences that found none have lost rows then, and the pool is to be started anew."""
        old = self.lengths
        if parents is None:
            src, new = None, old
        else:
            par = [int(p) for p in parents]
            if len(par) != self.num_seqs or any(p < -1 or p >= self.num_seqs for p in par):
                raise ValueError(f"parents are {self.num_seqs} sequences of this pool, or -1")
            src = torch.tensor(par, dtype=torch.int32, device=self.device)
            new = [old[p] if p >= 0 else 0 for p in par]
        if rows < 0 or max(new) + rows > self.capacity:
            raise ValueError(f"{max(new)} positions and {rows} rows exceed the capacity of {self.capacity}")
        if any(n > end for n, (_, end) in zip(old, self._rooms)):
            raise ValueError("a sequence's offset lies behind the positions that it has pages for")
        lengths = torch.tensor(old, dtype=torch.int32, device=self.device)
        self._set_rooms([(0, 0)] * self.num_seqs)
        with torch.cuda.device(self.refs.device):
            self.launch_fork(self.turn, lengths.data_ptr(), lengths.data_ptr(), None if src is None else src.data_ptr(), rows,
                             0, torch.cuda.current_stream().cuda_stream)
        if src is not None:
            self.turn = 1 - self.turn
        self._lengths = new
        for i, c in self._sequences.items():
            c.offset = new[i]
            c.page_table.view(-1).copy_(self.table[i])
        self.check()
        self._set_rooms([(n // PAGE * PAGE, _pages(n + rows) * PAGE) if rows else (n, n) for n in new])

    def _set_rooms(self, rooms: list[tuple[int, int]]) -> None:
        self._rooms = rooms
        for i, c in self._sequences.items():
            c.room = rooms[i]

    def check(self) -> None:
        """Raises if a fork since the last check found no page (waits for the stream)."""
        if int(self.status[0]):
            self.status.zero_()
            raise RuntimeError(f"the pool's {self.n_pages} pages are used up")

    def start(self, lengths) -> None:
        """Empties the pool and gives sequence i pages for its first lengths[i] positions."""
        need = [int(n) for n in lengths] + [0] * (self.num_seqs - len(lengths))
        if len(need) != self.num_seqs or min(need) < 0 or max(need) > self.capacity:
            raise ValueError("one length of at most the capacity per sequence")
        first = self.absent + 1
        if sum(_pages(n) for n in need) > self.n_pages - first:
            raise RuntimeError(f"the pool's {self.n_pages} pages are used up")
        table = torch.full(self.table.shape, self.absent, dtype=torch.int32)
        at = first
        for i, n in enumerate(need):
            table[i, :_pages(n)] = torch.arange(at, at + _pages(n))
            at += _pages(n)
        refs = torch.zeros(self.n_pages, dtype=torch.int32)
        refs[first:at] = 1
        self.table.copy_(table)
        self.refs.copy_(refs)
        self.status.zero_()
        self._lengths = [0] * self.num_seqs
        self._set_rooms([(0, _pages(n) * PAGE) for n in need])
        for i, c in self._sequences.items():
            c.offset = 0
            c.page_table.view(-1).copy_(self.table[i])

    # ---- the sequences as caches ----------------------------------------------------
    def _cache(self, table: torch.Tensor, num_seqs: int):
        """A cache object over the pool's pages with a page table of its own."""
        cls = PagedKVCacheQ8 if self.kv_bits == 8 else PagedKVCache
        c = cls.__new__(cls)
        c.layers, c.kv_heads, c.head_dim, c.n_pages = self.layers, self.kv_heads, self.head_dim, self.n_pages
        c.capacity, c.offset = self.capacity, 0
        c.k_pages, c.v_pages = self.k_pages, self.v_pages
        if self.kv_bits == 8:
            c.k_scales, c.v_scales, c.num_seqs = self.k_scales, self.v_scales, num_seqs
        c.page_table = table
        return c

    def sequence(self, i: int):
        """Sequence i as the engines take a cache. It follows the pool's forks: its page
        table and offset are those of sequence i after each. Its rows need room
        (``fork(..., rows=n)``) before an engine writes them: a step whose rows would lie
        in pages that other sequences hold, or in none, is refused."""
        if not 0 <= i < self.num_seqs:
            raise IndexError(i)
        if i not in self._sequences:
            row = self.table[i].clone()
            c = self._cache(row[None] if self.kv_bits == 8 else row, 1)
            c.offset, c.room = self._lengths[i], self._rooms[i]
            self._sequences[i] = c
        return self._sequences[i]

    def batch(self, turn: int) -> PagedKVCacheQ8:
        """All sequences of tables[turn] as one 8-bit batch."""
        if self.kv_bits != 8:
            raise ValueError("batches of sequences are stepped on the 8-bit cache")
        return self._cache(self.tables[turn], self.num_seqs)


class HypothesisCache:
    """A batch of hypotheses that continue one another from step to step.

    sources    [num_seqs] int32: the sequence that each continues in the next step, -1
               for one that begins (or has ended and gives its pages up)
    desc       the step's DtreeStepDesc, whose tokens and positions (views of it, int32)
               the device writes: the next tokens, the sequences' lengths
    ``turn`` says which of the two tables, windows and states the next step reads.
    """

    def __init__(self, engine, num_seqs: int, num_pages: int):
        c = engine.cfg
        if engine.kv_bits != 8:
            raise ValueError("batches of hypotheses are decoded on the 8-bit cache (kv_bits 8)")
        if not 1 <= num_seqs <= engine.max_nodes:
            raise ValueError(f"the engine steps up to {engine.max_nodes} rows (max_nodes), asked for {num_seqs}")
        dev = engine.dev
        hybrid = hasattr(c, "attention_layers")
        layers = len(c.attention_layers) if hybrid else c.num_hidden_layers
        self.num_seqs = num_seqs
        self.pool = PagedKVPool(layers, c.num_key_value_heads, c.head_dim, engine.max_past + engine.max_nodes, num_seqs,
                                num_pages=num_pages, kv_bits=8, device=dev)
        self.batches = [self.pool.batch(1 - turn) for turn in (0, 1)]  # of the step at `turn`
        self.sources = torch.full((num_seqs,), -1, dtype=torch.int32, device=dev)
        self.ones = torch.ones(num_seqs, dtype=torch.int32, device=dev)
        self.desc = torch.zeros(C.sizeof(N.StepDesc) // 4, dtype=torch.int32, device=dev)
        self.desc[N.StepDesc.num_nodes.offset // 4] = num_seqs
        self.tokens, self.positions = (self.desc[f.offset // 4:][:num_seqs] for f in (N.StepDesc.tokens, N.StepDesc.positions))
        self.max_past = 0  # bound of the step's lengths, on the host
        self.workspace = None
        self.slot = {li: i for i, li in enumerate(c.attention_layers)} if hybrid else {i: i for i in range(layers)}
        self.windows = self.states = None
        if hybrid:
            linear = c.linear_layers
            self.slot.update({li: i for i, li in enumerate(linear)})
            self.windows = torch.zeros(2, len(linear), num_seqs, c.linear_conv_kernel_dim - 1, c.conv_dim, device=dev)
            self.states = torch.zeros(2, len(linear), num_seqs, c.linear_num_value_heads, c.linear_value_head_dim,
                                      c.linear_key_head_dim, device=dev)

    @property
    def turn(self) -> int:
        return self.pool.turn

    def flip(self) -> None:
        """The step's tables, windows and states become the ones that the next reads."""
        self.pool.turn = 1 - self.pool.turn
