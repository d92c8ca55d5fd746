"""dtree_pages_fork and dtree_pages_copy against the rule in plain Python
(oracle/beam.py): whole numbers and bytes, so everything is equal."""
import ctypes as C

import numpy as np
import pytest
import torch

from dtree_hip import _native as N
from oracle import beam as ob

from gpu_util import stream

pytestmark = pytest.mark.gpu
PAGE = 64


class Pool:
    """Tables, counts and lengths on the device, and their copies in the oracle."""

    def __init__(self, dev, seqs, ld, pages, absent=-1, seed=0):
        g = np.random.default_rng(seed)
        self.dev, self.n, self.ld, self.absent, self.g = dev, seqs, ld, absent, g
        self.refs = np.zeros(pages, np.int32)
        self.tables = np.full((seqs, ld), absent, np.int32)
        self.lengths = np.zeros(seqs, np.int32)
        if absent >= 0:
            self.refs[absent] = 3  # (kept by the caller: whatever its count is, it is not taken)

    def fill(self, lengths, spread=True):
        order = [p for p in (self.g.permutation(len(self.refs)) if spread else range(len(self.refs))) if p != self.absent]
        for i, n in enumerate(lengths):
            self.lengths[i] = n
            for e in range(-(-n // PAGE)):
                p = order.pop()
                self.tables[i, e] = p
                self.refs[p] = 1
        return self

    def fork(self, parents, advance=0, rows=0, in_place=False, st=None):
        dev = self.dev
        t = lambda x: None if x is None else torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev)  # noqa: E731
        refs, tables, lengths, par = t(self.refs), t(self.tables), t(self.lengths), t(parents)
        tables_out = tables if in_place else torch.full_like(tables, 99)
        lengths_out = lengths if in_place else torch.full_like(lengths, 99)
        copies = torch.full((self.n, 3), 99, dtype=torch.int32, device=dev)
        status = torch.tensor([5, 99], dtype=torch.int32, device=dev)
        a = N.PagesFork()
        a.refs = refs.data_ptr(); a.num_pages = len(self.refs); a.num_seqs = self.n; a.ld_tables = self.ld
        a.tables = tables.data_ptr(); a.tables_out = tables_out.data_ptr()
        a.lengths = lengths.data_ptr(); a.lengths_out = lengths_out.data_ptr()
        a.parents = par.data_ptr() if par is not None else None
        a.advance = advance; a.rows = rows; a.absent = self.absent
        a.copies = copies.data_ptr(); a.status = status.data_ptr()
        N.check(N.lib().dtree_pages_fork(C.byref(a), stream() if st is None else st), "fork")
        torch.cuda.synchronize()
        want = ob.fork(self.refs, self.tables, self.lengths, parents, advance, rows, self.absent)
        got = copies.cpu().numpy()
        assert np.array_equal(lengths_out.cpu().numpy(), want[2])
        assert np.array_equal(tables_out.cpu().numpy(), want[1])
        assert np.array_equal(refs.cpu().numpy(), want[0])
        n = len(want[3])
        assert [tuple(c) for c in got[:n].tolist()] == want[3] and (got[n:] == -1).all()
        assert status.tolist() == [5 + want[4], n]
        if not in_place:
            assert np.array_equal(tables.cpu().numpy(), self.tables) and np.array_equal(lengths.cpu().numpy(), self.lengths)
        self.refs, self.tables, self.lengths = want[0].astype(np.int32), want[1].astype(np.int32), want[2].astype(np.int32)
        return want[3], want[4]

    def consistent(self):
        """Every count is the number of tables that hold the page."""
        held = np.zeros(len(self.refs), int)
        for t in self.tables:
            for p in t:
                if p >= 0 and p != self.absent:
                    held[p] += 1
        keep = np.arange(len(held)) != self.absent
        assert np.array_equal(held[keep], self.refs[keep])


@pytest.mark.parametrize("rows", [0, 1, 25, 64, 200])
@pytest.mark.parametrize("absent", [-1, 0, 17])
def test_a_prompt_becomes_beams(gpu_device, rows, absent):
    p = Pool(gpu_device, 8, 24, 150, absent, seed=rows).fill([1000])
    copies, missing = p.fork([0] * 8, rows=rows)
    assert missing == 0 and len(copies) == (7 if rows else 0)
    p.consistent()
    for _ in range(4):
        p.fork([3, 3, 0, 7, 7, 7, 1, -1], advance=min(rows, 1), rows=rows)
        p.consistent()


@pytest.mark.parametrize("seqs,ld,pages", [(1, 1, 1), (2, 3, 9), (7, 5, 40), (33, 17, 900), (64, 2000, 3000), (256, 9, 4000),
                                           (1024, 4, 5000), (1000, 3, 70001)])
def test_random_runs(gpu_device, seqs, ld, pages):
    g = np.random.default_rng(seqs)
    p = Pool(gpu_device, seqs, ld, pages, seed=seqs).fill([int(g.integers(0, ld * PAGE // 2 + 1)) for _ in range(seqs)]
                                                          if pages >= seqs * ld // 2 else [ld * PAGE // 2])
    for k in range(6):
        parents = g.integers(0, seqs, seqs)
        parents[g.random(seqs) < 0.1] = -1
        p.fork(parents, advance=int(g.choice([0, 1, 7, 64])), rows=int(g.choice([0, 1, 1, 30, 64, 65])))
        p.consistent()


def test_lengths_at_page_borders(gpu_device):
    for n in (0, 1, 63, 64, 65, 127, 128):
        for rows in (0, 1, 63, 64, 65):
            p = Pool(gpu_device, 3, 6, 30, seed=n).fill([n, 5])
            p.fork([0, 0, 1], rows=rows)
            p.consistent()
            p.fork([2, 0, 1], advance=rows, rows=rows)
            p.consistent()


def test_in_place_growth_and_rows_given_back(gpu_device):
    p = Pool(gpu_device, 5, 12, 60, seed=4).fill([100, 0, 64, 300, 1])
    p.fork(None, rows=130, in_place=True)
    p.consistent()
    p.fork(None, advance=3, rows=0, in_place=True)  # pages behind the lengths are free again
    p.consistent()
    p.fork(None, rows=0)
    p.consistent()


def test_shared_pages_that_grow_later(gpu_device):
    """Forked without room: the page is shared by more sequences than write to it."""
    p = Pool(gpu_device, 6, 8, 60, seed=5).fill([70, 200])
    p.fork([0, 0, 0, 1, 1, 0], rows=0)
    copies, _ = p.fork(None, rows=1, in_place=True)
    assert len(copies) == 4
    p.consistent()
    # held by a caller as well: every writer copies
    p = Pool(gpu_device, 2, 8, 60, seed=6).fill([70])
    p.refs[p.tables[0, 1]] += 1
    copies, _ = p.fork([0, 0], rows=1)
    assert len(copies) == 2


def test_no_pages_left(gpu_device):
    p = Pool(gpu_device, 6, 10, 12, seed=7).fill([500, 100])
    _, missing = p.fork([0, 0, 0, 1, 1, 1], rows=20)
    assert missing > 0
    p.consistent()
    p = Pool(gpu_device, 3, 4, 40, seed=8).fill([250, 200, 256])
    _, missing = p.fork(None, rows=70)  # the tables' ends
    assert missing == 4  # 320, 270 and 326 positions: 5, 5 and 6 pages, of 4 each
    p.consistent()


def test_parents_and_tables_that_are_not_there(gpu_device):
    p = Pool(gpu_device, 4, 4, 20, seed=9).fill([100, 50, 70])
    p.tables[0, 1] = 4000
    p.tables[2, 0] = -7
    p.refs[p.tables[1, 0]] = 1
    p.fork([0, 4, 2 ** 31 - 1, -5], rows=1)
    p.lengths[0] = -3
    p.lengths[1] = 1 << 30
    p.fork([0, 1, 1, 0], rows=0)


@pytest.mark.parametrize("ld,pages", [(7, 40), (7, 3000), (900, 9000)])
def test_arrays_side_by_side_in_memory(gpu_device, ld, pages):
    """One allocation holds all arrays, so that neighbours share cache lines with the counts
    that the launch changes and then reads (forks of one launch and of two)."""
    n = 12
    p = Pool(gpu_device, n, ld, pages, seed=ld).fill([200, 64, 130, 400, 1, 0, 63])
    sizes = dict(parents=n, lengths=n, refs=pages, out=n, tables=n * ld, tables_out=n * ld, copies=3 * n, status=2)
    flat = torch.zeros(sum(sizes.values()), dtype=torch.int32, device=gpu_device)
    at, view = 0, {}
    for k, m in sizes.items():
        view[k] = flat[at:at + m]
        at += m
    g = np.random.default_rng(ld)
    for k in range(6):
        parents = g.integers(-1, 7 if k == 0 else n, n)
        for name, x in (("parents", parents), ("lengths", p.lengths), ("refs", p.refs), ("tables", p.tables.reshape(-1))):
            view[name].copy_(torch.as_tensor(np.asarray(x, np.int32)))
        view["status"].zero_()
        a = N.PagesFork()
        a.refs = view["refs"].data_ptr(); a.num_pages = pages; a.num_seqs = n; a.ld_tables = ld
        a.tables = view["tables"].data_ptr(); a.tables_out = view["tables_out"].data_ptr()
        a.lengths = view["lengths"].data_ptr(); a.lengths_out = view["out"].data_ptr()
        a.parents = view["parents"].data_ptr(); a.advance = 1; a.rows = 5; a.absent = -1
        a.copies = view["copies"].data_ptr(); a.status = view["status"].data_ptr()
        N.check(N.lib().dtree_pages_fork(C.byref(a), stream()), "fork")
        torch.cuda.synchronize()
        ref = ob.fork(p.refs, p.tables, p.lengths, parents, 1, 5)
        assert np.array_equal(view["refs"].cpu().numpy(), ref[0])
        assert np.array_equal(view["tables_out"].cpu().numpy().reshape(n, ld), ref[1])
        assert np.array_equal(view["out"].cpu().numpy(), ref[2])
        assert [tuple(c) for c in view["copies"].view(n, 3)[:len(ref[3])].tolist()] == ref[3]
        assert view["status"].tolist() == [ref[4], len(ref[3])]
        p.refs, p.tables, p.lengths = ref[:3]


def kv(dev, layers, pages, heads, dim, bits, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    if bits == 16:
        return [torch.randn(layers, pages, heads, PAGE * dim, device=dev, generator=g).bfloat16() for _ in range(2)]
    q = [torch.randint(-127, 128, (layers, pages, heads, PAGE * dim), device=dev, generator=g, dtype=torch.int8)
         for _ in range(2)]
    return q + [torch.rand(layers, pages, heads, PAGE, device=dev, generator=g) for _ in range(2)]


def copy_args(pools, copies):
    a = N.PagesCopy()
    layers, pages, heads, _ = pools[0].shape
    a.copies = copies.data_ptr(); a.max_copies = len(copies); a.num_pages = pages; a.num_heads = heads; a.layers = layers
    for i, t in enumerate(pools):
        a.pools[i] = t.data_ptr(); a.block_bytes[i] = t.shape[3] * t.element_size()
    return a


@pytest.mark.parametrize("layers,heads,dim,bits", [(1, 1, 64, 8), (3, 8, 128, 8), (8, 4, 256, 8), (2, 3, 96, 16), (5, 8, 128, 16)])
def test_copies(gpu_device, layers, heads, dim, bits):
    pools = kv(gpu_device, layers, 40, heads, dim, bits, seed=dim)
    want = [t.clone() for t in pools]
    entries = [(3, 30, 1), (3, 31, 32), (4, 32, 33), (5, 33, 63), (6, 34, 64), (7, 40, 9), (41, 35, 9), (8, 36, 0),
               (9, -1, 5), (10, 37, 20), (-1, 38, 64), (11, 39, 64)]
    copies = torch.tensor(entries, dtype=torch.int32, device=gpu_device)
    for s, d, used in entries[:5] + [entries[9]]:
        for t in want:
            n = t.shape[3] if used > 32 else t.shape[3] // 2
            t[:, d, :, :n] = t[:, s, :, :n]
    N.check(N.lib().dtree_pages_copy(C.byref(copy_args(pools, copies)), stream()), "copy")
    for t, w in zip(pools, want):
        assert torch.equal(t, w)


def test_copied_half_pages_hold_the_first_positions(gpu_device):
    """The order of every kind of page: positions 0 .. 31 are its blocks' first half."""
    from dtree_hip.cache import _block_index, _block_index_q8

    for index in (_block_index, _block_index_q8):
        for which in "kv":
            assert int(index(128, which)[:32].max()) == 32 * 128 - 1


def test_replayed_graph(gpu_device):
    """Fork and copy in a graph whose tables change sides: two graphs, replayed in turn."""
    lib, dev = N.lib(), gpu_device
    n, ld, pages = 6, 5, 40
    pools = kv(dev, 2, pages, 2, 64, 8, seed=1)
    p = Pool(dev, n, ld, pages, seed=2).fill([100])
    t = lambda x: torch.as_tensor(x, dtype=torch.int32).to(dev)  # noqa: E731
    refs, tables, lengths = t(p.refs), [t(p.tables), t(p.tables)], [t(p.lengths), t(p.lengths)]
    parents, copies, status = t([0] * n), t(np.full((n, 3), -1)), t([0, 0])
    side = torch.cuda.Stream()
    graphs = []
    for turn in (0, 1):
        a = N.PagesFork()
        a.refs = refs.data_ptr(); a.num_pages = pages; a.num_seqs = n; a.ld_tables = ld
        a.tables = tables[turn].data_ptr(); a.tables_out = tables[1 - turn].data_ptr()
        a.lengths = lengths[turn].data_ptr(); a.lengths_out = lengths[1 - turn].data_ptr()
        a.parents = parents.data_ptr(); a.advance = 1; a.rows = 1; a.absent = -1
        a.copies = copies.data_ptr(); a.status = status.data_ptr()
        torch.cuda.synchronize()
        N.check(lib.dtree_graph_begin(side.cuda_stream), "begin")
        N.check(lib.dtree_pages_fork(C.byref(a), side.cuda_stream), "fork")
        N.check(lib.dtree_pages_copy(C.byref(copy_args(pools, copies)), side.cuda_stream), "copy")
        ex = C.c_void_p()
        N.check(lib.dtree_graph_end(side.cuda_stream, C.byref(ex)), "end")
        graphs.append(ex)
    g = np.random.default_rng(3)
    try:
        for k in range(8):
            par = [0] * n if k == 0 else g.integers(-1, n, n).tolist()
            parents.copy_(t(par))
            want = [x.clone() for x in pools]
            torch.cuda.synchronize()
            N.check(lib.dtree_graph_launch(graphs[k % 2], side.cuda_stream), "launch")
            torch.cuda.synchronize()
            ref = ob.fork(p.refs, p.tables, p.lengths, par, 1, 1)
            p.refs, p.tables, p.lengths = ref[:3]
            assert np.array_equal(tables[1 - k % 2].cpu().numpy(), ref[1]) and np.array_equal(refs.cpu().numpy(), ref[0])
            for s, d, used in ref[3]:
                for w in want:
                    m = w.shape[3] if used > 32 else w.shape[3] // 2
                    w[:, d, :, :m] = w[:, s, :, :m]
            for x, w in zip(pools, want):
                assert torch.equal(x, w)
    finally:
        torch.cuda.synchronize()
        for ex in graphs:
            lib.dtree_graph_destroy(ex)
