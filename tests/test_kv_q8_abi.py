"""Refusals of the 8-bit cache's entry points (nothing is launched), and the
host side of its layout. CPU only."""
import ctypes as C

import pytest
import torch

from dtree_hip import _native as N
from dtree_hip.cache import PAGE, PagedKVCacheQ8, _block_index_q8, quantise_q8


def cache(**kw):
    r = N.KvQ8()
    base = dict(k_pages=4096, v_pages=4096, k_scales=4096, v_scales=4096, num_pages=8, num_kv_heads=2, head_dim=128,
                num_seqs=1, page_tables=4096, ld_page_table=8, max_past_length=448, max_rows=64, total_rows=64,
                past_lengths=4096, row_counts=4096)
    base.update(kw)
    for k, v in base.items():
        setattr(r, k, v)
    return r


def attn(**kw):
    a = N.AttnQ8Args()
    base = dict(q=4096, ld_q=1024, q_stride=128, out=4096, ld_out=1024, num_heads=8, scale=0.1, eps=1e-6)
    base.update(kw)
    for k, v in base.items():
        setattr(a, k, v)
    return a


def refused(rc, word):
    assert rc == N.E_ARG
    msg = N.lib().dtree_last_error().decode()
    assert word in msg, msg


BAD_CACHE = [
    (dict(k_pages=None), "null"), (dict(v_scales=None), "null"), (dict(page_tables=None), "null"),
    (dict(past_lengths=None), "null"), (dict(row_counts=None), "null"), (dict(k_pages=4104), "aligned"),
    (dict(v_scales=4100), "aligned"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(num_kv_heads=0), "num_kv_heads"), (dict(num_pages=0), "num_pages"), (dict(num_seqs=0), "num_seqs"),
    (dict(max_rows=0), "max_rows"), (dict(max_rows=-1), "max_rows"), (dict(max_past_length=-1), "max_past_length"),
    (dict(max_past_length=1 << 30), "max_past_length"), (dict(total_rows=0), "total_rows"),
    (dict(max_past_length=513), "page tables"), (dict(ld_page_table=6), "page tables"), (dict(ld_page_table=0), "page tables"),
    (dict(num_seqs=65536, max_rows=1 << 20, ld_page_table=1 << 20), "row_starts"),
]


@pytest.mark.parametrize("kw,word", BAD_CACHE)
def test_cache_records_refused_by_every_entry(kw, word):
    lib = N.lib()
    r = cache(**kw)
    refused(lib.dtree_kv_q8_append(C.byref(r), 4096, 4096, N.T_F32, 256, 256, None, 0.0, None, None, 0, None), word)
    refused(lib.dtree_kv_q8_read(C.byref(r), 4096, 4096, N.T_F32, 256, 256, None), word)
    refused(lib.dtree_attention_q8(C.byref(r), C.byref(attn()), None), word)


def test_null_records():
    lib = N.lib()
    refused(lib.dtree_kv_q8_append(None, 4096, 4096, 0, 256, 256, None, 0.0, None, None, 0, None), "null")
    refused(lib.dtree_kv_q8_read(None, 4096, 4096, 0, 256, 256, None), "null")
    refused(lib.dtree_attention_q8(None, C.byref(attn()), None), "null")
    refused(lib.dtree_attention_q8(C.byref(cache()), None, None), "null")
    assert lib.dtree_attention_q8_workspace_bytes(None, None) == 0


@pytest.mark.parametrize("args,word", [
    ((None, 4096, 0, 256, 256, None, 0.0, None, None, 0), "null"),
    ((4096, None, 0, 256, 256, None, 0.0, None, None, 0), "null"),
    ((4096, 4096, 2, 256, 256, None, 0.0, None, None, 0), "type"),
    ((4100, 4096, 0, 256, 256, None, 0.0, None, None, 0), "aligned"),
    ((4096, 4096, 0, 255, 256, None, 0.0, None, None, 0), "k: rows"),
    ((4096, 4096, 0, 256, 252, None, 0.0, None, None, 0), "v: rows"),
    ((4096, 4096, 1, 260, 256, None, 0.0, None, None, 0), "k: rows"),
    ((4096, 4096, 0, 256, 256, None, 0.0, 4096, 4096, 48), "rope_dims"),
    ((4096, 4096, 0, 256, 256, None, 0.0, 4096, 4096, 160), "rope_dims"),
    ((4096, 4096, 0, 256, 256, None, 0.0, None, 4096, 64), "RoPE table"),
    ((4096, 4096, 0, 256, 256, None, -1.0, None, None, 0), "eps"),
])
def test_append_refusals(args, word):
    refused(N.lib().dtree_kv_q8_append(C.byref(cache()), *args, None), word)


@pytest.mark.parametrize("args,word", [
    ((None, None, 0, 256, 256), "null"), ((4096, 4096, 3, 256, 256), "type"), ((4096, 4096, 0, 128, 256), "k: rows"),
    ((4096, 4104, 1, 256, 256), "v: rows"),
])
def test_read_refusals(args, word):
    refused(N.lib().dtree_kv_q8_read(C.byref(cache()), *args, None), word)


@pytest.mark.parametrize("ckw,kw,word", [
    ({}, dict(q=None), "null"), ({}, dict(out=None), "null"), ({}, dict(num_heads=7), "num_heads"),
    ({}, dict(num_heads=0), "num_heads"), ({}, dict(num_heads=2048), "num_heads"), ({}, dict(q_type=2), "type"),
    ({}, dict(q=4104), "q rows"), ({}, dict(ld_q=1020), "q rows"), ({}, dict(q_stride=64), "q rows"),
    ({}, dict(q_stride=130), "q rows"), ({}, dict(gated=1), "q rows"), ({}, dict(q_type=1, ld_q=1028), "q rows"),
    ({}, dict(rope_dims=16, rope_cos=4096, rope_sin=4096), "rope_dims"), ({}, dict(rope_dims=64), "RoPE table"),
    ({}, dict(scale=0.0), "scale"), ({}, dict(scale=float("nan")), "scale"), ({}, dict(scale=float("inf")), "scale"),
    ({}, dict(eps=-1.0), "eps"), ({}, dict(window=-1), "window"), ({}, dict(sink=-1), "window"),
    ({}, dict(ancestors=4096, window=10), "tree"),
    (dict(max_rows=129), dict(ancestors=4096), "tree"),
    ({}, dict(out=4100), "out layout"), ({}, dict(ld_out=1022), "out layout"), ({}, dict(ld_out=512), "out layout"),
    ({}, dict(out_layout=N.W_TILED, ld_out=1088), "out layout"), ({}, dict(out_layout=N.W_Q4G64), "out layout"),
    ({}, dict(rows_padded=-1), "rows_padded"), ({}, dict(rows_padded=65), "rows_padded"),
    (dict(row_starts=4096), dict(rows_padded=64), "rows_padded"), (dict(num_seqs=2), dict(rows_padded=64), "rows_padded"),
])
def test_attention_refusals(ckw, kw, word):
    refused(N.lib().dtree_attention_q8(C.byref(cache(**ckw)), C.byref(attn(**kw)), None), word)


def test_compact_refusals():
    lib = N.lib()
    ok = dict(desc=4096, k=4096, v=4096, ks=4096, vs=4096, layers=1, pages=8, heads=2, dim=128, table=4096, entries=8,
              hin=None, w=0, hout=None)
    for kw, word in ((dict(desc=None), "null"), (dict(table=None), "null"), (dict(k=4104), "aligned"),
                     (dict(dim=32), "head_dim"), (dict(layers=0), "layers"), (dict(pages=0), "layers"),
                     (dict(entries=0), "table_pages"), (dict(hout=4096), "hidden"),
                     (dict(hout=4096, hin=4096, w=12), "hidden")):
        a = dict(ok)
        a.update(kw)
        refused(lib.dtree_kv_q8_compact(*a.values(), None), word)


def test_workspace_holds_the_ranges_partials():
    lib = N.lib()
    need = lib.dtree_attention_q8_workspace_bytes(C.byref(cache(max_past_length=0, ld_page_table=1)), C.byref(attn()))
    assert need == 0  # one page: one range
    long = cache(max_past_length=65536, ld_page_table=1100, max_rows=1, total_rows=1)
    row = 8 * (128 + 2) * 4
    need = lib.dtree_attention_q8_workspace_bytes(C.byref(long), C.byref(attn()))
    assert need > row and need % row == 0


@pytest.mark.parametrize("d", [64, 128, 256])
def test_page_order_is_a_permutation_in_the_documented_order(d):
    for which in "kv":
        off = _block_index_q8(d, which)
        assert sorted(off.reshape(-1).tolist()) == list(range(PAGE * d))
    s, i = 37, d - 5
    assert _block_index_q8(d, "k")[s, i] == (((s // 32) * (d // 32) + i // 32) * 64 + (i // 16 % 2) * 32 + s % 32) * 16 + i % 16
    assert _block_index_q8(d, "v")[s, i] == ((((s // 32) * (d // 32) + i // 32) * 64 + (s // 4 % 2) * 32 + i % 32) * 16
                                             + (s // 8 % 4) * 4 + s % 4)


def test_quantised_rows():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5], [0.0, 0.0, 0.0, 0.0], [1.0, float("nan"), 0.0, 0.0],
                      [float("-inf"), 1.0, 0.0, 0.0]])
    q, s = quantise_q8(x)
    assert q[0].tolist() == [127, 0, 2, -2] and s[0] == 1.0  # ties to even
    assert q[1].tolist() == [0] * 4 and s[1] == 0.0
    assert torch.isnan(s[2:]).all() and (q[2:] == 0).all()


def test_cache_class_on_the_cpu():
    g = torch.Generator().manual_seed(1)
    c = PagedKVCacheQ8(2, 3, 64, 130, num_seqs=2, device="cpu", page_order=torch.randperm(6, generator=g))
    assert c.capacity == 192 and c.n_pages == 6 and c.page_table.shape == (2, 3)
    k, v = torch.randn(100, 3, 64, generator=g), torch.randn(100, 3, 64, generator=g)
    c.write_logical(1, k, v, start=30, seq=1)
    for got, x in ((c.logical_keys(1, 130, 1)[30:], k), (c.logical_values(1, 130, 1)[30:], v)):
        step = x.abs().amax(-1, keepdim=True) / 127
        # half a step of the rounding, and the product's and the scale's own (2^-24 each, of at most 127 steps)
        assert bool(((got - x).abs() <= step * (0.5 + 2 * 127 * 2.0 ** -24)).all())
    assert bool((c.logical_keys(0, 192, 1) == 0).all()) and bool((c.logical_keys(1, 192, 0) == 0).all())
    with pytest.raises(ValueError):
        c.write_logical(0, k, v, start=150)
    with pytest.raises(ValueError):
        PagedKVCacheQ8(1, 1, 96, 64, device="cpu")
    with pytest.raises(IndexError):
        c.record(2, None, None, 0, 1, 1)
    with pytest.raises(ValueError):
        c.record(0, torch.zeros(2), torch.zeros(2, dtype=torch.int32), 0, 1, 1)


def test_cache_class_with_a_page_given_away():
    """Its positions read as zeros and take no rows; the pool's other pages stay."""
    c = PagedKVCacheQ8(1, 2, 64, 192, device="cpu")
    rows = torch.randn(192, 2, 64, generator=torch.Generator().manual_seed(0))
    c.write_logical(0, rows, -rows)
    keys = c.logical_keys(0, 192)
    c.page_table[0, 0] = -1
    assert torch.equal(c.logical_keys(0, 192)[64:], keys[64:])
    assert not c.logical_keys(0, 192)[:64].any() and not c.logical_values(0, 192)[:64].any()
    before = c.k_pages.clone()
    with pytest.raises(ValueError):
        c.write_logical(0, rows[:1], rows[:1], start=63)
    assert torch.equal(c.k_pages, before)
