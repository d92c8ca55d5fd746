"""Attention over the 8-bit cache in the forms that long contexts take: many key
ranges and their join, the 8-wave kernels, ranges longer than a wave's page ids.

Each case asserts the number of key ranges that it means to run, from the
workspace that the call asks for. The tolerance is test_gpu_kv_q8's; its fp32
share, 2^-16 A, counts sums of up to 64 terms, and here a lane adds up to T / 16
weights (16 lanes or more share a row's T keys), numerator and denominator alike:
2 T / 16 2^-24 A more. A is at most 2^11 of that tolerance (it holds 2^-11 A), so
T 2^-16 of it covers that."""
import ctypes as C

import pytest
import torch

from dtree_hip import _native as N

from gpu_util import device_desc, random_tree, stream
from test_gpu_kv_q8 import BF16, FP16, PAIR, Batch, check, i32

pytestmark = pytest.mark.gpu


def ranges(b, rec, a):
    """Key ranges of the call's plan (0: one, which needs no workspace)."""
    return N.lib().dtree_attention_q8_workspace_bytes(C.byref(rec), C.byref(a)) // (b.total * b.hq * (b.d + 2) * 4)


def long_tol(b, tol):
    return tol * (1 + max(p + n for p, n in zip(b.past, b.rows)) * 2.0 ** -16)


def run(b, least, rounding=BF16, **kw):
    """attend() against the reference, with a plan of `least` ranges or more."""
    rec = b.rec()
    n = ranges(b, rec, b.args(b.qkv, **kw))
    assert n >= least, n
    want, tol = b.reference(**{k: kw[k] for k in ("sink", "window") if k in kw})
    got = b.attend(pair=rounding == PAIR, rec=rec, **kw)
    check(got, want, long_tol(b, tol), rounding, kw)
    assert torch.equal(got, b.attend(pair=rounding == PAIR, rec=rec, **kw))


# ---- tokens --------------------------------------------------------------------------
@pytest.mark.parametrize("heads,past,least", [("128", 5000, 8), ("64", 9000, 16), ("mqa", 9000, 16), ("256g", 5000, 4),
                                              ("256", 5000, 4)])
def test_token_over_many_ranges(gpu_device, heads, past, least):
    """As many ranges as the join has groups for, or more."""
    b = Batch(gpu_device, heads, [past], [1], seed=51)
    b.append()
    run(b, least, rounding=PAIR)


@pytest.mark.parametrize("heads,seqs,keys,least", [("128", 40, 2500, 2), ("128", 20, 5000, 8), ("64", 40, 2500, 2),
                                                   ("64", 16, 9000, 16), ("256g", 28, 2500, 2)])
@pytest.mark.parametrize("rows", [1, 4])
def test_tokens_of_a_long_batch(gpu_device, heads, seqs, keys, least, rows):
    """More than 256 workgroups of several ranges each (4 waves), lengths from 1 to
    the longest: most ranges of the short sequences are empty."""
    past = [keys * (s + 1) // seqs - 1 for s in range(seqs)]
    past[1] = 0
    b = Batch(gpu_device, heads, past, [1 + s % rows for s in range(seqs)], seed=52)
    b.append()
    rec = b.rec()
    assert ranges(b, rec, b.args(b.qkv)) * seqs * b.hkv > 256
    run(b, least)


def test_token_range_past_the_page_ids_of_a_wave(gpu_device):
    """One range, more than 64 pages a wave: 8 waves (128 dims), 4 (256)."""
    for heads, past in ("128", 34000), ("256g", 20000):
        b = Batch(gpu_device, heads, [past], [1], seed=53)
        b.append()
        want, tol = b.reference()
        check(b.attend(workspace=False), want, long_tol(b, tol), BF16, heads)


# ---- rows: 8 waves from 2048 visible positions and over 128 pairs, with 128 dims -------
@pytest.mark.parametrize("heads", ["128", "128x1"])
@pytest.mark.parametrize("sink,window", [(0, 0), (5, 2200), (70, 2050), (0, 2300)])
@pytest.mark.parametrize("past,rows", [([2500, 2300], [300, 300]), ([2500, 0, 2100, 700], [300, 190, 1, 40])])
def test_rows_of_8_waves_in_a_batch(gpu_device, heads, sink, window, past, rows):
    b = Batch(gpu_device, heads, past, rows, seed=54, pad=2)
    b.append()
    run(b, 2, sink=sink, window=window)
    want, tol = b.reference(sink=sink, window=window)
    check(b.attend(workspace=False, sink=sink, window=window), want, long_tol(b, tol), BF16, "one range")


@pytest.mark.parametrize("nodes", [33, 64, 128])
@pytest.mark.parametrize("past", [2100, 4500])
def test_draft_tree_of_8_waves(gpu_device, nodes, past):
    b = Batch(gpu_device, "128", [past], [nodes], seed=55, pad=3)
    parents = random_tree(nodes, seed=nodes)
    b.append()
    desc = device_desc([0] * nodes, [past] * nodes, parents, past, gpu_device)
    anc = desc.data_ptr() + N.StepDesc.ancestors.offset
    want, tol = b.reference(parents=parents)
    tol = long_tol(b, tol)
    rec = b.rec(row_starts=None)
    assert ranges(b, rec, b.args(b.qkv, ancestors=anc)) >= 2
    for ws in (True, False):
        check(b.attend(ancestors=anc, rec=rec, workspace=ws), want, tol, BF16, ws)
    want[nodes:] = 0
    check(b.attend(ancestors=anc, rec=rec, rows_padded=b.total), want, tol, BF16, "padded")


@pytest.mark.parametrize("heads,rows", [("128", 100), ("128", 300), ("256g", 100)])
@pytest.mark.parametrize("workspace", [True, False])
def test_tiled_rows_over_a_long_prefix(gpu_device, heads, rows, workspace):
    """The engines' output layouts, rows behind the last one cleared."""
    dev = gpu_device
    past, pad = 2500, 32 * ((rows + 31) // 32) + 32
    b = Batch(dev, heads, [past], [rows], seed=56)
    b.total = pad
    b.qkv = torch.cat([b.qkv, torch.zeros(pad - rows, b.width, device=dev)])
    b.cos, b.sin = (torch.cat([t, torch.zeros(pad - rows, t.shape[1], device=dev)]) for t in (b.cos, b.sin))
    b.append()
    want, tol = b.reference()
    want[rows:] = 0
    tol = long_tol(b, tol)
    W = b.hq * b.d
    r, k = torch.arange(pad, device=dev)[:, None], torch.arange(W, device=dev)[None]
    at = ((((r >> 5) * (W >> 6) + (k >> 6)) * 4 + ((k & 31) >> 3)) * 512 + ((r & 31) + 32 * ((k & 63) >> 5)) * 8 + (k & 7))
    for layout, dt, rounding in ((N.W_TILED, torch.bfloat16, PAIR), (N.W_TILED_F16, torch.float16, FP16)):
        out = torch.full((2, pad * W), 7.0, dtype=dt, device=dev)
        a = b.args(out[0], out_layout=layout, out_lo=out[1].data_ptr(), rows_padded=pad)
        rec = b.rec(row_starts=None, max_rows=rows)
        need = N.lib().dtree_attention_q8_workspace_bytes(C.byref(rec), C.byref(a))
        assert ranges(b, rec, a) >= 2
        ws = torch.full((need,), 255, dtype=torch.uint8, device=dev)
        if workspace:
            a.workspace = ws.data_ptr(); a.workspace_bytes = need
        N.check(N.lib().dtree_attention_q8(C.byref(rec), C.byref(a), stream()), "attention")
        got = out[0].double() + (out[1].double() if layout == N.W_TILED else 0)
        check(got[at], want, tol + 2.0 ** -25, rounding, str(layout))


@pytest.mark.parametrize("heads,rows", [("128", 100), ("256g", 100), ("64", 100)])
def test_rows_range_past_the_page_ids_of_a_wave(gpu_device, heads, rows):
    """One range of more than 64 pages, absent pages before and behind the 64th."""
    b = Batch(gpu_device, heads, [4500], [rows], seed=57)
    b.append()
    for gone in ((), (3, 40, 63, 64, 68)):
        for i in gone:
            b.cache.page_table[0, i] = -1
        want, tol = b.reference()
        check(b.attend(workspace=False), want, long_tol(b, tol), BF16, gone)
    run(b, 2)


@pytest.mark.parametrize("workspace", [True, False])
def test_nan_rows_under_8_waves(gpu_device, workspace):
    """Keys and values that are not finite, seen by some rows and masked for others."""
    b = Batch(gpu_device, "128", [2600], [200], seed=58)
    b.append()
    pg = b.cache.page_table[0]
    b.cache.k_scales[0, int(pg[2700 // 64]), 0, 2700 % 64] = float("nan")  # key of new row 100, kv head 0
    b.cache.v_scales[0, int(pg[500 // 64]), 1, 500 % 64] = float("nan")  # kv head 1, seen without a window
    got = b.attend(workspace=workspace)
    G = b.hq // b.hkv * b.d
    assert not bool(torch.isnan(got[:100, :G]).any()) and bool(torch.isnan(got[100:, :G]).all())
    assert bool(torch.isnan(got[:, G:]).all())
    got = b.attend(workspace=workspace, window=2101)  # row 0 sees from position 500 on, row 1 from 501
    assert bool(torch.isnan(got[0, G:]).all()) and not bool(torch.isnan(got[1:, G:]).any())


# ---- graphs ------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,rows,most", [("128", 2, 5000), ("64", 1, 9000), ("128", 60, 5000), ("256g", 40, 5000)])
def test_replays_that_leave_ranges_empty(gpu_device, heads, rows, most):
    """A captured call of many ranges replayed with all of them in use, some and one: the
    workspace holds NaN or another call's partials before each."""
    dev = gpu_device
    b = Batch(dev, heads, [most, 300], [rows, rows], seed=59)
    c = b.cache
    rec = b.rec()
    for t in (c.k_scales, c.v_scales):
        t.nan_to_num_(0.01)
    out = torch.zeros(b.total, b.hq * b.d, dtype=torch.bfloat16, device=dev)
    a = b.args(out)
    assert ranges(b, rec, a) >= 4
    need = N.lib().dtree_attention_q8_workspace_bytes(C.byref(rec), C.byref(a))
    ws = torch.zeros(need, dtype=torch.uint8, device=dev)
    a.workspace = ws.data_ptr(); a.workspace_bytes = need
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = C.c_void_p()
    N.check(N.lib().dtree_graph_begin(side.cuda_stream), "begin")
    b.append(rec, side.cuda_stream)
    N.check(N.lib().dtree_attention_q8(C.byref(rec), C.byref(a), side.cuda_stream), "attention")
    N.check(N.lib().dtree_graph_end(side.cuda_stream, C.byref(g)), "end")
    try:
        for i, (past, n) in enumerate((([most, 300], [rows, rows]), ([1300, 20], [rows, rows]), ([0, 0], [rows, 1]),
                                       ([most, 0], [1, 0]), ([300, most], [rows, rows]), ([0, 5], [0, 0]),
                                       ([most, 300], [rows, rows]))):
            b.past, b.rows = past, n
            b.dpast.copy_(i32(past, dev))
            b.drows.copy_(i32(n, dev))
            out.fill_(7.0)
            if i % 2 == 0:
                ws.fill_(255)
            torch.cuda.synchronize()
            N.check(N.lib().dtree_graph_launch(g, stream()), "launch")
            torch.cuda.synchronize()
            got = out.clone()
            want, tol = b.reference()
            check(got, want, long_tol(b, tol), BF16, (past, n))
            assert torch.equal(got, b.attend(rec=rec))
    finally:
        N.lib().dtree_graph_destroy(g)
