"""Calls of the 8-bit cache's entries that their documentation allows beside the
ordinary ones: batches of trees, masks that leave rows empty, many query heads on
one KV head, addresses aligned to their type alone, shared pages, empty batches."""
import ctypes as C

import pytest
import torch

from dtree_hip import _native as N
from dtree_hip.cache import PAGE
from dtree_hip.engine import ancestor_bitsets

import test_gpu_kv_q8 as base
from gpu_util import random_tree, stream
from test_gpu_kv_q8 import BF16, PAIR, Batch, check, i32

pytestmark = pytest.mark.gpu


@pytest.fixture
def heads(request, monkeypatch):
    """A head layout of the test's own: (q heads, kv heads, head dim, rotary dims, gated)."""
    monkeypatch.setitem(base.HEADS, "own", request.param)
    return "own"


def words(trees, dev):
    """Ancestor words [rows][4] of trees one behind another."""
    return torch.cat([torch.from_numpy(ancestor_bitsets(t).astype("int64")) for t in trees]).to(torch.int32).to(dev).contiguous()


@pytest.mark.parametrize("layout", ["128", "256g", "64"])
@pytest.mark.parametrize("past,n", [([700, 0, 65], 40), ([300, 64, 5, 0], 4), ([2300, 2100], 100), ([0, 0], 1)])
def test_a_batch_of_draft_trees(gpu_device, layout, past, n):
    """Trees of their own over prefixes of their own."""
    b = Batch(gpu_device, layout, past, [n] * len(past), seed=61)
    b.append()
    trees = [random_tree(n, seed=s + 1) for s in range(len(past))]
    anc = words(trees, gpu_device)
    got = b.attend(ancestors=anc.data_ptr(), pair=True)
    one = b.attend(ancestors=anc.data_ptr(), pair=True, workspace=False)
    for s, t in enumerate(trees):
        want, tol = b.reference(parents=t)
        rows = slice(s * n, (s + 1) * n)
        check(got[rows], want[rows], tol[rows], PAIR, s)
        check(one[rows], want[rows], tol[rows], PAIR, s)


@pytest.mark.parametrize("layout", ["128", "256g"])
@pytest.mark.parametrize("past,n", [(0, 3), (0, 70), (130, 40)])
def test_tree_rows_without_a_key(gpu_device, layout, past, n):
    """Rows whose words are empty see the prefix alone, zeros if there is none; bits
    behind the last row mean nothing."""
    b = Batch(gpu_device, layout, [past], [n], seed=62)
    b.append()
    parents = random_tree(n, seed=3)
    anc = words([parents], gpu_device)
    none = torch.arange(n, device=gpu_device) % 3 == 1
    want, tol = b.reference(parents=parents)
    few, ftol = torch.zeros_like(want), torch.zeros_like(tol)
    if past:  # the prefix alone: as rows of a sequence that ends there, with a mask of nothing new
        b.past, b.rows = [past], [n]
        c, d = b.cache, b.d
        keep = anc.clone()
        keep[:] = 0
        alone = b.attend(ancestors=keep.data_ptr(), pair=True)
        qs = 2 * d if b.gated else d
        x = b.qkv[:, :b.hq * qs].double().view(n, b.hq, qs)
        q = base.norm_rope(x[..., :d], b.q_norm, b.cos, b.sin, b.rd)
        k, v = c.logical_keys(0, past).double(), c.logical_values(0, past).double()
        for h in range(b.hq):
            g = h // (b.hq // b.hkv)
            w = torch.softmax(q[:, h] @ k[:, g].T.contiguous() * d ** -0.5, -1)
            o = w @ v[:, g]
            E = 2.0 ** -11 * d ** -0.5 * (q[:, h].abs() @ k[:, g].abs().T.contiguous()).amax(-1, keepdim=True)
            t = (w @ v[:, g].abs()) * (torch.expm1(2 * E) + 2.0 ** -16 + 2.0 ** -11)
            t = t + 127 * past * 2.0 ** -31 * v[:, g].abs().max() / 127
            gate = torch.sigmoid(x[:, h, d:]) if b.gated else 1.0
            few[:, h * d:(h + 1) * d], ftol[:, h * d:(h + 1) * d] = o * gate, t * gate
        check(alone, few, ftol, PAIR, "prefix alone")
    anc[none] = 0
    if n < 128:  # (node bits from n on)
        for w in range(4):
            high = 0xffffffff if 32 * w >= n else (0xffffffff << (n - 32 * w)) & 0xffffffff if 32 * w + 32 > n else 0
            anc[:, w] |= high - (1 << 32) if high >= 1 << 31 else high
    want[none], tol[none] = few[none], ftol[none]
    got = b.attend(ancestors=anc.data_ptr(), pair=True)
    check(got, want, tol, PAIR)
    if not past:
        assert bool((got[none] == 0).all())


@pytest.mark.parametrize("heads", [(64, 1, 64, 64, False), (40, 1, 128, 0, True), (33, 1, 256, 32, False),
                                   (14, 2, 128, 64, True), (24, 8, 64, 32, True), (256, 2, 64, 0, False)], indirect=True)
@pytest.mark.parametrize("past,rows", [([200], [1]), ([77, 0, 1500], [3, 50, 1]), ([2200], [33])])
def test_other_head_layouts(gpu_device, heads, past, rows):
    """Groups that are no power of two or larger than a workgroup's rows, gated heads of every size."""
    b = Batch(gpu_device, heads, past, rows, seed=63, pad=1)
    want = b.append_reference()
    b.append()
    assert torch.equal(b.cache.k_pages, want[0]) and torch.equal(b.cache.v_pages, want[1])
    want, tol = b.reference()
    check(b.attend(pair=True), want, tol, PAIR)
    want, tol = b.reference(sink=7, window=100)
    check(b.attend(sink=7, window=100), want, tol, BF16, "window")


def moved(t, elements):
    """The tensor `elements` elements behind a 256-byte boundary."""
    big = torch.empty(t.numel() + elements + 64, dtype=t.dtype, device=t.device)
    at = big[elements:elements + t.numel()].view(t.shape)
    at.copy_(t)
    return at


@pytest.mark.parametrize("layout", ["128", "256g", "64"])
@pytest.mark.parametrize("past,rows", [([300], [1]), ([300, 20], [40, 2])])
def test_addresses_aligned_to_their_type_alone(gpu_device, layout, past, rows):
    """Norm weights and tables at any address of their type, outputs at 8 bytes."""
    b = Batch(gpu_device, layout, past, rows, seed=64)
    ref = Batch(gpu_device, layout, past, rows, seed=64)
    b.q_norm, b.k_norm = moved(b.q_norm, 3), moved(b.k_norm, 1)
    b.cos, b.sin = moved(b.cos, 1), moved(b.sin, 3)
    b.append()
    ref.append()
    assert torch.equal(b.cache.k_pages, ref.cache.k_pages) and torch.equal(b.cache.v_pages, ref.cache.v_pages)
    W = b.hq * b.d
    out = torch.full((b.total * (W + 4) + 8,), 7.0, dtype=torch.bfloat16, device=gpu_device)
    rec = b.rec()
    a = b.args(out, ld_out=W + 4)
    a.out = out.data_ptr() + 8
    need = N.lib().dtree_attention_q8_workspace_bytes(C.byref(rec), C.byref(a))
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=gpu_device)
    a.workspace = ws.data_ptr(); a.workspace_bytes = need
    N.check(N.lib().dtree_attention_q8(C.byref(rec), C.byref(a), stream()), "attention")
    rows_ = out[4:4 + b.total * (W + 4)].view(b.total, W + 4)
    assert torch.equal(rows_[:, :W], ref.attend()) and bool((rows_[:, W:] == 7).all()) and bool((out[:4] == 7).all())


@pytest.mark.parametrize("rows", [1, 40])
def test_sequences_that_share_a_prefix(gpu_device, rows):
    """Pages that several sequences read and no call writes."""
    past = 5 * PAGE
    b = Batch(gpu_device, "128", [past] * 3, [rows] * 3, seed=65)
    c = b.cache
    c.page_table[1:, :5] = c.page_table[0, :5]
    b.append()
    check(b.attend(pair=True), *b.reference(), PAIR)


@pytest.mark.parametrize("max_rows", [1, 40])
def test_batches_without_rows(gpu_device, max_rows):
    """Nothing is written, but for rows that are to be cleared."""
    b = Batch(gpu_device, "128", [100, 300], [1, 1], seed=66)
    b.drows.copy_(i32([0, 0], gpu_device))
    before = [t.clone() for t in (b.cache.k_pages, b.cache.v_pages)]
    rec = b.rec(max_rows=max_rows)
    b.append(rec)
    assert torch.equal(b.cache.k_pages, before[0]) and torch.equal(b.cache.v_pages, before[1])
    assert bool((b.attend(rec=rec) == 7).all())
    b = Batch(gpu_device, "128", [300], [max_rows], seed=66)
    b.drows.copy_(i32([0], gpu_device))
    out = b.attend(rec=b.rec(row_starts=None), rows_padded=b.total)
    assert bool((out == 0).all())
