"""The 8-bit paged KV cache: rows written, read back and moved, and the
attention over it, against plain 64-bit forms.

Bytes and scales are compared for equality: both sides take q as the integer
nearest to x / scale from values that are exact to 1e-15.

The attention's tolerance, per element, counts these roundings (A = sum_j w_j
|v_j|, w the exact softmax weights, u_j = 2^(t_j - m) as in the kernel):
* q to fp16: at most 2^-11 of each element, so a logit is off by at most
  E = 2^-11 scale sum_d |q_d k_d| (natural units), and a normalised weighted
  mean by at most (e^(2E) - 1) A;
* fp32 on the way to it (norm, rotation, products, exponents): 2^-16 A;
* the weights to fp16: 2^-11 A, and 2^-25 of a subnormal u_j, of which the
  largest is at least 2^6: 127 n 2^-31 max_j(w_j vs_j), vs the value scales;
* the output: 2^-8 of the element in bf16, 2^-16 as a pair hi + lo, 2^-11 in fp16."""
import ctypes as C

import pytest
import torch

from dtree_hip import _native as N
from dtree_hip.cache import PAGE, PagedKVCacheQ8, _block_index_q8, quantise_q8

from gpu_util import device_desc, random_tree, stream

pytestmark = pytest.mark.gpu
F64 = torch.float64
EPS = 1e-6
# q heads, kv heads, head dim, rotary dims, gated
HEADS = {"128": (8, 2, 128, 128, False), "256g": (4, 2, 256, 64, True), "64": (6, 2, 64, 32, False),
         "128x1": (5, 5, 128, 96, False), "256": (8, 1, 256, 256, False), "mqa": (16, 1, 64, 0, False)}


def gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def norm_rope(x, w, cos, sin, rd):
    """[rows, heads, D] in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    if rd:
        c, s = cos.double()[:, None], sin.double()[:, None]
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        x = torch.cat([a * c - b * s, a * s + b * c, x[..., rd:]], -1)
    return x


class Batch:
    """A cache of garbage (stale bytes, NaN scales) with sequences written into
    it, and the projections of their new rows."""

    def __init__(self, dev, heads, past, rows, *, typ=torch.float32, seed=0, starts=None, pad=0, norm=True, spread=0.0,
                 extra_pages=0):
        self.dev, self.past, self.rows = dev, past, rows
        self.hq, self.hkv, self.d, self.rd, self.gated = HEADS[heads]
        g = gen(dev, seed)
        d, hkv = self.d, self.hkv
        S = len(past)
        cap = max(p + n for p, n in zip(past, rows)) + extra_pages * PAGE
        pages = S * ((max(cap, 1) + PAGE - 1) // PAGE)
        c = PagedKVCacheQ8(1, hkv, d, max(cap, 1), S, device=dev,
                           page_order=torch.randperm(pages, generator=torch.Generator().manual_seed(seed)))
        c.k_pages.random_(-127, 128, generator=g)
        c.v_pages.random_(-127, 128, generator=g)
        c.k_scales.fill_(float("nan"))
        c.v_scales.fill_(float("nan"))
        self.cache = c
        self.k, self.v = [], []
        for s in range(S):
            def rows_(n):
                x = torch.randn(n, hkv, d, generator=g, device=dev)
                return x * torch.exp(spread * torch.randn(n, hkv, 1, generator=g, device=dev))
            if past[s]:
                c.write_logical(0, rows_(past[s]), 0.5 * rows_(past[s]), 0, s)
        self.starts = list(starts) if starts is not None else [sum(rows[:s]) for s in range(S)]
        self.total = max(s + n for s, n in zip(self.starts, rows)) + pad
        self.total = max(self.total, 1)
        qs = 2 * d if self.gated else d
        self.width = self.hq * qs + 2 * hkv * d + 8
        self.qkv = torch.randn(self.total, self.width, generator=g, device=dev).to(typ)
        self.koff = self.hq * qs
        self.q_norm = (1.2 + 0.1 * torch.randn(d, generator=g, device=dev)).bfloat16() if norm else None
        self.k_norm = (1.2 + 0.1 * torch.randn(d, generator=g, device=dev)).bfloat16() if norm else None
        pos = torch.zeros(self.total, dtype=F64, device=dev)
        for s in range(S):
            pos[self.starts[s]:self.starts[s] + rows[s]] = torch.arange(past[s], past[s] + rows[s], device=dev).double()
        ang = pos[:, None] * 1e4 ** (-torch.arange(0, max(self.rd, 2), 2, device=dev, dtype=F64) / max(self.rd, 2))
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        self.dpast, self.drows, self.dstarts = i32(past, dev), i32(rows, dev), i32(self.starts, dev)
        self.max_past, self.max_rows = max(past), max(max(rows), 1)

    def rec(self, **kw):
        a = dict(max_past_length=self.max_past, max_rows=self.max_rows, total_rows=self.total, row_starts=self.dstarts)
        a.update(kw)
        return self.cache.record(0, self.dpast, self.drows, **a)

    def new_kv(self):
        x = self.qkv[:, self.koff:self.koff + 2 * self.hkv * self.d].double().view(self.total, 2, self.hkv, self.d)
        return norm_rope(x[:, 0], self.k_norm, self.cos, self.sin, self.rd), x[:, 1]

    def append(self, rec=None, st=None):
        size = self.qkv.element_size()
        k = self.qkv.data_ptr() + self.koff * size
        typ = N.T_BF16 if self.qkv.dtype == torch.bfloat16 else N.T_F32
        rec = self.rec() if rec is None else rec
        N.check(N.lib().dtree_kv_q8_append(
            C.byref(rec), k, k + self.hkv * self.d * size, typ, self.width, self.width,
            self.k_norm.data_ptr() if self.k_norm is not None else None, EPS, self.cos.data_ptr(),
            self.sin.data_ptr(), self.rd, stream() if st is None else st), "append")

    def append_reference(self):
        """The pools after the append, by the definition."""
        c = self.cache
        k, v = self.new_kv()
        want = [t.clone() for t in (c.k_pages, c.v_pages, c.k_scales, c.v_scales)]
        for s, (p, n, at) in enumerate(zip(self.past, self.rows, self.starts)):
            for i in range(n):
                page, slot = int(c.page_table[s, (p + i) // PAGE]), (p + i) % PAGE
                if not 0 <= page < c.n_pages:
                    continue
                for j, (x, which) in enumerate(((k, "k"), (v, "v"))):
                    q, scale = quantise_q8(x[at + i])
                    off = _block_index_q8(self.d, which).to(self.dev)[slot]
                    want[j][0, page][:, off] = q
                    want[2 + j][0, page, :, slot] = scale
        return want

    def args(self, out, **kw):
        a = N.AttnQ8Args()
        a.q = self.qkv.data_ptr(); a.ld_q = self.width; a.q_stride = 2 * self.d if self.gated else self.d
        a.q_type = N.T_BF16 if self.qkv.dtype == torch.bfloat16 else N.T_F32
        a.q_norm = self.q_norm.data_ptr() if self.q_norm is not None else None; a.eps = EPS
        a.rope_cos = self.cos.data_ptr(); a.rope_sin = self.sin.data_ptr(); a.rope_dims = self.rd
        a.out = out.data_ptr(); a.ld_out = self.hq * self.d; a.out_layout = N.W_ROWMAJOR
        a.num_heads = self.hq; a.scale = self.d ** -0.5; a.gated = int(self.gated)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    def attend(self, *, workspace=True, pair=False, rec=None, st=None, **kw):
        """Fills `out` with 7 (a low half with 0) first: rows of no sequence have to keep it."""
        out = torch.zeros(2, self.total, self.hq * self.d, dtype=torch.bfloat16, device=self.dev)
        out[0] = 7.0
        rec = self.rec() if rec is None else rec
        a = self.args(out[0], **kw)
        if pair:
            a.out_lo = out[1].data_ptr()
        if workspace:
            need = N.lib().dtree_attention_q8_workspace_bytes(C.byref(rec), C.byref(a))
            need = need if workspace is True else min(need, int(workspace))
            ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=self.dev)
            a.workspace = ws.data_ptr(); a.workspace_bytes = need
            self.ws = ws
        N.check(N.lib().dtree_attention_q8(C.byref(rec), C.byref(a), stream() if st is None else st), "attention")
        return out.double().sum(0) if pair else out[0]

    def reference(self, *, sink=0, window=0, parents=None):
        """(output, tolerance without the output's rounding) in 64 bits, 7 in rows of no sequence."""
        c, d, hq = self.cache, self.d, self.hq
        G = hq // self.hkv
        qs = 2 * d if self.gated else d
        x = self.qkv[:, :hq * qs].double().view(self.total, hq, qs)
        q = norm_rope(x[..., :d], self.q_norm, self.cos, self.sin, self.rd)
        out = torch.full((self.total, hq, d), 7.0, dtype=F64, device=self.dev)
        tol = torch.zeros_like(out)
        for s, (p, n, at) in enumerate(zip(self.past, self.rows, self.starts)):
            if not n:
                continue
            T = p + n
            table = c.page_table[s, :(T + PAGE - 1) // PAGE]
            gone = ((table < 0) | (table >= c.n_pages)).repeat_interleave(PAGE)[:T]
            keep = c.page_table.clone()
            c.page_table[s] = c.page_table[s].clamp(0, c.n_pages - 1)
            k, v = c.logical_keys(0, T, s).double(), c.logical_values(0, T, s).double()
            pages = c.page_table[s, :(T + PAGE - 1) // PAGE].long()
            vs = c.v_scales[0][pages].permute(0, 2, 1).reshape(-1, self.hkv)[:T].double()
            c.page_table.copy_(keep)
            j = torch.arange(T, device=self.dev)
            pos = torch.arange(p, T, device=self.dev)[:, None]
            if parents is None:
                see = (j <= pos) & ((j < sink) | (pos - j < window) if window else torch.ones_like(j, dtype=torch.bool))
            else:
                see = (j < p).expand(n, T).clone()
                for i, par in enumerate(parents):
                    if par >= 0:
                        see[i, p:] = see[par, p:]
                    see[i, p + i] = True
            see = see & ~gone
            any_ = see.any(-1)
            dead = ~see.any(0)  # keys that no row sees: their values do not count, whatever they are
            k, v, vs = (torch.where(dead.view(-1, *[1] * (t.dim() - 1)), 0.0, t) for t in (k, v, vs))
            for h in range(hq):
                kk, vv, sc = k[:, h // G], v[:, h // G], vs[:, h // G]
                qq = q[at:at + n, h]
                lg = (qq @ kk.T.contiguous()) * d ** -0.5
                lg = lg.masked_fill(~see, float("-inf"))
                lg = torch.where(any_[:, None], lg, 0.0)
                w = torch.softmax(lg, -1) * any_[:, None]
                o = w @ vv
                E = 2.0 ** -11 * d ** -0.5 * torch.where(see, qq.abs() @ kk.abs().T.contiguous(), 0.0).amax(-1, keepdim=True)
                A = w @ vv.abs()
                t = A * (torch.expm1(2 * E) + 2.0 ** -16 + 2.0 ** -11)
                t = t + 127 * T * 2.0 ** -31 * (w * sc).amax(-1, keepdim=True)
                if self.gated:
                    gate = torch.sigmoid(x[at:at + n, h, d:])
                    o, t = o * gate, t * gate
                out[at:at + n, h] = o
                tol[at:at + n, h] = t
        return out.reshape(self.total, -1), tol.reshape(self.total, -1)


def check(got, want, tol, rounding, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    # sums of the tolerance's own evaluation and of fp32 division: a ten-thousandth more
    lim = 1.0001 * (tol + rounding * (want.abs() + tol)) + 1e-30
    bad = ((got - want).abs() > lim) & ~torch.isnan(want)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / lim)[~torch.isnan(want)].max()))


BF16, PAIR, FP16 = 2.0 ** -8, 2.0 ** -16, 2.0 ** -11


# ---- writing and reading ---------------------------------------------------------
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("past,rows", [([0], [1]), ([63], [2]), ([37], [200]), ([5, 0, 130, 64], [1, 64, 0, 65]),
                                       ([0, 17], [130, 3])])
def test_append_stores_the_definitions_bytes(gpu_device, heads, typ, past, rows):
    b = Batch(gpu_device, heads, past, rows, typ=typ, seed=len(past) + rows[0])
    want = b.append_reference()
    b.append()
    c = b.cache
    for got, w, what in zip((c.k_pages, c.v_pages, c.k_scales, c.v_scales), want, ("k", "v", "k scale", "v scale")):
        assert torch.equal(torch.nan_to_num(got, nan=-1.0) if got.is_floating_point() else got,
                           torch.nan_to_num(w, nan=-1.0) if w.is_floating_point() else w), what


def test_append_without_norm_rope_or_starts(gpu_device):
    b = Batch(gpu_device, "mqa", [3, 70], [9, 9], norm=False, seed=2)
    assert b.starts == [0, 9]  # s * max_rows
    want = b.append_reference()
    b.append(b.rec(row_starts=None))
    assert torch.equal(b.cache.k_pages, want[0]) and torch.equal(b.cache.v_pages, want[1])


def test_append_rows_that_are_not_finite_zero_or_huge(gpu_device):
    b = Batch(gpu_device, "128", [10], [6], norm=False, seed=3)
    x = b.qkv[:, b.koff:]
    x[0, 5] = float("inf")
    x[1, 3] = float("nan")
    x[2, :2 * b.hkv * b.d] = 0.0
    x[3, :2 * b.hkv * b.d] *= 1e30
    x[4, :2 * b.hkv * b.d] *= 1e-30
    b.cos.fill_(1.0)
    b.sin.fill_(0.0)
    want = b.append_reference()
    b.append()
    c = b.cache
    assert torch.equal(c.k_pages, want[0]) and torch.equal(c.v_pages, want[1])
    for got, w in ((c.k_scales, want[2]), (c.v_scales, want[3])):
        assert torch.equal(torch.isnan(got), torch.isnan(w))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(w))
    k = c.logical_keys(0, 16)[10:]
    assert bool(torch.isnan(k[0, 0]).all()) and bool(torch.isnan(k[1, 0]).all()) and bool((k[2] == 0).all())


def test_append_keeps_to_its_bounds(gpu_device):
    """Device lengths beyond the host's bounds, starts outside the rows, absent pages: skipped or clipped."""
    dev = gpu_device
    b = Batch(dev, "128", [5, 6, 7, 64, 8, 250], [4, 4, 4, 70, 4, 3], seed=4)
    c = b.cache
    assert c.capacity == 256
    c.page_table[3, 1] = -1                 # the page of sequence 3's positions 64 .. 127
    c.page_table[3, 2] = c.n_pages + 5
    b.dpast[0] = 1 << 20                    # past the bound: no rows
    b.drows[5] = 50                         # rows past the table's last position: 250 .. 255 alone
    b.dstarts[1] = -3                       # a start before the buffer: no rows
    b.drows[2] = 1 << 20                    # more rows than max_rows: here clipped at max_rows ...
    b.dstarts[4] = b.total - 2              # ... and at the buffer's end
    b.dstarts[5] = 20
    ref = Batch(dev, "128", [5, 6, 7, 64, 8, 250], [4, 4, 4, 70, 4, 3], seed=4)
    ref.cache.page_table.copy_(c.page_table)
    ref.rows = [0, 0, 70, 70, 2, 6]
    ref.starts = [0, 0, b.starts[2], b.starts[3], b.total - 2, 20]
    want = ref.append_reference()
    b.append()
    assert torch.equal(c.k_pages, want[0]) and torch.equal(c.v_pages, want[1])


@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first,rows", [([0], [1]), ([0], [200]), ([60, 0, 129], [70, 0, 1])])
def test_read_gives_the_values_rows_stand_for(gpu_device, heads, out, first, rows):
    dev = gpu_device
    b = Batch(dev, heads, [p + n for p, n in zip(first, rows)], [1] * len(rows), seed=7)
    b.dpast, b.drows = i32(first, dev), i32(rows, dev)
    starts = [sum(rows[:s]) + s for s in range(len(rows))]  # a row between sequences
    total = sum(rows) + len(rows)
    w = b.hkv * b.d
    k = torch.full((total, w + 8), 7.0, dtype=out, device=dev)
    v = torch.full((total, w + 16), 7.0, dtype=out, device=dev)
    rec = b.cache.record(0, b.dpast, b.drows, max(first), max(rows), total, i32(starts, dev))
    typ = N.T_F32 if out == torch.float32 else N.T_BF16
    N.check(N.lib().dtree_kv_q8_read(C.byref(rec), k.data_ptr(), v.data_ptr(), typ, w + 8, w + 16, stream()), "read")
    wk, wv = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    for s, (p, n, at) in enumerate(zip(first, rows, starts)):
        wk[at:at + n, :w] = b.cache.logical_keys(0, p + n, s)[p:].reshape(n, w).to(out)
        wv[at:at + n, :w] = b.cache.logical_values(0, p + n, s)[p:].reshape(n, w).to(out)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    only = torch.full_like(v, 7.0)  # one of the two alone
    N.check(N.lib().dtree_kv_q8_read(C.byref(rec), None, only.data_ptr(), typ, 0, w + 16, stream()), "read")
    assert torch.equal(only, wv)


def test_read_of_absent_pages_and_nan_rows(gpu_device):
    dev = gpu_device
    b = Batch(dev, "128", [200], [1], seed=8)
    b.cache.page_table[0, 1] = -1
    b.cache.k_scales[0, int(b.cache.page_table[0, 2]), 0, 3] = float("nan")
    k = torch.full((200, b.hkv * b.d), 7.0, device=dev)
    v = torch.full_like(k, 7.0)
    rec = b.cache.record(0, i32([0], dev), i32([200], dev), 0, 200, 200)
    N.check(N.lib().dtree_kv_q8_read(C.byref(rec), k.data_ptr(), v.data_ptr(), N.T_F32, k.shape[1], k.shape[1],
                                     stream()), "read")
    assert bool((k[64:128] == 0).all()) and bool((v[64:128] == 0).all())
    assert bool(torch.isnan(k[131, :b.d]).all()) and int(torch.isnan(k).sum()) == b.d


# ---- attention --------------------------------------------------------------------
SHAPES = [
    ([0], [1]), ([63], [1]), ([64], [1]), ([1000], [1]), ([517, 3, 0, 2000], [1, 1, 1, 1]), ([300, 40], [3, 1]),
    ([0], [33]), ([100], [64]), ([0], [300]), ([700], [129]), ([700, 5, 0, 64], [70, 1, 0, 200]),
]


@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("past,rows", SHAPES)
def test_attention_causal(gpu_device, heads, past, rows):
    b = Batch(gpu_device, heads, past, rows, seed=11, pad=2)
    b.append()
    want, tol = b.reference()
    check(b.attend(), want, tol, BF16, "workspace")
    if rows in ([1], [129]):
        check(b.attend(pair=True), want, tol, PAIR, "pair")
    one = b.attend(workspace=False)
    check(one, want, tol, BF16, "no workspace")
    assert torch.equal(one, b.attend(workspace=False)) and torch.equal(b.attend(), b.attend())  # bit for bit


@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("pairs", [1, 32])
def test_attention_of_many_sequences(gpu_device, heads, pairs):
    """More workgroups than CUs (fewer waves each): one row a sequence, and up to 32 pairs."""
    hq, hkv = HEADS[heads][:2]
    S, n = 256 // hkv + 5, max(1, pairs // (hq // hkv))
    past = [(37 * s) % 150 for s in range(S)]
    rows = [1 + s % n for s in range(S)]
    b = Batch(gpu_device, heads, past, rows, seed=17)
    b.append()
    want, tol = b.reference()
    check(b.attend(), want, tol, BF16)
    want, tol = b.reference(sink=3, window=70)
    check(b.attend(sink=3, window=70), want, tol, BF16, "window")


@pytest.mark.parametrize("heads", ["128", "256g", "64"])
@pytest.mark.parametrize("sink,window", [(0, 1), (1, 1), (0, 64), (4, 100), (64, 65), (70, 257), (0, 5000), (5000, 3)])
@pytest.mark.parametrize("past,rows", [([900], [1]), ([900, 30, 64], [1, 1, 1]), ([0], [200]), ([450], [140]),
                                       ([600, 0, 10], [2, 90, 1])])
def test_attention_window_and_sinks(gpu_device, heads, sink, window, past, rows):
    b = Batch(gpu_device, heads, past, rows, seed=12, pad=1)
    b.append()
    want, tol = b.reference(sink=sink, window=window)
    check(b.attend(sink=sink, window=window), want, tol, BF16)


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,past,rows", [("128", [300], [1]), ("256g", [129, 5], [40, 1])])
def test_attention_bf16_projections(gpu_device, heads, past, rows, typ):
    b = Batch(gpu_device, heads, past, rows, typ=typ, seed=13)
    b.append()
    check(b.attend(pair=True), *b.reference(), PAIR)


@pytest.mark.parametrize("heads", ["128", "256g", "64"])
@pytest.mark.parametrize("nodes,past", [(1, 0), (2, 70), (25, 1000), (33, 0), (65, 129), (128, 700)])
def test_attention_draft_tree(gpu_device, heads, nodes, past):
    b = Batch(gpu_device, heads, [past], [nodes], seed=14, pad=3)
    parents = random_tree(nodes, seed=nodes)
    b.append()
    desc = device_desc([0] * nodes, [past] * nodes, parents, past, gpu_device)
    anc = desc.data_ptr() + N.StepDesc.ancestors.offset
    # lengths straight from the step descriptor, as a captured step has them
    rec = b.cache.record(0, desc.data_ptr() + N.StepDesc.past_length.offset, desc.data_ptr() + N.StepDesc.num_nodes.offset,
                         past, max(nodes, 2), b.total)
    want, tol = b.reference(parents=parents)
    check(b.attend(ancestors=anc, rec=rec), want, tol, BF16)
    got = b.attend(ancestors=anc, rec=rec, rows_padded=b.total)
    want[nodes:] = 0
    check(got, want, tol, BF16, "padded")


@pytest.mark.parametrize("heads,past,rows", [("128", [130], [1]), ("128", [130], [50]), ("256g", [70], [33])])
def test_attention_output_layouts(gpu_device, heads, past, rows):
    dev = gpu_device
    b = Batch(dev, heads, past, rows, seed=15)
    b.total = 64
    b.qkv = torch.cat([b.qkv, torch.zeros(64 - len(b.qkv), b.width, device=dev)])
    b.cos, b.sin = (torch.cat([t, torch.zeros(64 - len(t), t.shape[1], device=dev)]) for t in (b.cos, b.sin))
    b.append()
    want, tol = b.reference()
    want[rows[0]:] = 0
    W = b.hq * b.d
    r, k = torch.arange(64, device=dev)[:, None], torch.arange(W, device=dev)[None]
    at = ((((r >> 5) * (W >> 6) + (k >> 6)) * 4 + ((k & 31) >> 3)) * 512 + ((r & 31) + 32 * ((k & 63) >> 5)) * 8 + (k & 7))
    for layout, dt, rounding in ((N.W_TILED, torch.bfloat16, PAIR), (N.W_TILED_F16, torch.float16, FP16)):
        out = torch.full((2, 64 * W), 7.0, dtype=dt, device=dev)
        a = b.args(out[0], out_layout=layout, out_lo=out[1].data_ptr(), rows_padded=64)
        rec = b.rec(row_starts=None, max_rows=rows[0])
        N.check(N.lib().dtree_attention_q8(C.byref(rec), C.byref(a), stream()), "attention")
        got = out[0].double() + (out[1].double() if layout == N.W_TILED else 0)
        if layout == N.W_TILED_F16:
            assert bool((out[1] == 7.0).all())  # one plane
        check(got[at], want, tol + 2.0 ** -25, rounding, str(layout))


@pytest.mark.parametrize("past,rows", [([900], [1]), ([500], [100])])
def test_attention_scales_far_apart(gpu_device, past, rows):
    """Rows of 1e-6 to 1e6: a weight's exponent takes the value scale with it."""
    b = Batch(gpu_device, "128", past, rows, seed=16, spread=5.0, norm=False)
    b.qkv *= torch.exp(2 * torch.randn(b.total, 1, generator=gen(gpu_device, 1), device=gpu_device))
    b.qkv[:, :b.koff] *= 0.01
    b.append()
    check(b.attend(pair=True), *b.reference(), PAIR)


def test_attention_of_zero_queries_zero_values_and_one_key(gpu_device):
    dev = gpu_device
    b = Batch(dev, "128", [100, 0], [1, 1], seed=17, norm=False)
    b.qkv[0, :b.koff] = 0.0  # all keys alike
    b.qkv[1, b.koff + b.hkv * b.d:] = 0.0  # the only value row is zero
    b.append()
    want, tol = b.reference()
    got = b.attend(pair=True)
    check(got, want, tol, PAIR)
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("rows", [1, 60])
def test_attention_absent_pages_and_rows_that_see_nothing(gpu_device, rows):
    dev = gpu_device
    b = Batch(dev, "128", [200, 130], [rows, rows], seed=18)
    b.append()
    b.cache.page_table[0, 0] = -1
    b.cache.page_table[0, 2] = b.cache.n_pages
    b.cache.page_table[1, :] = -7
    want, tol = b.reference()
    assert bool((want[rows:] == 0).all())
    check(b.attend(), want, tol, BF16)
    # under a window the pages before it are never read
    b = Batch(dev, "128", [400], [rows], seed=19)
    b.append()
    want, tol = b.reference(sink=3, window=100)
    b.cache.page_table[0, 1:4] = -1
    check(b.attend(sink=3, window=100), want, tol, BF16)


@pytest.mark.parametrize("rows", [1, 60])
def test_attention_nan_stays_where_it_is_seen(gpu_device, rows):
    dev = gpu_device
    b = Batch(dev, "128", [200], [rows], seed=20)
    b.append()
    pg = b.cache.page_table[0]
    b.cache.k_scales[0, int(pg[1]), 0, 5] = float("nan")  # key 69 of kv head 0
    b.cache.v_scales[0, int(pg[2]), 1, 9] = float("nan")  # value 137 of kv head 1
    got = b.attend()
    assert bool(torch.isnan(got).all())
    got = b.attend(sink=10, window=200 - 70)  # row 0 sees from 71 on
    G = b.hq // b.hkv * b.d
    assert not bool(torch.isnan(got[:, :G]).any()) and bool(torch.isnan(got[0, G:]).all())
    # and a query that is not finite spoils its own head and row alone
    b = Batch(dev, "128", [200], [rows], seed=21, norm=False)
    b.append()
    want, tol = b.reference()
    b.qkv[0, 0] = float("inf")
    b.qkv[rows - 1, b.d + 1] = float("nan")
    got = b.attend()
    bad = torch.zeros_like(want, dtype=torch.bool)
    bad[0, :b.d] = True
    bad[rows - 1, b.d:2 * b.d] = True
    assert bool(torch.isnan(got)[bad].all()) and not bool(torch.isnan(got)[~bad].any())
    got = torch.where(bad, 0.0, got.double())
    # the largest finite query of a workgroup sets the others' fp16 exponent: none here
    check(got, torch.where(bad, 0.0, want), tol, BF16)


def test_attention_with_less_workspace(gpu_device):
    for past, rows in ([5000], [1]), ([3000], [40]):
        b = Batch(gpu_device, "128", past, rows, seed=22)
        b.append()
        want, tol = b.reference()
        row = b.total * b.hq * (b.d + 2) * 4
        for parts in (0, 1, 2, 3, 5):
            check(b.attend(workspace=max(parts * row, 8)), want, tol, BF16, parts)


def test_attention_offsets_past_32_bits(gpu_device):
    """A pool of over 2^32 bytes of K, the sequence's pages at its end."""
    dev = gpu_device
    hkv, d = 8, 256
    pages = (1 << 32) // (hkv * PAGE * d) + 8
    b = Batch(dev, "256", [150], [20], seed=23)
    HEADS["tmp"] = (8, hkv, d, 64, False)
    try:
        b = Batch(dev, "tmp", [150], [20], seed=23)
    finally:
        del HEADS["tmp"]
    small = b.cache
    big = PagedKVCacheQ8.__new__(PagedKVCacheQ8)
    big.__dict__.update(small.__dict__)
    big.n_pages = pages
    big.k_pages = torch.empty(1, pages, hkv, PAGE * d, dtype=torch.int8, device=dev)
    big.v_pages = torch.empty_like(big.k_pages)
    big.k_scales = torch.empty(1, pages, hkv, PAGE, device=dev)
    big.v_scales = torch.empty_like(big.k_scales)
    big.page_table = torch.arange(pages - 1, pages - 4, -1, dtype=torch.int32, device=dev)[None].contiguous()
    for s in range(3):
        for a, z in ((big.k_pages, small.k_pages), (big.v_pages, small.v_pages), (big.k_scales, small.k_scales),
                     (big.v_scales, small.v_scales)):
            a[0, int(big.page_table[0, s])] = z[0, int(small.page_table[0, s])]
    b.append()
    want = b.attend()
    b.cache = big
    b.append()
    assert torch.equal(b.attend(), want)
    k = torch.zeros(170, hkv * d, device=dev)
    rec = big.record(0, i32([0], dev), i32([170], dev), 0, 170, 170)
    N.check(N.lib().dtree_kv_q8_read(C.byref(rec), k.data_ptr(), None, N.T_F32, hkv * d, 0, stream()), "read")
    assert torch.equal(k, small.logical_keys(0, 170).reshape(170, -1))


def test_graph_replays_follow_the_device_lengths(gpu_device):
    """One captured append + attention serves every length; the workspace comes back dirty."""
    dev = gpu_device
    b = Batch(dev, "128", [900, 100], [2, 2], seed=24)
    rec = b.rec()
    out = torch.zeros(b.total, b.hq * b.d, dtype=torch.bfloat16, device=dev)
    a = b.args(out)
    need = N.lib().dtree_attention_q8_workspace_bytes(C.byref(rec), C.byref(a))
    ws = torch.zeros(max(need, 16), dtype=torch.uint8, device=dev)
    a.workspace = ws.data_ptr(); a.workspace_bytes = need
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = C.c_void_p()
    N.check(N.lib().dtree_graph_begin(side.cuda_stream), "begin")
    b.append(rec, side.cuda_stream)
    N.check(N.lib().dtree_attention_q8(C.byref(rec), C.byref(a), side.cuda_stream), "attention")
    N.check(N.lib().dtree_graph_end(side.cuda_stream, C.byref(g)), "end")
    try:
        for past, rows in ([900, 100], [2, 2]), ([3, 40], [1, 2]), ([640, 100], [2, 0]), ([900, 100], [2, 2]):
            b.past, b.rows = past, rows
            b.dpast.copy_(i32(past, dev))
            b.drows.copy_(i32(rows, dev))
            c = b.cache
            for t in (c.k_scales, c.v_scales):
                t.nan_to_num_(0.01)
            out.fill_(7.0)
            ws.fill_(255)
            torch.cuda.synchronize()
            N.check(N.lib().dtree_graph_launch(g, stream()), "launch")
            torch.cuda.synchronize()
            got = out.clone()
            eager = b.attend()
            assert torch.equal(got, eager)
            check(got, *b.reference(), BF16)
    finally:
        N.lib().dtree_graph_destroy(g)


def test_two_streams_with_their_own_workspaces(gpu_device):
    batches = [Batch(gpu_device, "128", [2000], [1], seed=s) for s in (25, 26)]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    outs = []
    for b, st in zip(batches, streams):
        with torch.cuda.stream(st):
            b.append(st=st.cuda_stream)
            outs.append(b.attend(st=st.cuda_stream))
    torch.cuda.synchronize()
    for b, o in zip(batches, outs):
        check(o, *b.reference(), BF16)


# ---- a run of them, as they are used ------------------------------------------------
@pytest.mark.parametrize("heads", ["128", "256g", "64"])
def test_tree_step_then_compaction_then_a_token(gpu_device, heads):
    """Draft tree appended and attended, its accepted path compacted, the next
    token decoded: as if the accepted tokens had come one after another."""
    dev = gpu_device
    nodes, past = 20, 118
    parents = random_tree(nodes, seed=5)
    path = [nodes - 1]
    while parents[path[0]] >= 0:
        path.insert(0, parents[path[0]])
    n = len(path)
    b = Batch(dev, heads, [past], [nodes], seed=30, extra_pages=1)
    desc = device_desc([0] * nodes, [past] * nodes, parents, past, dev, accepted=path)
    anc = desc.data_ptr() + N.StepDesc.ancestors.offset
    b.append()
    want, tol = b.reference(parents=parents)
    check(b.attend(ancestors=anc, workspace=False), want, tol, BF16)
    c = b.cache
    k0, v0 = c.logical_keys(0, past + nodes), c.logical_values(0, past + nodes)
    hid = torch.randn(nodes, 64, generator=gen(dev, 9), device=dev).bfloat16()
    sel = torch.full((nodes, 64), 7.0, dtype=torch.bfloat16, device=dev)
    N.check(N.lib().dtree_kv_q8_compact(
        desc.data_ptr(), c.k_pages.data_ptr(), c.v_pages.data_ptr(), c.k_scales.data_ptr(), c.v_scales.data_ptr(), 1,
        c.n_pages, c.kv_heads, c.head_dim, c.page_table.data_ptr(), c.page_table.shape[1], hid.data_ptr(), 64,
        sel.data_ptr(), stream()), "compact")
    keep = list(range(past)) + [past + i for i in path]
    assert torch.equal(c.logical_keys(0, past + n), k0[keep]) and torch.equal(c.logical_values(0, past + n), v0[keep])
    assert torch.equal(sel[:n], hid[path]) and bool((sel[n:] == 7).all())
    b.past, b.rows = [past + n], [1]
    b.dpast.copy_(i32(b.past, dev))
    b.drows.copy_(i32(b.rows, dev))
    b.max_past = past + n
    b.append()
    want, tol = b.reference()
    want[1:] = 7.0
    check(b.attend(), want, tol, BF16)


def test_prompt_in_chunks_equals_the_prompt_at_once(gpu_device):
    """Rows of 0, 1 and many per call, with a window: the same cache bytes, and outputs within both tolerances."""
    dev = gpu_device
    whole = Batch(dev, "128", [0], [260], seed=31)
    whole.append()
    full = whole.attend(sink=5, window=90)
    want, tol = whole.reference(sink=5, window=90)
    check(full, want, tol, BF16)
    part = Batch(dev, "128", [0], [260], seed=31)
    done = 0
    for n in (1, 63, 1, 130, 0, 65):
        part.dpast.copy_(i32([done], dev))
        part.drows.copy_(i32([n], dev))
        rec = part.cache.record(0, part.dpast, part.drows, 260, 130, 260, i32([done], dev))
        part.cache.page_table = torch.cat([part.cache.page_table[:, :5], torch.full((1, 2), -1, dtype=torch.int32,
                                                                                      device=dev)], 1).contiguous()
        rec.page_tables = part.cache.page_table.data_ptr(); rec.ld_page_table = 7
        part.append(rec)
        out = part.attend(rec=rec, sink=5, window=90)
        check(out[done:done + n], want[done:done + n], tol[done:done + n], BF16)
        assert bool((out[done + n:] == 7).all()) and bool((out[:done] == 7).all())
        done += n
    assert torch.equal(part.cache.logical_keys(0, 260), whole.cache.logical_keys(0, 260))
    assert torch.equal(part.cache.logical_values(0, 260), whole.cache.logical_values(0, 260))
