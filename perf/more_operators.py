"""Several hypotheses decoded side by side: cases, plain form and the
framework's calls.

select   beam search's selection: of every request the best (beam, token)
         continuations by summed log-probability, over beams and vocabulary.
fork     the hypotheses' paged caches after a selection: page tables of the
         chosen parents, pages shared, copied before a write, taken and freed,
         and the copied pages' contents in all layers.
step     one token of every hypothesis through a GatedDeltaNet layer's core,
         each from the convolution window and recurrent state of the hypothesis
         that it continues.

select: x = logits of row (group, beam), NaN as -inf, +inf as fp32's largest;
lse = log sum exp x. A live beam's continuation by token t has the sum
s = score + (x_t - lse) and length + 1; a finished beam has the one continuation
`pad` with its own score and length. The best are those of the largest
s / length^penalty, ties to the lower beam, then the lower token; what has no
finite sum is none (-1, score -inf).

fork: sequence i continues parents[i] (-1: an empty one) at its length L. Its
table holds the parent's pages of positions 0 .. L - 1, then pages for `rows`
more positions; refs counts a page's holders, 0 is free. A sequence whose next row
falls into a page that others hold too takes a copy, in ascending order, so the
last holder keeps it; pages are taken in ascending order, by ascending sequence,
a copy before the others. Copies carry the half pages (32 positions) in use.

step: columns of proj [q k v inputs C | z | b | a]; causal convolution of
window + 1 taps, SiLU, q = rms(q) / Dk, k = rms(k) / sqrt(Dk), g = exp(-exp(A)
softplus(a + dt)), beta = sigmoid(b); S = g S; S += beta (v - S k) k^T; y = S q;
out = rms(y) w silu(z).

Head layouts are those of the package's own configurations.
"""
import ctypes as C
import math
import random
import sys
from pathlib import Path

import torch

own = False

PAGE = 64
EPS = 1e-6
F64 = torch.float64
DEV = "cuda"
BIG = torch.finfo(torch.float32).max

# caches whose pages are forked: (layers, kv heads, head dim, bits)
POOLS = {
    "q8_36x8x128": (36, 8, 128, 8),    # the 36-layer model's 8-bit cache
    "bf16_36x8x128": (36, 8, 128, 16),  # and its bf16 cache
    "q8_8x4x256": (8, 4, 256, 8),      # the hybrid's attention layers
    "q8_1x2x64": (1, 2, 64, 8),        # one small layer: the tables are the work
}


# ---- the cases -------------------------------------------------------------------
def listed():
    return [
        # One request's next step: the smallest, all latency.
        dict(name="select_1x4", kind="select", groups=1, beams=4, select=4, vocab=151936, type="f32", penalty=0.0,
             mix=0),
        # The step behind the prompts: one row each, as many beams as are wanted.
        dict(name="select_16x1_first", kind="select", groups=16, beams=1, select=8, vocab=151936, type="f32",
             penalty=0.0, mix=1),
        # A serving batch's step, with finished beams and a length penalty.
        dict(name="select_16x8", kind="select", groups=16, beams=8, select=8, vocab=151936, type="f32", penalty=0.7,
             mix=2),
        # Wide beams of many requests, twice the beams kept: the largest.
        dict(name="select_64x16_bf16", kind="select", groups=64, beams=16, select=32, vocab=151936, type="bf16",
             penalty=1.0, mix=3),
        # One request's eight beams over a 1000-token prompt.
        dict(name="fork_1x8_p1000", kind="fork", pool="q8_36x8x128", groups=1, beams=8, prompt=1000, made=20, rows=1,
             mix=4),
        # A prompt becomes four candidates that drafted trees will be verified on.
        dict(name="fork_1x4_bf16_tree", kind="fork", pool="bf16_36x8x128", groups=1, beams=4, prompt=2000, made=0,
             rows=25, mix=5),
        # A serving batch's beams over prompts of 4000 tokens, the hybrid's attention layers.
        dict(name="fork_16x8_p4000", kind="fork", pool="q8_8x4x256", groups=16, beams=8, prompt=4000, made=100, rows=1,
             mix=6),
        # Long contexts of many hypotheses: the tables and counts.
        dict(name="fork_64x8_p32768", kind="fork", pool="q8_1x2x64", groups=64, beams=8, prompt=32768, made=40, rows=1,
             mix=7),
        # One sequence's token.
        dict(name="step_1", kind="step", seqs=1, k_heads=16, v_heads=32, keep=3, mix=8),
        # One request's eight beams.
        dict(name="step_8", kind="step", seqs=8, k_heads=16, v_heads=32, keep=3, mix=9),
        # A batch of beams of an odd number.
        dict(name="step_37", kind="step", seqs=37, k_heads=16, v_heads=32, keep=3, mix=10),
        # As many as a step's rows hold.
        dict(name="step_128", kind="step", seqs=128, k_heads=16, v_heads=32, keep=3, mix=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["select", "select", "fork", "fork", "step"])
    mix = rng.randrange(1, 1 << 20)
    if kind == "select":
        vocab = rng.choice([151936, _log(rng, 100, 160000), _log(rng, 1000, 160000)])
        typ = rng.choice(["f32", "f32", "bf16"])
        rows = _log(rng, 1, min(1024, 64 * 16 * 151936 // (vocab * (2 if typ == "f32" else 1))))
        beams = min(rows, rng.choice([1, 2, 4, 5, 8, 16, rng.randint(1, 64)]))
        return dict(kind=kind, groups=max(1, rows // beams), beams=beams, select=rng.choice([beams, beams, min(64, 2 * beams), rng.randint(1, 64)]),
                    vocab=vocab, type=typ, penalty=rng.choice([0.0, 0.0, 1.0, round(rng.uniform(0.2, 1.5), 2)]), mix=mix)
    if kind == "fork":
        pool = rng.choice(list(POOLS))
        layers, heads, dim, bits = POOLS[pool]
        beams = rng.choice([2, 4, 8, rng.randint(1, 16)])
        groups = _log(rng, 1, {36: 4, 8: 16, 1: 48}[layers])
        prompt = _log(rng, 1, {36: 4000, 8: 4000, 1: 32768}[layers] // max(1, groups // 4))
        return dict(kind=kind, pool=pool, groups=groups, beams=beams, prompt=prompt,
                    made=rng.choice([0, rng.randint(0, 200)]), rows=rng.choice([1, 1, 1, rng.randint(0, 128)]), mix=mix)
    k_heads, per = rng.choice([(16, 2), (16, 2), (2, 2), (4, 1), (3, 3)])
    return dict(kind=kind, seqs=_log(rng, 1, min(128, 4096 // (k_heads * per))), k_heads=k_heads,
                v_heads=k_heads * per, keep=rng.choice([3, 3, 3, rng.randint(1, 7)]), mix=mix)


def _parents(case):
    """The slot that every sequence continues: its group's better beams more often, -1 now and then. Before the first
    fork a group's first slot alone holds its prompt."""
    rng = random.Random(case["mix"])
    out = []
    if case["kind"] == "step":
        n = case["seqs"]
        return [-1 if n > 4 and rng.random() < 0.03 else min(n - 1, i // 8 * 8 + int(8 * rng.random() ** 2))
                for i in range(n)]
    for g in range(case["groups"]):
        for b in range(case["beams"]):
            first = g * case["beams"]
            at = first + (int(case["beams"] * rng.random() ** 2) if case["made"] else 0)
            out.append(-1 if case["made"] and rng.random() < 0.05 else at)
    return out


def _lengths(case):
    """The slots' lengths: a prompt per group, of the case's length or shorter, and the tokens made since."""
    rng = random.Random(case["mix"] + 1)
    out = []
    for g in range(case["groups"]):
        prompt = case["prompt"] if g == 0 else rng.randint((case["prompt"] + 1) // 2, case["prompt"])
        for b in range(case["beams"]):
            out.append(prompt + case["made"] if case["made"] or b == 0 else 0)
    return out


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _finished(case):
    """Which beams have ended: a fifth, where there is more than one."""
    rng = random.Random(case["mix"] + 2)
    return [case["beams"] > 1 and rng.random() < 0.2 for _ in range(case["groups"] * case["beams"])]


def work(case):
    if case["kind"] == "select":  # the logits of the beams that go on
        n = _finished(case).count(False) * case["vocab"]
        return {"bytes": n * (2 if case["type"] == "bf16" else 4) + 24 * case["groups"] * (case["beams"] + case["select"]),
                "flops": 4 * n}
    if case["kind"] == "step":
        src = _parents(case)
        dims = 2 * case["k_heads"] * 128 + case["v_heads"] * 128
        window, state = case["keep"] * dims, case["v_heads"] * 128 * 128
        proj = dims + case["v_heads"] * 130
        read = len({s for s in src if s >= 0})
        return {"bytes": 4 * ((read + len(src)) * (window + state) + len(src) * proj + (case["keep"] + 1) * dims)
                + 2 * len(src) * case["v_heads"] * 128, "flops": 7 * len(src) * state}
    layers, heads, dim, bits = POOLS[case["pool"]]
    parents, lengths = _parents(case), _lengths(case)
    kids = {p: parents.count(p) for p in set(parents) if p >= 0}
    copied = sum((n - 1) * (1 if lengths[p] % PAGE > 32 else 0.5) for p, n in kids.items()
                 if lengths[p] % PAGE and case["rows"])
    entries = sum(_pages(lengths[p]) for p in kids) + sum(_pages(lengths[p] + case["rows"]) for p in parents if p >= 0)
    page = 2 * layers * heads * PAGE * (dim * bits // 8 + (4 if bits == 8 else 0))
    counts = sum(_pages(n) for p, n in enumerate(lengths) if kids.get(p, 0) != 1)
    return {"bytes": 4 * entries + 8 * counts + int(2 * copied * page), "flops": entries}


# ---- seeded inputs ---------------------------------------------------------------
def _generator(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + case["mix"] * 7919 + 29)
    return g


def _select_inputs(case, seed):
    g = _generator(case, seed)
    G, K, V = case["groups"], case["beams"], case["vocab"]
    dt = torch.bfloat16 if case["type"] == "bf16" else torch.float32
    x = torch.empty(G * K, V, device=DEV).normal_(0.0, 2.0, generator=g)
    # a peaked distribution: a few tokens well above the rest
    peaks = torch.randint(0, V, (G * K, 16), generator=g, device=DEV)
    x.scatter_add_(1, peaks, torch.empty(G * K, 16, device=DEV).normal_(7.0, 2.0, generator=g))
    # tokens that the caller forbids
    x[:, torch.randint(0, V, (max(1, V // 50),), generator=g, device=DEV)] = float("-inf")
    steps = torch.randint(1, 60, (G, 1), generator=g, device=DEV, dtype=torch.int32)
    lengths = (steps - torch.randint(0, 8, (G, K), generator=g, device=DEV, dtype=torch.int32)).clamp(min=1)
    over = torch.tensor(_finished(case), device=DEV).view(G, K)
    lengths = torch.where(over, lengths, steps.expand(G, K)).contiguous()
    scores = -torch.rand(G, K, generator=g, device=DEV) * 6 - lengths * 0.8
    return dict(case=case, x=x.to(dt), scores=scores.contiguous(), lengths=lengths, over=over.to(torch.int32),
                eos=min(2, V - 1), pad=0)


def _fork_inputs(case, seed):
    g = _generator(case, seed)
    layers, heads, dim, bits = POOLS[case["pool"]]
    parents, lengths = _parents(case), _lengths(case)
    n = len(parents)
    ld = _pages(max(lengths) + max(case["rows"], 1)) + 1
    # logical page i of a slot: the group's shared ones hold whole prompt pages, the others are its own
    shared, held, at = [], [], 0
    for p in range(n):
        first = p // case["beams"] * case["beams"]
        common = (lengths[p] - case["made"]) // PAGE if case["made"] else 0
        if p == first or not case["made"]:
            shared = list(range(at, at + common))
            at += common
        own_pages = _pages(lengths[p]) - common
        row = shared + list(range(at, at + own_pages))
        at += own_pages
        held.append(row + [-1] * (ld - len(row)))
    total = at + n * (2 + _pages(case["rows"])) + 5
    place = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    held = torch.tensor(held, device=DEV)
    tables = torch.where(held >= 0, place[held.clamp(min=0)], -1).to(torch.int32)
    refs = torch.zeros(total, dtype=torch.int32, device=DEV)
    refs.index_add_(0, tables.clamp(min=0).reshape(-1).long(), (tables >= 0).reshape(-1).to(torch.int32))
    kv = {}
    for name in ("k", "v"):
        shape = (layers, total, heads, PAGE * dim)
        if bits == 8:
            kv[name] = torch.empty(shape, dtype=torch.int8, device=DEV).random_(-127, 128, generator=g)
            kv[name + "_scales"] = torch.rand(layers, total, heads, PAGE, generator=g, device=DEV)
        else:
            kv[name] = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, 1.0, generator=g)
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(case=case, kv=kv, refs=refs, tables=[tables.contiguous(), torch.full_like(tables, -1)],
                lengths=[torch.tensor(lengths, **i32), torch.zeros(n, **i32)], turn=0,
                parents=torch.tensor(parents, **i32), copies=torch.full((n, 3), -1, **i32),
                status=torch.zeros(2, **i32))


def _step_inputs(case, seed):
    g = _generator(case, seed)
    n, hk, hv, keep = case["seqs"], case["k_heads"], case["v_heads"], case["keep"]
    dims = 2 * hk * 128 + hv * 128
    width = (dims + hv * 130 + 63) // 64 * 64
    rand = lambda *s: torch.empty(*s, device=DEV).normal_(0.0, 1.0, generator=g)  # noqa: E731
    return dict(case=case, dims=dims, proj=rand(n, width), window=rand(n, keep, dims),
                state=rand(n, hv, 128, 128) * 0.3, conv=rand(keep + 1, dims) * 0.5,
                a_log=torch.rand(hv, generator=g, device=DEV) * 2.5, dt=rand(hv) - 2.0,
                norm=(rand(128) * 0.1 + 1.0).bfloat16(), source=torch.tensor(_parents(case), dtype=torch.int32, device=DEV),
                out=torch.empty(n, hv * 128, dtype=torch.bfloat16, device=DEV),
                window_out=torch.empty(n, keep, dims, device=DEV), state_out=torch.empty(n, hv, 128, 128, device=DEV))


def _inputs(case, seed):
    return {"select": _select_inputs, "fork": _fork_inputs, "step": _step_inputs}[case["kind"]](case, seed)


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["kind"] == "select":
        G, M = case["groups"], case["select"]
        i32 = dict(dtype=torch.int32, device=DEV)
        st["best"] = dict(scores=torch.empty(G, M, device=DEV), tokens=torch.empty(G, M, **i32),
                          parents=torch.empty(G, M, **i32), lengths=torch.empty(G, M, **i32),
                          finished=torch.empty(G, M, **i32))
    if own:
        st["plan"] = _plan(st)
    return st


# ---- the framework's calls --------------------------------------------------------
def _plan(st):
    """The argument records a program keeps between calls, and the workspace."""
    pkg = str(Path(__file__).resolve().parent.parent / "dtree-mlx_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from dtree_hip import _native as N

    lib, case = N.lib(), st["case"]
    plan = dict(lib=lib, check=N.check)
    if case["kind"] == "select":
        a = N.BeamArgs()
        a.logits = st["x"].data_ptr(); a.type = N.T_BF16 if case["type"] == "bf16" else N.T_F32
        a.ld_logits = case["vocab"]; a.vocab = case["vocab"]
        a.groups = case["groups"]; a.beams = case["beams"]; a.num_select = case["select"]
        a.scores = st["scores"].data_ptr(); a.lengths = st["lengths"].data_ptr(); a.finished = st["over"].data_ptr()
        a.eos_token = st["eos"]; a.pad_token = st["pad"]; a.length_penalty = case["penalty"]
        for name, t in st["best"].items():
            setattr(a, name + "_out", t.data_ptr())
        size = lib.dtree_beam_select_workspace_bytes(C.byref(a))
        st["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEV)
        a.workspace = st["workspace"].data_ptr(); a.workspace_bytes = size
        plan["args"] = a
    elif case["kind"] == "fork":
        layers, heads, dim, bits = POOLS[case["pool"]]
        plan["fork"] = []
        for turn in (0, 1):
            a = N.PagesFork()
            a.refs = st["refs"].data_ptr(); a.num_pages = st["refs"].numel()
            a.num_seqs = len(st["parents"]); a.ld_tables = st["tables"][0].shape[1]
            a.tables = st["tables"][turn].data_ptr(); a.tables_out = st["tables"][1 - turn].data_ptr()
            a.lengths = st["lengths"][turn].data_ptr(); a.lengths_out = st["lengths"][1 - turn].data_ptr()
            a.parents = st["parents"].data_ptr(); a.rows = case["rows"]; a.absent = -1
            a.copies = st["copies"].data_ptr(); a.status = st["status"].data_ptr()
            plan["fork"].append(a)
        c = N.PagesCopy()
        c.copies = st["copies"].data_ptr(); c.max_copies = len(st["parents"])
        c.num_pages = st["refs"].numel(); c.num_heads = heads; c.layers = layers
        for i, t in enumerate(st["kv"].values()):
            c.pools[i] = t.data_ptr(); c.block_bytes[i] = t.shape[3] * t.element_size()
        plan["copy"] = c
    else:
        a = N.GdnArgs()
        a.rows_padded = case["seqs"]; a.num_k_heads = case["k_heads"]; a.num_v_heads = case["v_heads"]
        a.head_k_dim = a.head_v_dim = 128; a.conv_keep = case["keep"]
        a.proj = st["proj"].data_ptr(); a.ld_proj = st["proj"].shape[1]
        a.window = st["window"].data_ptr(); a.conv_w = st["conv"].data_ptr()
        a.A_log = st["a_log"].data_ptr(); a.dt_bias = st["dt"].data_ptr(); a.state = st["state"].data_ptr()
        a.norm_w = st["norm"].data_ptr(); a.eps = EPS
        a.out = st["out"].data_ptr(); a.out_layout = N.W_ROWMAJOR; a.ld_out = st["out"].shape[1]
        a.window_out = st["window_out"].data_ptr(); a.state_out = st["state_out"].data_ptr()
        plan["args"] = a
    return plan


def _run_own(st):
    p, kind = st["plan"], st["case"]["kind"]
    lib, stream = p["lib"], torch.cuda.current_stream().cuda_stream
    if kind == "select":
        p["check"](lib.dtree_beam_select(C.byref(p["args"]), stream), "select")
        return st["best"]
    if kind == "fork":
        p["check"](lib.dtree_pages_fork(C.byref(p["fork"][st["turn"]]), stream), "fork")
        p["check"](lib.dtree_pages_copy(C.byref(p["copy"]), stream), "copy")
        st["turn"] = 1 - st["turn"]
        return _fork_outputs(st)
    p["check"](lib.dtree_gdn_layer_batch(C.byref(p["args"]), st["source"].data_ptr(), st["case"]["seqs"], stream), "step")
    return _step_outputs(st)


def _fork_outputs(st):
    return dict(st["kv"], tables=st["tables"][st["turn"]], lengths=st["lengths"][st["turn"]], refs=st["refs"],
                copies=st["copies"], status=st["status"])


def _step_outputs(st):
    return dict(out=st["out"], window=st["window_out"], state=st["state_out"])


# ---- the plain form ---------------------------------------------------------------
def _run_select(st):
    case = st["case"]
    G, K, V, M = case["groups"], case["beams"], case["vocab"], case["select"]
    x = torch.nan_to_num(st["x"].float(), nan=float("-inf"), posinf=BIG, neginf=float("-inf"))
    top = x.amax(-1, keepdim=True).clamp(min=-BIG)
    lse = (x - top).exp_().sum(-1, dtype=F64).log() + top[:, 0].double()
    # every row's best M, by value and then by the lower token: one whole number each
    bits = (x + 0.0).view(torch.int32).long()  # (-0 as 0)
    word = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    m = min(M, V)
    best = torch.topk(word * (1 << 20) - torch.arange(V, device=DEV), m, dim=-1).values
    token = -best % (1 << 20)
    val = torch.gather(x, 1, token).double()
    score = st["scores"].double().view(-1, 1)
    total = torch.where(val > -math.inf, score + (val - lse[:, None]), -math.inf)
    over = st["over"].bool().view(-1, 1)
    first = torch.arange(m, device=DEV)[None] == 0
    total = torch.where(over, torch.where(first, score, -math.inf), total)
    token = torch.where(over, st["pad"], token)
    length = (st["lengths"].view(-1, 1) + (~over)).expand(-1, m)
    # in the order of beam and token, then by rank: ties stay in that order
    token, at = torch.sort(token.reshape(G, K, m), dim=-1, stable=True)
    total = torch.gather(total.view(G, K, m), 2, at).view(G, K * m)
    token, length = token.view(G, K * m), torch.gather(length.reshape(G, K, m), 2, at).view(G, K * m)
    rank = total * length.clamp(min=1).double() ** -case["penalty"] if case["penalty"] else total
    at = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :M]
    got = [torch.gather(t, 1, at) for t in (total, token, length)]
    beam = at // m
    done = torch.gather(st["over"].view(G, K), 1, beam).bool() | (got[1] == st["eos"])
    none = ~(got[0] > -math.inf)
    fill = dict(scores=-math.inf, tokens=-1, parents=-1, lengths=0, finished=0)
    row = beam + torch.arange(G, device=DEV)[:, None] * K
    for name, t in zip(fill, (got[0], got[1], row, got[2], done)):
        out = st["best"][name]
        out.fill_(fill[name])
        out[:, :at.shape[1]] = torch.where(none, fill[name], t.to(F64)).to(out.dtype)
    return st["best"]


def _run_fork(st):
    case, rows = st["case"], st["case"]["rows"]
    old, lengths = st["tables"][st["turn"]], st["lengths"][st["turn"]]
    parents, refs = st["parents"].long(), st["refs"]
    n, ld = old.shape
    total = len(refs)
    live = parents >= 0
    L = torch.where(live, lengths[parents.clamp(min=0)].long(), 0).clamp(0, ld * PAGE)
    e = torch.arange(ld, device=DEV)[None]
    covered = (L + PAGE - 1) // PAGE
    table = torch.where(live[:, None] & (e < covered[:, None]), old[parents.clamp(min=0)].long(), -1)

    def count(pages, by):  # a page of -1 counts for nobody
        flat = pages.reshape(-1)
        refs.index_add_(0, flat.clamp(min=0), torch.where(flat >= 0, by, 0).to(torch.int32))

    count(old.long(), -1)
    count(table, 1)
    # the page that the next row falls into, where others hold it too
    at = (L // PAGE).clamp(max=ld - 1)
    page = torch.gather(table, 1, at[:, None])[:, 0]
    writes = (L % PAGE > 0) & (rows > 0) & (page >= 0)
    same = (page[:, None] == page[None]) & writes[:, None] & writes[None]
    rank = same.tril(-1).sum(1)
    copies = writes & (refs[page.clamp(min=0)] - rank > 1)
    count(torch.where(copies, page, -1), -1)
    # pages taken, ascending
    wanted = (L + rows + PAGE - 1) // PAGE if rows else covered
    last = wanted.clamp(max=ld)
    need = copies.long() + (last - covered).clamp(min=0)
    start = torch.cumsum(need, 0) - need
    free = torch.sort((refs != 0).to(torch.uint8), stable=True).indices
    room = (refs == 0).sum()
    is_copy = copies[:, None] & (e == at[:, None])
    taken = is_copy | ((e >= covered[:, None]) & (e < last[:, None]))
    order = start[:, None] + torch.where(is_copy, 0, copies.long()[:, None] + e - covered[:, None])
    got = torch.where(order < room, free[order.clamp(0, total - 1)], -1)
    table = torch.where(taken, got, table)
    count(torch.where(taken, got, -1), 1)
    st["tables"][1 - st["turn"]].copy_(table)
    st["lengths"][1 - st["turn"]].copy_(L)
    st["status"][0] += ((need.sum() - room).clamp(min=0) + (wanted - last).sum()).to(torch.int32)
    # the copies, by sequence: source, destination, positions in use
    to = torch.gather(table, 1, at[:, None])[:, 0]
    made = copies & (to >= 0)
    spot = torch.where(made, torch.cumsum(made.long(), 0) - 1, n)
    listed = torch.full((n + 1, 3), -1, dtype=torch.int32, device=DEV)
    listed[spot] = torch.stack([page, to, L % PAGE], 1).to(torch.int32)
    st["copies"].copy_(listed[:n])
    st["status"][1] = made.sum().to(torch.int32)
    # their contents; what is no copy does the first one again (or nothing, page 0 to itself)
    c = st["copies"].long()
    c = torch.where(c[:, :1] >= 0, c, torch.where(c[:1, :1] >= 0, c[:1], 0))
    whole = (c[:, 2] > 32)[None, :, None, None]
    for pool in st["kv"].values():
        a, b = pool[:, c[:, 0]], pool[:, c[:, 1]]
        half = torch.arange(pool.shape[3], device=DEV) < pool.shape[3] // 2
        pool[:, c[:, 1]] = torch.where(whole | half, a, b)
    st["turn"] = 1 - st["turn"]
    return _fork_outputs(st)


def _run_step(st):
    case = st["case"]
    n, hk, hv, keep, dims = case["seqs"], case["k_heads"], case["v_heads"], case["keep"], st["dims"]
    src = st["source"].long()
    live = (src >= 0).float()
    rows = torch.cat([st["window"][src.clamp(min=0)] * live[:, None, None], st["proj"][:, None, :dims]], 1)
    st["window_out"].copy_(rows[:, 1:])
    y = (rows * st["conv"]).sum(1)
    y = y * torch.sigmoid(y)
    q, k = (t.view(n, hk, 128) for t in (y[:, :hk * 128], y[:, hk * 128:2 * hk * 128]))
    v = y[:, 2 * hk * 128:].view(n, hv, 128)
    rms = lambda t, eps: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps)  # noqa: E731
    q = (rms(q, 1e-6) / 128).repeat_interleave(hv // hk, 1)
    k = (rms(k, 1e-6) / math.sqrt(128)).repeat_interleave(hv // hk, 1)
    rest = st["proj"][:, dims:]
    z, b, a = rest[:, :hv * 128].view(n, hv, 128), rest[:, hv * 128:hv * 129], rest[:, hv * 129:hv * 130]
    t = a + st["dt"]
    soft = t.clamp(min=0) + torch.log1p(torch.exp(-t.abs()))
    g = torch.exp(-torch.exp(st["a_log"]) * soft)
    s = st["state"][src.clamp(min=0)] * (live[:, None] * g)[:, :, None, None]
    delta = (v - (s * k[:, :, None]).sum(-1)) * torch.sigmoid(b)[..., None]
    torch.add(s, delta[..., None] * k[:, :, None], out=st["state_out"])
    y = (st["state_out"] * q[:, :, None]).sum(-1)
    y = rms(y, EPS) * st["norm"].float() * z * torch.sigmoid(z)
    st["out"].copy_(y.view(n, hv * 128))
    return _step_outputs(st)


def run(st):
    if own:
        return _run_own(st)
    return {"select": _run_select, "fork": _run_fork, "step": _run_step}[st["case"]["kind"]](st)


# ---- the definition in 64 bits ------------------------------------------------------
def _exact_select(case, seed):
    st = _inputs(case, seed)
    K, M, V = case["beams"], case["select"], case["vocab"]
    if case["groups"] * K * V > 40_000_000:
        return None
    scores = torch.full((case["groups"], M), -math.inf, dtype=F64, device=DEV)
    for g in range(case["groups"]):
        x = st["x"][g * K:(g + 1) * K].double()
        x[torch.isnan(x)] = -math.inf
        x = x.clamp(max=BIG)
        sums = st["scores"][g].double()[:, None] + torch.log_softmax(x, -1)
        sums[torch.isnan(sums)] = -math.inf
        size = st["lengths"][g].double()[:, None] + 1
        for b in range(K):
            if st["over"][g, b]:
                sums[b] = -math.inf
                sums[b, 0] = st["scores"][g, b].double()
                size[b] -= 1
        ranked = (sums / size.clamp(min=1) ** case["penalty"]).view(-1)
        best = ranked.sort(descending=True, stable=True).indices[:M]
        scores[g, :len(best)] = sums.view(-1)[best]
    return dict(scores=scores, tokens=None, parents=None, lengths=None, finished=None)


def _exact_step(case, seed):
    st = _inputs(case, seed)
    n, hk, hv, dims = case["seqs"], case["k_heads"], case["v_heads"], st["dims"]
    out = torch.empty(n, hv * 128, dtype=F64, device=DEV)
    window = torch.empty(st["window"].shape, dtype=F64, device=DEV)
    state = torch.empty(st["state"].shape, dtype=F64, device=DEV)
    taps, w = st["conv"].double(), st["norm"].double()

    def unit(t, eps):
        return t / (t.pow(2).mean(-1, keepdim=True) + eps).sqrt()

    for i, s in enumerate(_parents(case)):
        row = st["proj"][i].double()
        past = st["window"][s].double() if s >= 0 else torch.zeros(case["keep"], dims, dtype=F64, device=DEV)
        seen = torch.vstack([past, row[None, :dims]])
        window[i] = seen[1:]
        y = torch.nn.functional.silu((seen * taps).sum(0))
        q = unit(y[:hk * 128].view(hk, 128), 1e-6) / 128
        k = unit(y[hk * 128:2 * hk * 128].view(hk, 128), 1e-6) / 128 ** 0.5
        v = y[2 * hk * 128:].view(hv, 128)
        z, b, a = row[dims:dims + hv * 128].view(hv, 128), *row[dims + hv * 128:dims + hv * 130].view(2, hv)
        g = (-st["a_log"].double().exp() * torch.nn.functional.softplus(a + st["dt"].double())).exp()
        S = st["state"][s].double() if s >= 0 else torch.zeros(hv, 128, 128, dtype=F64, device=DEV)
        at = torch.arange(hv, device=DEV) // (hv // hk)
        kk, qq = k[at].unsqueeze(-1), q[at].unsqueeze(-1)
        S = S * g[:, None, None]
        S = S + (b.sigmoid()[:, None, None] * (v.unsqueeze(-1) - S @ kk)) @ kk.transpose(1, 2).contiguous()
        state[i] = S
        o = unit((S @ qq).squeeze(-1), EPS) * w * torch.nn.functional.silu(z)
        out[i] = o.view(-1)
    return dict(out=out, window=window, state=state)


def exact(case, seed):
    if case["kind"] == "fork":  # whole numbers and copies
        return None
    return _exact_select(case, seed) if case["kind"] == "select" else _exact_step(case, seed)
