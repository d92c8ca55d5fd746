"""The 8-bit paged KV cache and the attention over it: cases, plain form and
the framework's calls.

write    k_norm + RoPE of new K rows, quantisation of K and V rows as they are
         written into the pages, and those rows read back as the values they
         stand for.
read     cached positions of sequences as rows of bf16.
attend   attention of new rows (single tokens, chunks, prompts, draft trees)
         of a batch of sequences over their pages, with a sliding window and
         sinks where the case has them.

A cached row (one position of one kv head) is D integers in [-127, 127] and one
fp32 scale: scale = fp32(max |x| / 127), q = the integer nearest to x / scale
(ties to even), value = q * scale. Pages hold 64 positions.

Head layouts are those of the package's own configurations (32 / 8 heads of
128, rotary over all dims; 16 / 4 heads of 256 with 64 rotary dims and an output
gate) and a small one of 64 dims.
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

# name: (query heads, kv heads, head dim, rotary dims, rope base, gated)
LAYOUTS = {
    "h32x128": (32, 8, 128, 128, 1e6, False),
    "h8x128": (8, 2, 128, 128, 1e6, False),
    "g16x256": (16, 4, 256, 64, 1e5, True),
    "h12x64": (12, 4, 64, 64, 1e4, False),
}


# ---- the cases -------------------------------------------------------------------
def listed():
    return [
        # One decoded token of one sequence enters a layer's cache: the smallest call.
        dict(name="write_1", kind="write", layout="h32x128", seqs=1, rows=1, past=1000, mix=0, type="f32"),
        # A prompt segment that starts inside a page.
        dict(name="write_4000", kind="write", layout="h32x128", seqs=1, rows=4000, past=37, mix=0, type="f32"),
        # A short sequence's cache handed to a path that takes bf16 rows.
        dict(name="read_1000", kind="read", layout="h32x128", seqs=1, rows=1000, past=0, mix=0),
        # The caches of several long sequences of the hybrid's gated heads.
        dict(name="read_4x8192_d256", kind="read", layout="g16x256", seqs=4, rows=8192, past=0, mix=1),
        # One token of one sequence over a short context.
        dict(name="decode_1_p1000", kind="attend", layout="h32x128", seqs=1, rows=1, past=1000, mix=0, tree=False,
             sink=0, window=0, type="f32"),
        # One token over a long document.
        dict(name="decode_1_p65535", kind="attend", layout="h32x128", seqs=1, rows=1, past=65535, mix=0, tree=False,
             sink=0, window=0, type="f32"),
        # A decode step of a batch of sequences of very different lengths.
        dict(name="decode_32_p8192", kind="attend", layout="h32x128", seqs=32, rows=1, past=8192, mix=2, tree=False,
             sink=0, window=0, type="f32"),
        # The verify step's drafted tree (25 nodes) over a 2048-key prefix.
        dict(name="tree_25_p2048", kind="attend", layout="h32x128", seqs=1, rows=25, past=2048, mix=3, tree=True,
             sink=0, window=0, type="f32"),
        # A further turn of a conversation: 1000 tokens over a long cache, gated heads.
        dict(name="chunk_1000_p8192_d256", kind="attend", layout="g16x256", seqs=1, rows=1000, past=8192, mix=0,
             tree=False, sink=0, window=0, type="f32"),
        # A whole prompt segment without a prefix: the largest.
        dict(name="prompt_4096", kind="attend", layout="h32x128", seqs=1, rows=4096, past=0, mix=0, tree=False,
             sink=0, window=0, type="f32"),
        # Streams that have run far past their window decode one token each.
        dict(name="window_decode_16", kind="attend", layout="h32x128", seqs=16, rows=1, past=16384, mix=4, tree=False,
             sink=64, window=1024, type="f32"),
        # Several streams take in chunks of their own sizes under a window.
        dict(name="window_chunks_4x700", kind="attend", layout="h32x128", seqs=4, rows=700, past=8192, mix=5,
             tree=False, sink=64, window=1024, type="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk", "tree", "window", "window"])
    layout = rng.choice(list(LAYOUTS))
    mix = rng.randrange(1, 1 << 20)
    typ = rng.choice(["f32", "f32", "bf16"])
    if kind == "write":
        seqs = _log(rng, 1, 64)
        return dict(kind=kind, layout=layout, seqs=seqs, rows=_log(rng, 1, max(1, 4096 // seqs)),
                    past=_log(rng, 1, 4096) - 1, mix=mix, type=typ)
    if kind == "read":
        seqs = _log(rng, 1, 16)
        return dict(kind=kind, layout=layout, seqs=seqs, rows=_log(rng, 1, 32768 // seqs),
                    past=rng.choice([0, 0, rng.randint(1, 100)]), mix=mix)
    c = dict(kind="attend", layout=layout, seqs=1, rows=1, past=0, mix=mix, tree=False, sink=0, window=0, type=typ)
    if kind == "decode":
        c["seqs"] = _log(rng, 1, 48)
        c["past"] = _log(rng, 1, 196608 // c["seqs"]) - 1
        c["rows"] = rng.choice([1, 1, 1, rng.randint(2, 8)])
    elif kind == "chunk":
        c["seqs"] = rng.choice([1, 1, rng.randint(2, 8)])
        c["rows"] = _log(rng, 2, 3000 // c["seqs"])
        c["past"] = rng.choice([0, _log(rng, 1, 8192 // c["seqs"])])
    elif kind == "tree":
        c.update(tree=True, rows=rng.randint(2, 128), past=_log(rng, 1, 16384) - 1)
    else:
        c["seqs"] = _log(rng, 1, 16)
        c["rows"] = rng.choice([1, 1, _log(rng, 2, 2000 // c["seqs"] + 2)])
        c["past"] = _log(rng, 1, 65536 // c["seqs"]) - 1
        c["sink"] = rng.choice([0, 1, 4, 64, rng.randint(1, 200)])
        c["window"] = _log(rng, 1, 4096)
    return c


def _lengths(case):
    """(past, count) of every sequence: the first has the case's own, the others
    of a batch come from `mix`. Chunk batches hold single tokens too."""
    rng = random.Random(case["mix"])
    past, rows = [case["past"]], [case["rows"]]
    for _ in range(case["seqs"] - 1):
        past.append(_log(rng, 1, case["past"] + 1) - 1)
        rows.append(rng.choice([1, rng.randint(1, case["rows"]), rng.randint(1, case["rows"])]))
    if case["kind"] == "read":
        past = [case["past"]] * case["seqs"]
    return past, rows


def _tree(case):
    """Parents of a drafted tree, nodes in heap order."""
    rng = random.Random(case["mix"])
    return [-1] + [rng.randrange(max(0, i - 8), i) for i in range(1, case["rows"])]


def _visible(case):
    """Sum over rows of the keys that a row sees, and the cached rows that a
    sequence's rows see between them."""
    past, rows = _lengths(case)
    pairs = keys = 0
    if case.get("tree"):
        depth = []
        for p in _tree(case):
            depth.append(0 if p < 0 else depth[p] + 1)
        return sum(past[0] + d + 1 for d in depth), past[0] + rows[0]
    for p, n in zip(past, rows):
        w, s = case["window"], case["sink"]
        for q in range(p, p + n):
            pairs += q + 1 if not w else min(q + 1, w + min(s, max(0, q + 1 - w)))
        keys += p + n if not w else min(p + n, w + n - 1 + min(s, max(0, p + 1 - w)))
    return pairs, keys


def work(case):
    hq, hkv, d, _, _, gated = LAYOUTS[case["layout"]]
    _, rows = _lengths(case)
    total = sum(rows)
    row = hkv * (d + 4)  # a cached row of all kv heads, K or V
    size = 2 if case.get("type") == "bf16" else 4
    if case["kind"] == "write":  # rows in, cache rows out, values out
        return {"bytes": 2 * total * (hkv * d * size + row + hkv * d * 4), "flops": 2 * total * hkv * d * 8}
    if case["kind"] == "read":
        return {"bytes": 2 * total * (row + hkv * d * 2), "flops": 2 * total * hkv * d}
    pairs, keys = _visible(case)
    return {"bytes": 2 * keys * row + total * hq * d * ((2 if gated else 1) * size + 2), "flops": 4 * pairs * hq * d}


# ---- seeded inputs ---------------------------------------------------------------
def _inputs(case, seed):
    """Logical inputs: per page and kv head the cached integers and scales, the
    page tables, the new rows' projections and the tables of their positions."""
    hq, hkv, d, rd, base, gated = LAYOUTS[case["layout"]]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + case["mix"] * 7919 + 17)
    past, rows = _lengths(case)
    per = max((p + n + PAGE - 1) // PAGE for p, n in zip(past, rows))  # pages per sequence
    n_pages = per * case["seqs"] + 1
    tables = torch.randperm(n_pages, generator=g, device=DEV)[:per * case["seqs"]].view(case["seqs"], per)

    def cached(channel):
        x = torch.empty(n_pages, hkv, PAGE, d, device=DEV).normal_(0.0, 1.0, generator=g) * channel
        scale = (x.abs().amax(-1).double() / 127).float()
        return torch.round(x.double().div_(scale.double()[..., None])).to(torch.int8), scale

    # keys have a few large channels, values are even
    kc = torch.empty(d, device=DEV).normal_(0.0, 0.6, generator=g).exp_()
    vc = torch.full((d,), 0.5, device=DEV)
    kq, ks = cached(kc)
    vq, vs = cached(vc)
    total = sum(rows)
    dt = torch.bfloat16 if case.get("type") == "bf16" else torch.float32
    qs = 2 * d if gated else d
    width = hq * qs + 2 * hkv * d  # [q heads | k heads | v heads], the fused projection's rows
    qkv = torch.empty(total, width, device=DEV).normal_(0.0, 1.0, generator=g).to(dt)
    q_norm = torch.empty(d, device=DEV).normal_(1.2, 0.1, generator=g).bfloat16()
    k_norm = torch.empty(d, device=DEV).normal_(1.2, 0.1, generator=g).bfloat16()
    if case.get("tree"):
        depth, words = [], []
        for i, p in enumerate(_tree(case)):
            depth.append(0 if p < 0 else depth[p] + 1)
            words.append((words[p] if p >= 0 else 0) | 1 << i)
        pos = [past[0] + x for x in depth]
        anc = torch.tensor([[((w >> (32 * k)) & 0xffffffff) - ((w >> (32 * k) & 0x80000000) << 1) for k in range(4)]
                            for w in words], dtype=torch.int32, device=DEV)
    else:
        pos = [p + i for p, n in zip(past, rows) for i in range(n)]
        anc = None
    ang = torch.tensor(pos, device=DEV, dtype=F64)[:, None] * base ** (
        -torch.arange(0, rd, 2, device=DEV, dtype=F64) / rd)
    i32 = dict(dtype=torch.int32, device=DEV)
    starts = [sum(rows[:i]) for i in range(len(rows))]
    return dict(case=case, kq=kq, ks=ks, vq=vq, vs=vs, tables=tables.to(torch.int32).contiguous(), qkv=qkv,
                q_norm=q_norm, k_norm=k_norm, anc=anc, cos=ang.cos().float(), sin=ang.sin().float(),
                past=torch.tensor(past, **i32), count=torch.tensor(rows, **i32), start=torch.tensor(starts, **i32),
                host=(past, rows, starts))


# A page of a kv head: 64 positions x D dims in the order in which the
# attention's 32x32x16 products read 16 bytes a lane. K: [slot / 32][dim / 32]
# [dim / 16 % 2][slot % 32][dim % 16]. V: [slot / 32][dim / 32][slot / 4 % 2]
# [dim % 32][slot / 8 % 4][slot % 4].
def _to_pages(kq, vq):
    n, h, _, d = kq.shape
    k = kq.view(n, h, 2, 32, d // 32, 2, 16).permute(0, 1, 2, 4, 5, 3, 6)
    v = vq.view(n, h, 2, 4, 2, 4, d // 32, 32).permute(0, 1, 2, 6, 4, 7, 3, 5)
    return k.reshape(n, h, PAGE * d).contiguous(), v.reshape(n, h, PAGE * d).contiguous()


def _from_pages(kp, vp, d):
    """[..., 64 D] pages to [..., 64, D]."""
    lead = kp.shape[:-1]
    k = kp.view(-1, 2, d // 32, 2, 32, 16).permute(0, 1, 4, 2, 3, 5).reshape(*lead, PAGE, d)
    v = vp.view(-1, 2, d // 32, 2, 32, 4, 4).permute(0, 1, 5, 3, 6, 2, 4).reshape(*lead, PAGE, d)
    return k, v


def prepare(case, seed):
    hq, hkv, d, rd, _, gated = LAYOUTS[case["layout"]]
    st = _inputs(case, seed)
    st["kp"], st["vp"] = _to_pages(st.pop("kq"), st.pop("vq"))
    past, rows, starts = st["host"]
    total, width = sum(rows), st["qkv"].shape[1]
    st["koff"] = width - 2 * hkv * d
    if case["kind"] == "attend":
        st["out"] = torch.empty(total, hq * d, dtype=torch.bfloat16, device=DEV)
    else:
        dt = torch.float32 if case["kind"] == "write" else torch.bfloat16
        st["k_out"] = torch.empty(total, hkv, d, dtype=dt, device=DEV)
        st["v_out"] = torch.empty(total, hkv, d, dtype=dt, device=DEV)
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

    case = st["case"]
    hq, hkv, d, rd, _, gated = LAYOUTS[case["layout"]]
    past, rows, _ = st["host"]
    kv = N.KvQ8()
    kv.k_pages = st["kp"].data_ptr(); kv.v_pages = st["vp"].data_ptr()
    kv.k_scales = st["ks"].data_ptr(); kv.v_scales = st["vs"].data_ptr()
    kv.num_pages = st["kp"].shape[0]; kv.num_kv_heads = hkv; kv.head_dim = d
    kv.num_seqs = case["seqs"]
    kv.page_tables = st["tables"].data_ptr(); kv.ld_page_table = st["tables"].shape[1]
    kv.past_lengths = st["past"].data_ptr(); kv.row_counts = st["count"].data_ptr()
    kv.row_starts = st["start"].data_ptr()
    kv.max_past_length = max(past); kv.max_rows = max(rows); kv.total_rows = sum(rows)
    lib = N.lib()
    plan = dict(lib=lib, check=N.check, kv=kv, f32=N.T_F32, bf16=N.T_BF16)
    if case["kind"] == "attend":
        a = N.AttnQ8Args()
        a.q = st["qkv"].data_ptr(); a.ld_q = st["qkv"].shape[1]; a.q_stride = 2 * d if gated else d
        a.q_type = N.T_BF16 if st["qkv"].dtype == torch.bfloat16 else N.T_F32
        a.q_norm = st["q_norm"].data_ptr(); a.eps = EPS
        a.rope_cos = st["cos"].data_ptr(); a.rope_sin = st["sin"].data_ptr(); a.rope_dims = rd
        a.ancestors = st["anc"].data_ptr() if st["anc"] is not None else None
        a.sink = case["sink"]; a.window = case["window"]
        a.out = st["out"].data_ptr(); a.ld_out = hq * d; a.out_layout = N.W_ROWMAJOR
        a.num_heads = hq; a.scale = d ** -0.5; a.gated = int(gated)
        size = lib.dtree_attention_q8_workspace_bytes(C.byref(kv), C.byref(a))
        st["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
        a.workspace = st["workspace"].data_ptr(); a.workspace_bytes = size
        plan["attn"] = a
    return plan


def _run_own(st):
    case, p = st["case"], st["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["kind"] == "attend":
        p["check"](p["lib"].dtree_attention_q8(C.byref(p["kv"]), C.byref(p["attn"]), stream), "attention")
        return st["out"]
    _, hkv, d, rd, _, _ = LAYOUTS[case["layout"]]
    out = torch.float32 if case["kind"] == "write" else torch.bfloat16
    if case["kind"] == "write":
        x = st["qkv"]
        bf = x.dtype == torch.bfloat16
        k = x.data_ptr() + st["koff"] * x.element_size()
        p["check"](p["lib"].dtree_kv_q8_append(
            C.byref(p["kv"]), k, k + hkv * d * x.element_size(), p["bf16"] if bf else p["f32"], x.shape[1],
            x.shape[1], st["k_norm"].data_ptr(), EPS, st["cos"].data_ptr(), st["sin"].data_ptr(), rd, stream),
            "append")
    p["check"](p["lib"].dtree_kv_q8_read(
        C.byref(p["kv"]), st["k_out"].data_ptr(), st["v_out"].data_ptr(),
        p["f32"] if out == torch.float32 else p["bf16"], hkv * d, hkv * d, stream), "read")
    return {"k": st["k_out"], "v": st["v_out"]}


# ---- the plain form ---------------------------------------------------------------
def _norm_rope(x, w, cos, sin, rd):
    """RMSNorm over the last dim, then rotation of dims (i, i + rd / 2); x [rows, heads, D]."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    a, b = x[..., :rd // 2], x[..., rd // 2:rd]
    c, s = cos.to(x.dtype)[:, None, :], sin.to(x.dtype)[:, None, :]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., rd:]], -1)


def _quantise(x):
    """x [..., D] in 64 bits (values next to a border between two integers)."""
    scale = (x.abs().amax(-1) / 127).float()
    inv = torch.where(scale > 0, 1.0 / scale.double(), torch.zeros_like(scale, dtype=F64))
    return torch.round(x * inv[..., None]).to(torch.int8), scale


def _places(st):
    """Page and slot of every new row of the batch, in row order."""
    count = st["count"].long()
    seq = torch.repeat_interleave(torch.arange(len(count), device=DEV), count, output_size=st["qkv"].shape[0])
    pos = torch.arange(len(seq), device=DEV) - st["start"].long()[seq] + st["past"].long()[seq]
    return st["tables"].long()[seq, pos // PAGE], pos % PAGE


def _offsets(slot, d):
    """Places of the (slot, dim) elements in a page: [rows, D] of K and of V."""
    s, i = slot[:, None], torch.arange(d, device=DEV)[None]
    block = (s // 32 * (d // 32) + i // 32) * 64
    return ((block + i // 16 % 2 * 32 + s % 32) * 16 + i % 16,
            (block + s // 4 % 2 * 32 + i % 32) * 16 + s // 8 % 4 * 4 + s % 4)


def _run_rows(st):
    case = st["case"]
    _, hkv, d, rd, _, _ = LAYOUTS[case["layout"]]
    page, slot = _places(st)
    koff, voff = _offsets(slot, d)
    at = (page[:, None, None], torch.arange(hkv, device=DEV)[None, :, None])
    head = (page[:, None], at[1][..., 0], slot[:, None])
    if case["kind"] == "write":
        x = st["qkv"][:, st["koff"]:].double().view(-1, 2, hkv, d)
        kq, ks = _quantise(_norm_rope(x[:, 0], st["k_norm"], st["cos"], st["sin"], rd))
        vq, vs = _quantise(x[:, 1])
        st["kp"][(*at, koff[:, None])] = kq
        st["vp"][(*at, voff[:, None])] = vq
        st["ks"][head], st["vs"][head] = ks, vs
    out = torch.float32 if case["kind"] == "write" else torch.bfloat16
    return {"k": (st["kp"][(*at, koff[:, None])].float() * st["ks"][head][..., None]).to(out),
            "v": (st["vp"][(*at, voff[:, None])].float() * st["vs"][head][..., None]).to(out)}


def _run_attend(st):
    case = st["case"]
    hq, hkv, d, rd, _, gated = LAYOUTS[case["layout"]]
    seqs, total = case["seqs"], st["qkv"].shape[0]
    tables, count = st["tables"].long(), st["count"].long()
    rows, group = case["rows"], hq // hkv
    # keys and values of every sequence, padded to the longest
    k, v = _from_pages(st["kp"][tables], st["vp"][tables], d)  # [seqs, pages, hkv, 64, d]
    k = (k.float() * st["ks"][tables][..., None]).transpose(1, 2).reshape(seqs, hkv, -1, d)
    v = (v.float() * st["vs"][tables][..., None]).transpose(1, 2).reshape(seqs, hkv, -1, d)
    # queries, padded to the longest chunk
    qs = 2 * d if gated else d
    x = st["qkv"][:, :hq * qs].float().view(total, hq, qs)
    q = _norm_rope(x[..., :d], st["q_norm"], st["cos"], st["sin"], rd) * d ** -0.5
    r = torch.arange(rows, device=DEV)
    live = r[None] < count[:, None]
    at = (st["start"].long()[:, None] + r[None]).clamp(max=total - 1)
    qp = q[at].view(seqs, rows, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, group * rows, d)
    # visible keys of every row
    p = (st["past"].long()[:, None] + r[None])[..., None]
    j = torch.arange(k.shape[2], device=DEV)
    if case["tree"]:
        n = j - st["past"].long()[0]
        word = st["anc"][:, n.clamp(0, 127) // 32]
        see = ((n < 0) | ((n < rows) & ((word >> (n.clamp(0, 127) % 32)) & 1).bool()))[None]
    else:
        see = j <= p
        if case["window"]:
            see = see & ((j < case["sink"]) | (p - j < case["window"]))
    see = see & live[..., None]
    s = torch.matmul(qp, k.transpose(2, 3).contiguous()).view(seqs, hkv, group, rows, -1)
    s = s.masked_fill_(~see[:, None, None], float("-inf"))
    s = s - s.amax(-1, keepdim=True).clamp(min=-3e38)
    s = s.exp_()
    o = torch.matmul(s.view(seqs, hkv, group * rows, -1), v).view(seqs, hkv, group, rows, d)
    o = o / s.sum(-1, keepdim=True).clamp(min=1e-38)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, rows, hq, d)[live]
    if gated:
        o = o * torch.sigmoid(x[..., d:])
    return o.to(torch.bfloat16).view(total, hq * d)


def run(st):
    if own:
        return _run_own(st)
    return _run_attend(st) if st["case"]["kind"] == "attend" else _run_rows(st)


# ---- the definition in 64 bits ------------------------------------------------------
def _rope64(x, w, cos, sin, rd):
    y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
    z = y.clone()
    half = rd // 2
    c, s = cos.double().unsqueeze(1), sin.double().unsqueeze(1)
    z[..., :half] = y[..., :half] * c - y[..., half:rd] * s
    z[..., half:rd] = y[..., half:rd] * c + y[..., :half] * s
    return z


def exact(case, seed):
    hq, hkv, d, rd, _, gated = LAYOUTS[case["layout"]]
    st = _inputs(case, seed)
    past, rows, starts = st["host"]
    if case["kind"] == "write":
        kv = st["qkv"][:, -2 * hkv * d:].double()
        k = _rope64(kv[:, :hkv * d].reshape(-1, hkv, d), st["k_norm"], st["cos"], st["sin"], rd)
        v = kv[:, hkv * d:].reshape(-1, hkv, d)

        def stands_for(x):
            scale = (x.abs().max(-1, keepdim=True).values / 127).float().double()
            return (x / scale).round() * scale

        return {"k": stands_for(k), "v": stands_for(v)}
    ks, vs = [], []
    for s, (p, n) in enumerate(zip(past, rows)):
        pages = st["tables"][s, :(p + n + PAGE - 1) // PAGE].long()
        for parts, q8, scale in ((ks, st["kq"], st["ks"]), (vs, st["vq"], st["vs"])):
            x = q8[pages].double() * scale[pages].double().unsqueeze(-1)  # [pages, hkv, 64, d]
            parts.append(x.transpose(0, 1).reshape(hkv, -1, d)[:, :p + n])
    if case["kind"] == "read":
        return {"k": torch.cat([x[:, p:].transpose(0, 1) for x, p in zip(ks, past)]),
                "v": torch.cat([x[:, p:].transpose(0, 1) for x, p in zip(vs, past)])}
    qs = 2 * d if gated else d
    x = st["qkv"][:, :hq * qs].double().reshape(-1, hq, qs)
    q = _rope64(x[..., :d], st["q_norm"], st["cos"], st["sin"], rd)
    out = torch.zeros(sum(rows), hq, d, dtype=F64, device=DEV)
    for s, (p, n) in enumerate(zip(past, rows)):
        see = torch.ones(n, p + n, dtype=torch.bool, device=DEV)
        if case["tree"]:
            see[:, p:] = False
            for i, par in enumerate(_tree(case)):
                if par >= 0:
                    see[i, p:] = see[par, p:]
                see[i, p + i] = True
        else:
            see = see.tril(p)
            if case["window"]:
                near = see.triu(p - case["window"] + 1)
                near[:, :case["sink"]] |= see[:, :case["sink"]]
                see = near
        hide = torch.zeros(n, p + n, dtype=F64, device=DEV).masked_fill(~see, float("-inf"))
        for h in range(hq):
            g = h * hkv // hq
            w = torch.softmax(q[starts[s]:starts[s] + n, h] @ ks[s][g].T.contiguous() / math.sqrt(d) + hide, -1)
            out[starts[s]:starts[s] + n, h] = w @ vs[s][g]
    if gated:
        out = out / (1 + torch.exp(-x[..., d:]))
    return out.reshape(-1, hq * d)
