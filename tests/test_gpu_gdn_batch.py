"""dtree_gdn_layer_batch against the layer's core in 64 bits (oracle/gdn.py).

Tolerances. conv: keep + 1 <= 8 products, SiLU with the fast exponential (2^-22 + |x|
2^-23, |x| < 16 here): below 64 * 2^-24 of the taps' absolute sum. The norms of q and k
keep that relative to the head's largest element; dots over 128 columns add 128 * 2^-24
of their absolute sum. So a state element is off by less than 512 * 2^-24 of
A = g |s| + beta (|v| + g sum |s| |k|) |k| with the row's absolute sums, v and k being
bounded by their taps' absolute sums; y by the same of its own absolute sum, and the
norm's division makes that relative to y's root mean square. Outputs: half a step of
their type (16 bits with the low half), then that."""
import ctypes as C

import numpy as np
import pytest
import torch

from dtree_hip import _native as N
from oracle import gdn as og

from gpu_util import stream

pytestmark = pytest.mark.gpu
U = 512 * 2.0 ** -24
EPS = 1e-6


def case(dev, n, hk, hv, keep, seed, pad=32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    dims = 2 * hk * 128 + hv * 128
    width = dims + hv * 130 + (-(hv * 130) % 4) + 4
    c = dict(n=n, hk=hk, hv=hv, keep=keep, dims=dims, proj=r(n, width), window=r(n, keep, dims),
             state=r(n, hv, 128, 128) * 0.3, conv=r(keep + 1, dims) * 0.5, a_log=torch.rand(hv, generator=g) * 2,
             dt=r(hv) - 2, norm=(1 + 0.1 * r(128)).bfloat16())
    c = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    c["window_out"], c["state_out"] = torch.full_like(c["window"], 9.0), torch.full_like(c["state"], 9.0)
    return c


def args(c, out, lo, layout, padded):
    a = N.GdnArgs()
    a.rows_padded = padded; a.num_k_heads = c["hk"]; a.num_v_heads = c["hv"]; a.head_k_dim = a.head_v_dim = 128
    a.conv_keep = c["keep"]; a.proj = c["proj"].data_ptr(); a.ld_proj = c["proj"].shape[1]
    a.window = c["window"].data_ptr(); a.conv_w = c["conv"].data_ptr(); a.A_log = c["a_log"].data_ptr()
    a.dt_bias = c["dt"].data_ptr(); a.state = c["state"].data_ptr()
    a.norm_w = c["norm"].data_ptr(); a.eps = EPS
    a.out = out.data_ptr(); a.out_lo = lo.data_ptr() if lo is not None else None
    a.out_layout = layout; a.ld_out = out.shape[1]
    a.window_out = c["window_out"].data_ptr(); a.state_out = c["state_out"].data_ptr()
    return a


def run(c, sources, layout=N.W_ROWMAJOR, low=True, padded=None, st=None):
    dev = c["proj"].device
    padded = padded or c["n"]
    dt = torch.float16 if layout == N.W_TILED_F16 else torch.bfloat16
    out = torch.full((padded, c["hv"] * 128), 3.0, dtype=dt, device=dev)
    lo = torch.full_like(out, 3.0) if low and dt == torch.bfloat16 else None
    src = None if sources is None else torch.tensor(sources, dtype=torch.int32, device=dev)
    a = args(c, out, lo, layout, padded)
    N.check(N.lib().dtree_gdn_layer_batch(C.byref(a), src.data_ptr() if src is not None else None, c["n"],
                                          stream() if st is None else st), "batch")
    torch.cuda.synchronize()
    return out, lo


def untile(t):
    """[rows, width] in the tiled order -> row-major."""
    rows, width = t.shape
    x = t.reshape(rows // 32, width // 64, 4, 2, 32, 8)  # block row, block column, i, half, row, e
    return x.permute(0, 4, 1, 3, 2, 5).reshape(rows, width)


def check(c, sources, out, lo, layout=N.W_ROWMAJOR):
    h = {k: v.double().cpu().numpy() for k, v in c.items() if isinstance(v, torch.Tensor)}
    hk, hv, dims, keep = c["hk"], c["hv"], c["dims"], c["keep"]
    if layout != N.W_ROWMAJOR:
        out, lo = untile(out), None if lo is None else untile(lo)
    got = out.double().cpu().numpy()
    half = 2.0 ** -12 if layout == N.W_TILED_F16 else 2.0 ** -9  # (of a value rounded to the type: eps / 2, its own share)
    if lo is not None:
        got, half = got + lo.double().cpu().numpy(), 2.0 ** -17
    half *= 2
    assert (got[c["n"]:] == 0).all()
    rms = lambda t, eps: t / np.sqrt((t * t).mean(-1, keepdims=True) + eps)  # noqa: E731
    grp = np.arange(hv) // (hv // hk)
    for i in range(c["n"]):
        s = i if sources is None else sources[i]
        live = 0 <= s < c["n"]
        win = h["window"][s] if live else np.zeros((keep, dims))
        S0 = h["state"][s] if live else np.zeros((hv, 128, 128))
        x = h["proj"][i, :dims]
        y, new = og.chain_conv1d(x[None], win, h["conv"])
        assert np.array_equal(h["window_out"][i], new)
        mag = (np.abs(np.vstack([win, x[None]])) * np.abs(h["conv"])).sum(0)  # bounds of the conv outputs
        q, k, v = (y[0, a:b].reshape(-1, 128) for a, b in ((0, hk * 128), (hk * 128, 2 * hk * 128), (2 * hk * 128, dims)))
        q, k = rms(q, 1e-6) / 128, rms(k, 1e-6) / np.sqrt(128)
        z, b, a = (h["proj"][i, dims + lo_:dims + hi_] for lo_, hi_ in ((0, hv * 128), (hv * 128, hv * 129), (hv * 129, hv * 130)))
        g = np.exp(-np.exp(h["a_log"]) * np.logaddexp(0, a + h["dt"]))
        beta = 1 / (1 + np.exp(-b))
        o, S = og.chain_gated_delta(q[None], k[None], v[None], g[None], beta[None], S0)
        # bounds: the heads' norms take a relative error of mag over the head's rms
        qm, km = mag[:hk * 128].reshape(hk, 128), mag[hk * 128:2 * hk * 128].reshape(hk, 128)
        wide = lambda m, y_, f: m / np.sqrt((y_ ** 2).mean(-1, keepdims=True) + 1e-6) * f  # noqa: E731
        ka = wide(km, y[0, hk * 128:2 * hk * 128].reshape(hk, 128), 128 ** -0.5)[grp]
        qa = wide(qm, y[0, :hk * 128].reshape(hk, 128), 1 / 128)[grp]
        va = mag[2 * hk * 128:].reshape(hv, 128)
        G = g[:, None]
        delta = beta[:, None] * (va + G * np.einsum("hvk,hk->hv", np.abs(S0), ka))
        A = G[..., None] * np.abs(S0) + delta[..., None] * ka[:, None]
        err = np.abs(h["state_out"][i] - S)
        # (a gate below fp32's smallest normal number, 2^-126, may be 0: exp(-90) = 2^-129.8 is one)
        tiny = 2.0 ** -126 * (1 + np.abs(S0) + (va + np.einsum("hvk,hk->hv", np.abs(S0), ka))[..., None] * ka[:, None])
        assert (err <= U * A + tiny).all(), (err / (U * A + tiny)).max()
        Y = np.einsum("hvk,hk->hv", A, qa)
        r = np.sqrt((o[0] ** 2).mean(-1, keepdims=True) + EPS)
        w, zz = h["norm"][None], z.reshape(hv, 128)
        want = o[0] / r * w * (zz / (1 + np.exp(-zz)))
        # y's own error, and its share in the norm (the mean over the row)
        rel = U * (Y / r + np.abs(o[0] / r) * np.sqrt(((Y / r) ** 2).mean(-1, keepdims=True)) + np.abs(o[0] / r))
        rel = rel + np.einsum("hvk,hk->hv", tiny, qa) / r  # (the gates' own share of y)
        tol = rel * np.abs(w) * np.abs(zz) + 2.0 ** -126 + half * np.abs(want) + 2.0 ** -24 * (layout == N.W_TILED_F16)
        e = np.abs(got[i].reshape(hv, 128) - want)
        assert (e <= tol).all(), (e / tol).max()


@pytest.mark.parametrize("n,hk,hv,keep", [(1, 16, 32, 3), (3, 2, 4, 3), (5, 1, 1, 1), (8, 3, 3, 7), (2, 2, 8, 2), (37, 2, 4, 3),
                                          (4, 1, 4, 4), (3, 2, 2, 5), (2, 1, 2, 6)])
def test_batch(gpu_device, n, hk, hv, keep):
    c = case(gpu_device, n, hk, hv, keep, seed=n + keep)
    src = [(3 * i + 1) % n for i in range(n)]
    if n > 3:
        src[1], src[2], src[3] = src[0], -1, n + 5  # one source twice, two sequences that begin
    before = {k: c[k].clone() for k in ("window", "state")}
    out, lo = run(c, src)
    check(c, src, out, lo)
    assert all(torch.equal(before[k], c[k]) for k in before)


@pytest.mark.parametrize("layout,low", [(N.W_ROWMAJOR, False), (N.W_TILED, True), (N.W_TILED, False), (N.W_TILED_F16, False)])
@pytest.mark.parametrize("n,padded", [(1, 32), (32, 32), (33, 96)])
def test_layouts_and_padding_rows(gpu_device, layout, low, n, padded):
    c = case(gpu_device, n, 2, 4, 3, seed=n)
    out, lo = run(c, None, layout, low, padded)
    check(c, None, out, lo, layout)


def test_gates_at_their_ends(gpu_device):
    """g from 0 to 1, beta 0 and 1, z and conv inputs far out: finite, and right."""
    c = case(gpu_device, 4, 1, 2, 3, seed=5)
    b0 = c["dims"] + 2 * 128
    c["proj"][:, b0:b0 + 2] = torch.tensor([[-200.0, 200.0], [90.0, -90.0], [0.0, 0.0], [-20.0, 20.0]], device=gpu_device)
    c["proj"][:, b0 + 2:b0 + 4] = torch.tensor([[80.0, -80.0], [-300.0, 300.0], [19.0, 22.0], [0.0, 5.0]], device=gpu_device)
    out, lo = run(c, None)
    assert torch.isfinite(out).all() and torch.isfinite(c["state_out"]).all()
    check(c, None, out, lo)
    c["proj"][0, :c["dims"]] = 0.0  # q = k = v = 0 for a sequence that begins: all zeros
    c["window"][0] = 0.0
    out, lo = run(c, [-1, 1, 2, 3])
    assert (out[0] == 0).all() and (c["state_out"][0] == 0).all()


def test_a_sequences_nan_stays_its_own(gpu_device):
    c = case(gpu_device, 4, 2, 4, 3, seed=6)
    ref, _ = run(c, [0, 1, 2, 3])
    state = c["state_out"].clone()
    c["state"][2] = float("nan")
    c["proj"][1] = float("inf")
    out, _ = run(c, [0, 1, 2, 3])
    for i in (0, 3):
        assert torch.equal(out[i], ref[i]) and torch.equal(c["state_out"][i], state[i])


def test_states_past_32_bit_offsets(gpu_device):
    """2064 sequences of 32 heads: 1.08e9 state elements, 4.3 GB."""
    n, dev = 2064, gpu_device
    c = case(dev, 1, 1, 32, 3, seed=7)
    big = dict(c, n=n, proj=c["proj"].expand(n, -1).contiguous(), window=c["window"].expand(n, -1, -1).contiguous(),
               state=torch.zeros(n, 32, 128, 128, device=dev))
    big["state"][n - 1] = c["state"][0]
    big["window_out"] = torch.empty_like(big["window"])
    big["state_out"] = torch.empty_like(big["state"])
    ref, _ = run(c, None)
    out, _ = run(big, [n - 1] * 2 + [5] * (n - 4) + [n - 1] * 2)
    for i in (0, 1, n - 2, n - 1):
        assert torch.equal(big["state_out"][i], c["state_out"][0]) and torch.equal(out[i], ref[0])


def test_follows_the_chain(gpu_device):
    """Tokens one by one, beside another sequence: the layer over a prompt (dtree_gdn_layer_chain)."""
    lib, dev, T = N.lib(), gpu_device, 6
    c = case(dev, T, 2, 4, 3, seed=8)
    f32 = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    ref = dict(window=c["window"][0].clone(), state=c["state"][0].clone())
    out = torch.zeros(32, 512, dtype=torch.bfloat16, device=dev)
    a = args(c, out, None, N.W_ROWMAJOR, 32)
    proj = f32(32, c["proj"].shape[1])
    proj[:T] = c["proj"]
    bufs = dict(q=f32(32, 256), k=f32(32, 256), v=f32(32, 512), g=f32(32, 4), beta=f32(32, 4), y=f32(32, 512))
    for k, t in bufs.items():
        setattr(a, k, t.data_ptr())
    a.proj = proj.data_ptr(); a.window = ref["window"].data_ptr(); a.state = ref["state"].data_ptr()
    a.window_out = a.state_out = None
    N.check(lib.dtree_gdn_layer_chain(C.byref(a), T, stream()), "chain")
    two = case(dev, 2, 2, 4, 3, seed=9)
    for k in ("conv", "a_log", "dt", "norm"):
        two[k] = c[k]
    two["window"][1], two["state"][1] = c["window"][0], c["state"][0]
    got = []
    for t in range(T):
        two["proj"][1] = c["proj"][t]
        got.append(run(two, None, low=False)[0][1].clone())
        for k in ("window", "state"):
            two[k], two[k + "_out"] = two[k + "_out"], two[k]
    assert torch.equal(two["window"][1], ref["window"])
    # two ways of one recurrence in fp32 over T steps: each within U of the absolute sums (below 4 here)
    assert float((two["state"][1] - ref["state"]).abs().max()) <= 2 * T * U * 4
    got = torch.stack(got).float()
    scale = out[:T].float().abs().amax(-1, keepdim=True)
    assert bool(((got - out[:T].float()).abs() <= 2 * 2.0 ** -8 * out[:T].float().abs() + 2 * T * U * scale).all())


def test_replayed_graph(gpu_device):
    """Window and state sides change between two graphs, as a decoder's do."""
    lib, dev = N.lib(), gpu_device
    c = case(dev, 3, 2, 4, 3, seed=10)
    src = torch.tensor([2, 0, 0], dtype=torch.int32, device=dev)
    out = torch.zeros(3, 512, dtype=torch.bfloat16, device=dev)
    side = torch.cuda.Stream()
    graphs = []
    for turn in (0, 1):
        a = args(c, out, None, N.W_ROWMAJOR, 3)
        if turn:
            a.window, a.window_out, a.state, a.state_out = a.window_out, a.window, a.state_out, a.state
        torch.cuda.synchronize()
        N.check(lib.dtree_graph_begin(side.cuda_stream), "begin")
        N.check(lib.dtree_gdn_layer_batch(C.byref(a), src.data_ptr(), 3, side.cuda_stream), "batch")
        ex = C.c_void_p()
        N.check(lib.dtree_graph_end(side.cuda_stream, C.byref(ex)), "end")
        graphs.append(ex)
    eager = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    try:
        for k in range(5):
            x = torch.randn(c["proj"].shape, generator=torch.Generator().manual_seed(k)).to(dev)
            c["proj"].copy_(x)
            eager["proj"].copy_(x)
            torch.cuda.synchronize()
            N.check(lib.dtree_graph_launch(graphs[k % 2], side.cuda_stream), "launch")
            torch.cuda.synchronize()
            ref, _ = run(eager, [2, 0, 0], low=False)
            assert torch.equal(out, ref)
            assert torch.equal(c["state" if k % 2 else "state_out"], eager["state_out"])
            for name in ("window", "state"):
                eager[name], eager[name + "_out"] = eager[name + "_out"], eager[name]
    finally:
        torch.cuda.synchronize()
        for ex in graphs:
            lib.dtree_graph_destroy(ex)
