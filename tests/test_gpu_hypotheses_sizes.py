"""The forms that selections, forks and copies take at larger sizes: scans of two blocks of
4096 logits a workgroup (8192 blocks of bf16 and more in all rows), forks of more table entries
than one workgroup shares by itself, copies of more units than there are workgroups."""
import ctypes as C

import numpy as np
import pytest
import torch

from dtree_hip import _native as N

from gpu_util import stream
from test_gpu_beam_select import LSE, Select
from test_gpu_pages import Pool, copy_args, kv


pytestmark = pytest.mark.gpu
CHUNK = 4096


def _logits(dev, n, V, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(n, V, device=dev, generator=g) * 3).to(dtype)


# (3 blocks a row with a last one of 37 logits, 37 with 5, 4 whole ones, 2 with 4095)
@pytest.mark.parametrize("G,K,M,V,dtype", [(86, 64, 5, 2 * CHUNK + 37, torch.float32),
                                           (28, 16, 32, 36 * CHUNK + 5, torch.bfloat16),
                                           (64, 64, 3, 4 * CHUNK, torch.bfloat16),
                                           (43, 64, 5, 2 * CHUNK + 37, torch.bfloat16),
                                           (1025, 8, 8, 2 * CHUNK - 1, torch.float32)])
def test_scans_of_two_blocks(gpu_device, G, K, M, V, dtype):
    """Against the selection in 64 bits, and bit for bit what the same groups give a few at
    a time, whose scans take the blocks one by one."""
    chunks = -(-V // CHUNK)
    assert G * K * chunks >= 8192
    n = G * K
    x = _logits(gpu_device, n, V, dtype, seed=V)
    x[5, CHUNK:] = float("-inf")   # rows whose later blocks hold nothing, or all of it
    x[6, :CHUNK] = float("-inf")
    x[7] = float("nan")
    x[9, 1::2] = -1e10
    g = torch.Generator().manual_seed(G)
    scores = -torch.rand(n, generator=g) * 4
    finished = (torch.rand(n, generator=g) < 0.1).int()
    lengths = torch.randint(0, 9, (n,), generator=g)
    s = Select(gpu_device, G, K, M, V, x, scores, lengths, finished, eos=17, pad=3, penalty=0.7)
    out = s.run()
    few = max(1, min(G // 3, 8191 // (K * chunks)))
    for at in range(0, G, few):
        m = min(few, G - at)
        r = slice(at * K, (at + m) * K)
        part = Select(gpu_device, m, K, M, V, x[r], scores[r], lengths[r], finished[r], eos=17, pad=3, penalty=0.7)
        for k, t in part.run().items():
            whole = out[k][at:at + m]
            if k in ("parents", "sources"):
                whole = torch.where(whole >= 0, whole - at * K, whole)
            assert torch.equal(t, whole), (k, at)
        # in 64 bits
        y = x[r].double().nan_to_num(nan=float("-inf"), neginf=float("-inf"))
        total = s.scores[r].double()[:, None] + torch.log_softmax(y, -1).nan_to_num(nan=float("-inf"), neginf=float("-inf"))
        over = finished[r].bool().to(gpu_device)
        total[over] = float("-inf")
        total[over, 3] = s.scores[r].double()[over]
        size = (lengths[r].to(gpu_device) + (~over).long()).clamp(min=1).double() ** -0.7
        rank = (total * size[:, None]).view(m, K * V)
        best = rank.topk(M, dim=-1).values
        got = ((out["parents"][at:at + m].long() - at * K) % K) * V + out["tokens"][at:at + m].long()
        assert (rank.gather(1, got) - best).abs().max() <= 2 * LSE
        exact = total.view(m, K * V).gather(1, got)
        assert ((out["scores"][at:at + m].double() - exact).abs() <= LSE + 2.0 ** -24 * exact.abs()).all()


# numbers of sequences that are and are no multiple of 4, tables on both sides of 4096
# entries and of its neighbours among the powers of two
@pytest.mark.parametrize("seqs,ld", [(67, 130), (301, 33), (1023, 9), (5, 1700), (3, 2731), (2, 4096), (128, 65), (6, 86),
                                     (33, 32), (41, 50), (64, 64), (91, 45), (127, 64), (64, 128)])
@pytest.mark.parametrize("absent", [-1, 0, 500])
def test_forks_by_several_workgroups(gpu_device, seqs, ld, absent):
    g = np.random.default_rng(seqs + ld)
    pages = max(600, min(seqs * ld // 3, 9000))
    lengths, left = [], pages - 2
    for i in range(seqs):
        n = int(g.integers(0, ld * 64 // 2 + 1)) if i < 8 else int(g.integers(0, 3 * 64))
        n = min(n, max(0, left // 2) * 64)
        left -= -(-n // 64)
        lengths.append(n)
    p = Pool(gpu_device, seqs, ld, pages, absent, seed=ld).fill(lengths)
    p.fork(None, rows=3, in_place=True)
    p.consistent()
    for k in range(4):
        parents = np.minimum(g.integers(0, seqs, seqs), g.integers(0, seqs, seqs))
        parents[g.random(seqs) < 0.1] = -1
        p.fork(parents, advance=int(g.choice([0, 1, 3])), rows=int(g.choice([0, 1, 30])))
        p.consistent()
        p.fork(None, rows=int(g.choice([0, 1, 64])), in_place=bool(k % 2))  # without parents
        p.consistent()
    p.fork([0] * seqs, rows=1)
    p.consistent()
    p.fork(range(seqs), advance=1, rows=0)
    p.consistent()


@pytest.mark.parametrize("layers,heads,dim,bits,n", [(36, 8, 64, 8, 8), (40, 5, 64, 8, 33), (1, 3, 64, 16, 1000)])
def test_copies_of_more_units_than_workgroups(gpu_device, layers, heads, dim, bits, n):
    """Lists that are full and that end early; entries of every kind behind one another."""
    assert n * layers * heads > 2048
    pages = 2 * n + 1
    for count in (n, n - 2, 2, 0):
        pools = kv(gpu_device, layers, pages, heads, dim, bits, seed=n + count)
        want = [t.clone() for t in pools]
        g = np.random.default_rng(n)
        order = g.permutation(pages)
        entries = []
        for i in range(n):
            used = int(g.choice([0, 1, 31, 32, 33, 63, 64]))
            d = int(order[n + i]) if g.random() > 0.1 else pages + i
            entries.append((int(order[i]), d, used) if i < count else (-1, -1, -1))
            if i < count and used and d < pages:
                for t in want:
                    m = t.shape[3] if used > 32 else t.shape[3] // 2
                    t[:, d, :, :m] = t[:, int(order[i]), :, :m]
        copies = torch.tensor(entries, dtype=torch.int32, device=gpu_device)
        N.check(N.lib().dtree_pages_copy(C.byref(copy_args(pools, copies)), stream()), "copy")
        for t, w in zip(pools, want):
            assert torch.equal(t, w), count
