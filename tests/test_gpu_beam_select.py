"""dtree_beam_select against the selection in 64 bits (oracle/beam.py).

Tolerance of the sums: lse is a sum of V terms exp2((x - m) log2 e) in fp32. A term is
off by |x - m| 2^-23 (two roundings of the argument) + 2^-22 (the instruction), which
weighted with the terms is at most log(V) 2^-23 + 2^-22 of the sum (the mean of m - x is
below log V); the additions (16 in a thread, 8 levels above) by 24 * 2^-24; that and the
chunks' factors stay below 64 * 2^-24 = 3.8e-6 for V up to 2^20. The output's rounding is
2^-24 of it. Ranks are compared where the oracle's own differ by more than twice that."""
import ctypes as C

import numpy as np
import pytest
import torch

from dtree_hip import _native as N
from oracle import beam as ob

from gpu_util import stream

pytestmark = pytest.mark.gpu
LSE = 64 * 2.0 ** -24


class Select:
    def __init__(self, dev, G, K, M, V, logits, scores, lengths=None, finished=None, eos=-1, pad=0, penalty=0.0, ld=None):
        self.G, self.K, self.M, self.V = G, K, M, V
        self.eos, self.pad, self.penalty = eos, pad, penalty
        self.logits = logits
        self.scores = torch.as_tensor(scores, dtype=torch.float32).to(dev).contiguous()
        i32 = lambda t: None if t is None else torch.as_tensor(t, dtype=torch.int32).to(dev).contiguous()  # noqa: E731
        self.lengths, self.finished = i32(lengths), i32(finished)
        self.out = dict(scores=torch.full((G, M), 7.0, device=dev))
        for k in ("tokens", "parents", "lengths", "finished", "sources"):
            self.out[k] = torch.full((G, M), 77, dtype=torch.int32, device=dev)
        a = self.args = N.BeamArgs()
        a.logits = logits.data_ptr(); a.type = N.T_BF16 if logits.dtype == torch.bfloat16 else N.T_F32
        a.ld_logits = ld or logits.stride(0); a.vocab = V; a.groups = G; a.beams = K; a.num_select = M
        a.scores = self.scores.data_ptr()
        a.lengths = self.lengths.data_ptr() if lengths is not None else None
        a.finished = self.finished.data_ptr() if finished is not None else None
        a.eos_token = eos; a.pad_token = pad; a.length_penalty = penalty
        for k, t in self.out.items():
            setattr(a, k + "_out", t.data_ptr())
        size = N.lib().dtree_beam_select_workspace_bytes(C.byref(a))
        assert size > 0
        self.ws = torch.full((size,), 255, dtype=torch.uint8, device=dev)  # (NaN in every word)
        a.workspace = self.ws.data_ptr(); a.workspace_bytes = size

    def run(self, st=None):
        N.check(N.lib().dtree_beam_select(C.byref(self.args), stream() if st is None else st), "select")
        return self.out

    def want(self):
        n = self.G * self.K
        zeros = np.zeros(n, int)
        return (self.scores.cpu().numpy().reshape(-1),
                zeros if self.lengths is None else self.lengths.cpu().numpy().reshape(-1),
                zeros if self.finished is None else self.finished.cpu().numpy().reshape(-1))

    def check(self, out=None, exact=False, inputs=None):
        out = {k: v.cpu().numpy() for k, v in (out or self.out).items()}
        scores, lengths, finished = inputs or self.want()
        x = self.logits[:, :self.V].float().nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf")).cpu().numpy()
        ref = ob.select(x, scores, lengths, finished, self.G, self.K, self.M, self.eos, self.pad, self.penalty)
        if exact:
            for k in ("tokens", "parents", "lengths", "finished", "sources"):
                assert np.array_equal(out[k], ref[k]), (k, out[k], ref[k])
        for g in range(self.G):
            r = slice(g * self.K, (g + 1) * self.K)
            total, rank = ob.continuations(x[r], scores[r], lengths[r], finished[r], self.V, self.pad, self.penalty)
            best = np.sort(rank.reshape(-1))[::-1][:self.M]
            best = best[best > -np.inf]
            n = len(best)
            assert (out["tokens"][g, n:] == -1).all() and (out["parents"][g, n:] == -1).all()
            assert (out["scores"][g, n:] == -np.inf).all() and (out["sources"][g, n:] == -1).all()
            assert (out["lengths"][g, n:] == 0).all() and (out["finished"][g, n:] == 0).all()
            b, t = out["parents"][g, :n] - g * self.K, out["tokens"][g, :n]
            assert (b >= 0).all() and (b < self.K).all() and (t >= 0).all() and (t < self.V).all()
            assert len(set(zip(b.tolist(), t.tolist()))) == n  # no continuation twice
            got = total[b, t]
            assert np.isfinite(got).all()
            with np.errstate(invalid="ignore"):
                off = np.abs(out["scores"][g, :n] - got)
            assert (off <= LSE + 2.0 ** -24 * np.abs(got)).all(), off.max()
            # each rank's value, with the sums' error scaled as the ranks are
            size = np.maximum(lengths[r][b] + (finished[r][b] == 0), 1).astype(float) ** -self.penalty
            tol = 2 * LSE * max(1.0, float(size.max(initial=1.0)))
            assert (np.abs(rank[b, t] - best) <= tol).all()
            over = finished[r][b] != 0
            end = over | (t == self.eos)
            assert np.array_equal(out["finished"][g, :n], end.astype(int))
            assert np.array_equal(out["sources"][g, :n], np.where(end, -1, b + g * self.K))
            assert np.array_equal(out["lengths"][g, :n], lengths[r][b] + np.where(over, 0, 1))


def rows(dev, n, V, dtype=torch.float32, seed=0, spread=3.0, pad_cols=0, offset=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    flat = torch.randn(n * (V + pad_cols) + offset, generator=g) * spread
    return flat.to(dev).to(dtype)[offset:].view(n, V + pad_cols)


def scores_of(n, seed=0):
    return (-torch.rand(n, generator=torch.Generator().manual_seed(seed + 1)) * 4).tolist()


SHAPES = [(1, 1, 1, 1), (1, 1, 4, 3), (2, 1, 8, 31), (3, 5, 10, 4097), (2, 64, 64, 1000), (5, 3, 2, 33),
          (1, 4, 4, 151936), (7, 8, 16, 12289), (1, 64, 64, 32), (2, 2, 64, 4096), (1, 7, 64, 8191)]


@pytest.mark.parametrize("G,K,M,V", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select(gpu_device, G, K, M, V, dtype):
    s = Select(gpu_device, G, K, M, V, rows(gpu_device, G * K, V, dtype, seed=V + K), scores_of(G * K, V))
    s.run()
    s.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad_cols,offset", [(1, 1), (3, 5), (8, 7)])
def test_rows_at_any_address(gpu_device, dtype, pad_cols, offset):
    x = rows(gpu_device, 12, 5001, dtype, seed=3, pad_cols=pad_cols, offset=offset)
    x[:, 5001:] = 1e30  # what stands between the rows is not read
    s = Select(gpu_device, 3, 4, 9, 5001, x, scores_of(12))
    s.run()
    s.check()


@pytest.mark.parametrize("penalty", [0.0, 0.6, 1.0, -0.5, 16.0])
def test_finished_beams_lengths_and_penalty(gpu_device, penalty):
    G, K, M, V = 6, 8, 16, 3001
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 30, (G * K,), generator=g)
    finished = (torch.rand(G * K, generator=g) < 0.4).int()
    finished[:K] = 1  # a group of finished beams alone
    x = rows(gpu_device, G * K, V, seed=6)
    x[:, 17] += 14.0  # the end token is among the best
    s = Select(gpu_device, G, K, M, V, x, scores_of(G * K, 7), lengths, finished, eos=17, pad=V - 1, penalty=penalty)
    s.run()
    s.check()
    out = s.out["finished"].cpu()
    assert out[0, :K].all() and out[1:].any() and not out[1:].all()


def test_ties_go_to_the_lower_beam_then_the_lower_token(gpu_device):
    """Equal rows and scores: every rank is met by all beams at once."""
    G, K, M, V = 2, 5, 40, 9000
    x = (rows(gpu_device, 1, V, seed=9, spread=2.0) * 4).round() / 4
    s = Select(gpu_device, G, K, M, V, x.expand(G * K, V).contiguous(), [-1.5] * (G * K))
    s.run()
    s.check(exact=True)


@pytest.mark.parametrize("V", [1, 50, 4095, 20000])
@pytest.mark.parametrize("K,M", [(1, 64), (3, 64), (64, 2)])
def test_equal_logits(gpu_device, K, M, V):
    """More ties than any list holds: the first positions win."""
    s = Select(gpu_device, 1, K, M, V, torch.zeros(K, V, device=gpu_device), [0.0] * K)
    s.run()
    s.check(exact=True)


def test_two_values(gpu_device):
    """The best are spread thinly; the rest of the places go to ties behind them."""
    V = 30000
    x = torch.zeros(4, V, device=gpu_device)
    x[:, 777::1013] = 1.0
    s = Select(gpu_device, 2, 2, 64, V, x, [-1.0, -1.0, -2.0, -2.0])
    s.run()
    s.check(exact=True)


def test_best_tokens_in_one_segment_and_in_order(gpu_device):
    """Rising and falling rows: all of the best are neighbours."""
    V = 16384
    up = torch.arange(V, device=gpu_device, dtype=torch.float32) * 1e-3
    s = Select(gpu_device, 1, 2, 64, V, torch.stack([up, up.flip(0)]), [0.0, 0.0])
    s.run()
    s.check(exact=True)


def test_masked_rows_infinities_and_nan(gpu_device):
    G, K, M, V = 5, 4, 8, 6000
    x = rows(gpu_device, G * K, V, seed=11)
    inf = float("inf")
    x[0:4] = -inf                       # a group without any continuation
    x[4] = -inf; x[5, 3:] = -inf        # one row empty, one of three tokens
    x[8, ::3] = float("nan"); x[8, 1::3] = -inf
    x[9, 100] = inf; x[9, 4200] = inf   # all its probability, on the two equally
    x[10] = torch.finfo(torch.float32).min
    x[12:16, 5:] = -torch.finfo(torch.float32).max
    x[13] = float("nan")
    x[16, 10] = 3e38; x[17, 11] = -3e38
    x[18].view(torch.int32)[5::7] = 0x7F800001  # signalling NaNs, of both signs
    x[18].view(torch.int32)[6::7] = -8388607
    s = Select(gpu_device, G, K, M, V, x, scores_of(G * K, 12))
    s.run()
    s.check()
    assert (s.out["tokens"][0] == -1).all()
    b = Select(gpu_device, G, K, M, V, x.bfloat16(), scores_of(G * K, 12))
    b.logits[18].view(torch.int16)[5::7] = 0x7F81
    b.logits[18].view(torch.int16)[6::7] = -127
    b.run()
    b.check()


def test_huge_logits(gpu_device):
    """Rows around 1e30 and at fp32's ends, where differences alone say anything."""
    G, K, M, V = 1, 5, 20, 9001
    x = rows(gpu_device, G * K, V, seed=31)
    x[1] = x[1] * 1e37
    x[2] = x[2] * 1e-38
    x[3] = torch.finfo(torch.float32).max
    x[4] = -3e38
    s = Select(gpu_device, G, K, M, V, x, [0.0, -3.0, -1.0, -2.0, -2.5])
    s.run()
    s.check()


def test_beams_without_a_score(gpu_device):
    """The step behind a prompt run with all beams: one alone is alive."""
    G, K, M, V = 3, 6, 6, 700
    scores = [0.0 if i % K == 0 else float("-inf") for i in range(G * K)]
    scores[K + 2] = float("nan")
    scores[2 * K] = float("-inf")  # a group with no beam at all
    fin = [int(i == 2 * K + 1) for i in range(G * K)]  # (a finished beam without a score neither)
    s = Select(gpu_device, G, K, M, V, rows(gpu_device, G * K, V, seed=13), scores, finished=fin)
    s.run()
    s.check()
    assert (s.out["parents"][2] == -1).all() and (s.out["parents"][0] == 0).all()


@pytest.mark.parametrize("K,V", [(64, 266241), (5, 1 << 20), (3, (1 << 20) - 1)])
def test_more_chunks_than_the_quick_way_takes_and_the_largest_vocabulary(gpu_device, K, V):
    s = Select(gpu_device, 1, K, 64, V, rows(gpu_device, K, V, torch.bfloat16, seed=21), scores_of(K, 22))
    s.run()
    s.check()


@pytest.mark.parametrize("score", [3.0e38, 1e30, 0.0, -1e30, -3.0e38])
@pytest.mark.parametrize("penalty", [0.0, 2.0, -3.0])
def test_scores_at_fp32s_ends(gpu_device, score, penalty):
    """Ranks beyond fp32, and sums in which the logits are lost (all of a beam tie)."""
    s = Select(gpu_device, 1, 3, 12, 5000, rows(gpu_device, 3, 5000, seed=23), [score, score * 0.5, score * 0.25],
               lengths=[3, 9, 70], penalty=penalty)
    out = {k: v.cpu() for k, v in s.run().items()}
    scores, lengths, finished = s.want()
    ref = ob.select(s.logits.cpu().numpy(), scores, lengths, finished, 1, 3, 12, -1, 0, penalty)
    if abs(score) >= 1e30:  # (every sum of a beam rounds to its score: positions decide)
        assert np.array_equal(out["tokens"].numpy(), ref["tokens"]) and np.array_equal(out["parents"].numpy(), ref["parents"])
    assert np.allclose(out["scores"].double().numpy(), ref["scores"], rtol=2.0 ** -23, atol=2 * LSE)


def test_rows_past_32_bit_offsets(gpu_device):
    G, K, V, ld = 33, 64, 90, 1 << 20  # 2112 rows, 2.2e9 elements apart
    x = torch.empty(G * K, ld, dtype=torch.bfloat16, device=gpu_device)
    x[:, :V] = rows(gpu_device, G * K, V, torch.bfloat16, seed=14)
    s = Select(gpu_device, G, K, 8, V, x, scores_of(G * K, 15))
    s.run()
    s.check()


def test_outputs_in_place_of_the_inputs_and_optional_ones(gpu_device):
    G, K, V = 4, 8, 5000
    s = Select(gpu_device, G, K, K, V, rows(gpu_device, G * K, V, seed=16), scores_of(G * K, 17),
               lengths=list(range(G * K)), finished=[i % 5 == 0 for i in range(G * K)], eos=3, penalty=1.0)
    inputs = s.want()
    ref = {k: v.clone() for k, v in s.run().items()}
    s.check()
    s.args.scores_out = s.scores.data_ptr(); s.args.lengths_out = s.lengths.data_ptr()
    s.args.finished_out = s.finished.data_ptr(); s.args.sources_out = None
    s.run()
    for k, t in (("scores", s.scores), ("lengths", s.lengths), ("finished", s.finished)):
        assert torch.equal(t.view(G, K), ref[k]), k
    s.check(dict(ref), inputs=inputs)
    s.args.lengths_out = s.args.finished_out = None
    s.run()
    torch.cuda.synchronize()


def test_replayed_graph_and_another_stream(gpu_device):
    s = Select(gpu_device, 4, 8, 8, 20000, rows(gpu_device, 32, 20000, seed=18), scores_of(32, 19))
    lib = N.lib()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    N.check(lib.dtree_graph_begin(side.cuda_stream), "begin")
    s.run(side.cuda_stream)
    ex = C.c_void_p()
    N.check(lib.dtree_graph_end(side.cuda_stream, C.byref(ex)), "end")
    try:
        for seed in range(4):
            s.logits.copy_(rows(gpu_device, 32, 20000, seed=20 + seed))
            side.wait_stream(torch.cuda.current_stream())
            N.check(lib.dtree_graph_launch(ex, side.cuda_stream), "launch")
            torch.cuda.synchronize()
            got = {k: v.clone() for k, v in s.out.items()}
            s.check(got)
            for v in s.out.values():
                v.zero_()
            s.run()
            assert all(torch.equal(got[k], s.out[k]) for k in got)
    finally:
        torch.cuda.synchronize()
        lib.dtree_graph_destroy(ex)
