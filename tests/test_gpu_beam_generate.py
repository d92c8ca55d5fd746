"""Beam search over the targets (selection, forked caches, batched recurrent steps
together), and forked pools under the verify engines.

Each step's logits are compared, hypothesis by hypothesis, with a run of the same engine
over that hypothesis' tokens alone on a cache of its own: the paths differ (one token in a
batch against a prompt), so within the 2e-2 of the row maximum that the engines' other
tests grant. The selections made of the step's own logits are checked in 64 bits."""
import numpy as np
import pytest
import torch

from dtree_hip import BeamDecoder, PagedKVPool, Qwen3TreeModel, Qwen3Weights, beam_generate, tiny_qwen3, tiny_qwen35
from dtree_hip.adapters import load_target_model
from dtree_hip.api import DFlashGenerator
from dtree_hip.synthetic import make_tree, random_prefix
from oracle import beam as ob

from test_gpu_beam_select import LSE

pytestmark = pytest.mark.gpu
TOL = 2e-2


def _target(family, max_past=400):
    cfg = tiny_qwen3() if family == "qwen3" else tiny_qwen35()
    return load_target_model(cfg, seed=0, max_past=max_past, norm_jitter=0.1, kv_bits=8)


def _prompts(target, lengths):
    return [list(map(int, random_prefix(n, target.model.args.vocab_size, seed=7 + n))) for n in lengths]


def _alone(target, tokens):
    cache = target.make_cache()
    logits, _ = target.forward_with_hidden_states(torch.tensor([tokens]), cache, list(target.model.engine.layer_ids))
    return logits[0, -1].double().cpu().numpy()


@pytest.mark.parametrize("family", ["qwen3", "qwen3_5"])
@pytest.mark.parametrize("lengths,beams,use_graph", [((63, 5, 140), 4, True), ((64,), 8, False), ((1, 130), 3, True)])
def test_every_hypothesis_is_its_own_sequence(gpu_device, family, lengths, beams, use_graph):
    target = _target(family)
    eng, V = target.model.engine, target.model.args.vocab_size
    prompts = _prompts(target, lengths)
    steps = 7
    first = BeamDecoder(target, prompts, beams, 3, use_graph=False)
    first.start()
    stop = int(first.tokens[1])  # a second-best first token ends that hypothesis at once
    d = BeamDecoder(target, prompts, beams, steps, stop_token=stop, pad_token=1, length_penalty=0.8, use_graph=use_graph)
    d.start()
    assert int(d.finished[1]) == 1 and int(d.cache.sources[1]) == -1
    texts = [[prompts[g] + [t] for t in d.tokens[g * beams:(g + 1) * beams].tolist()] for g in range(len(prompts))]
    texts = [t for group in texts for t in group]
    compared = 0
    while d.made < steps:
        before = [t.cpu().numpy().copy() for t in (d.scores, d.lengths, d.finished)]
        d.step()
        torch.cuda.synchronize()
        logits = eng.logits[:d.rows].double().cpu().numpy()
        ended = before[2] != 0
        for i in range(d.rows):
            if not ended[i] and d.made in (2, 4, steps):
                want = _alone(target, texts[i])
                assert np.abs(logits[i] - want).max() <= TOL * np.abs(want).max(), (d.made, i)
                compared += 1
        # the selection among them
        for g in range(d.groups):
            r = slice(g * beams, (g + 1) * beams)
            total, rank = ob.continuations(logits[r], before[0][r], before[1][r], ended[r], V, 1, 0.8)
            best = np.sort(rank.reshape(-1))[::-1][:beams]
            b, t = d.parents[r].cpu().numpy() - g * beams, d.tokens[r].cpu().numpy()
            assert (np.abs(rank[b, t] - best) <= 2 * LSE).all()
            assert (np.abs(d.scores[r].cpu().numpy() - total[b, t]) <= LSE + 2.0 ** -24 * np.abs(total[b, t])).all()
        parents, tokens = d.parents.tolist(), d.tokens.tolist()
        texts = [texts[p] + ([] if ended[p] else [t]) for p, t in zip(parents, tokens)]
        # the pages: every count is the number of tables that hold the page
        held = torch.bincount(d.cache.pool.table[d.cache.pool.table >= 0].flatten().long(), minlength=d.cache.pool.n_pages)
        assert torch.equal(held.to(torch.int32), d.cache.pool.refs)
    assert compared >= 3 * (d.rows - 3)
    for g, hyps in enumerate(d.hypotheses()):
        for i, h in enumerate(hyps):
            assert prompts[g] + h.tokens == texts[g * beams + i]
            assert h.finished == (h.tokens[-1] == stop) and stop not in h.tokens[:-1]
    d.release()


@pytest.mark.parametrize("family", ["qwen3", "qwen3_5"])
def test_graphs_and_eager_steps_agree(gpu_device, family):
    """Twice by graphs, with the engine's own steps between, and once without."""
    target = _target(family)
    prompts = _prompts(target, (200, 30))
    runs = []
    for use_graph in (True, False, True):
        out, metrics = beam_generate(target, prompts, num_beams=5, max_new_tokens=70, length_penalty=1.0, use_graph=use_graph)
        runs.append([[(h.tokens, h.score, h.finished) for h in hyps] for hyps in out])
        cache = target.make_cache()
        target.model.engine.prefill(cache, prompts[1])
    assert runs[0] == runs[1] == runs[2]
    assert metrics["steps"] == 69 and all(len(h[0]) == 70 for hyps in runs[0] for h in hyps)
    for hyps in runs[0]:
        assert len({tuple(h[0]) for h in hyps}) == 5  # no hypothesis twice
        assert [h[1] for h in hyps] == sorted((h[1] for h in hyps), reverse=True)


@pytest.mark.parametrize("family,quant,max_nodes,groups,beams", [
    ("qwen3", "q4", 32, 2, 6), ("qwen3_5", "q4", 32, 1, 4), ("qwen3", "bf16", 128, 3, 40), ("qwen3_5", "bf16", 64, 7, 9)])
def test_quantised_targets_and_more_rows_than_a_block(gpu_device, family, quant, max_nodes, groups, beams):
    target = load_target_model(tiny_qwen3() if family == "qwen3" else tiny_qwen35(), seed=0, max_past=300, norm_jitter=0.1,
                               quant=quant, kv_bits=8)
    m = target.model
    target.model = type(m)(m.args, m.weights, max_past=300, max_nodes=max_nodes, kv_bits=8)
    prompts = _prompts(target, [20 + 9 * g for g in range(groups)])
    d = BeamDecoder(target, prompts, beams, 4)
    d.start()
    texts = [prompts[i // beams] + [t] for i, t in enumerate(d.tokens.tolist())]
    for _ in range(3):
        d.step()
        torch.cuda.synchronize()
        logits = target.model.engine.logits[:d.rows].double().cpu().numpy()
        for i in range(0, d.rows, 5):
            want = _alone(target, texts[i])
            assert np.abs(logits[i] - want).max() <= TOL * np.abs(want).max(), (d.made, i)
        texts = [texts[p] + [t] for p, t in zip(d.parents.tolist(), d.tokens.tolist())]
    assert [prompts[g] + h.tokens for g, hyps in enumerate(d.hypotheses()) for h in hyps] == texts
    d.release()


def test_two_decoders_and_the_engines_own_steps_in_turns(gpu_device):
    """Decoders interleaved with each other, with verify steps and with a change of the
    engine's hidden layers (whose buffers a captured step holds)."""
    target = _target("qwen3")
    eng = target.model.engine
    prompts = _prompts(target, (40, 90))
    want = [beam_generate(target, [p], num_beams=4, max_new_tokens=9)[0][0] for p in prompts]
    ds = [BeamDecoder(target, [p], 4, 9) for p in prompts]
    for d in ds:
        d.start()
    cache = eng.new_cache()
    eng.prefill(cache, prompts[0])
    for k in range(8):
        if k == 4:
            eng.set_layer_ids([1])
            junk = [torch.full((eng.MP, eng.cfg.hidden_size), 3.0, dtype=torch.bfloat16, device=gpu_device) for _ in range(8)]
        for d in ds:
            d.step()
            _step(eng, cache, k)
    assert all(bool((j == 3.0).all()) for j in junk)
    for d, w in zip(ds, want):
        assert [(h.tokens, h.score) for h in d.hypotheses()[0]] == [(h.tokens, h.score) for h in w]
        with pytest.raises(RuntimeError, match="once"):
            d.start()


def test_another_stream(gpu_device):
    target = _target("qwen3_5")
    prompts = _prompts(target, (50,))
    want, _ = beam_generate(target, prompts, num_beams=3, max_new_tokens=6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = beam_generate(target, prompts, num_beams=3, max_new_tokens=6)
    assert [h.tokens for h in got[0]] == [h.tokens for h in want[0]]


def test_requests_beyond_the_engines_rows_run_in_turns(gpu_device):
    target = _target("qwen3")
    prompts = _prompts(target, (10, 20, 30, 40, 50))
    out, _ = beam_generate(target, prompts, num_beams=12, max_new_tokens=6)  # 2 requests of 12 at a time
    assert [len(h) for h in out] == [12] * 5
    one, _ = beam_generate(target, prompts[2:3], num_beams=12, max_new_tokens=6)
    # (beside another request the GEMMs see other rows, not other sums)
    assert [h.tokens for h in out[2]] == [h.tokens for h in one[0]]


def test_one_beam_is_the_greedy_continuation(gpu_device):
    target = _target("qwen3")
    prompt = _prompts(target, (40,))[0]
    gen = DFlashGenerator(target_model=target, draft_model=object())
    res = gen.generate_from_tokens(prompt, max_new_tokens=20, decode_mode="beam", num_beams=1)
    assert res.metrics["decode_mode"] == "beam" and len(res.generated_tokens) == 20
    assert res.output_tokens == prompt + res.generated_tokens
    for n in (0, 7, 19):
        want = _alone(target, prompt + res.generated_tokens[:n])
        assert want[res.generated_tokens[n]] >= want.max() - TOL * np.abs(want).max()


def test_all_hypotheses_end(gpu_device):
    """Every first token of one beam is the stop token: the search ends behind the prompts."""
    target = _target("qwen3")
    prompt = _prompts(target, (33,))[0]
    out, _ = beam_generate(target, [prompt], num_beams=1, max_new_tokens=1)
    stop = out[0][0].tokens[0]
    out, metrics = beam_generate(target, [prompt], num_beams=1, max_new_tokens=50, stop_token_ids={stop})
    assert out[0][0].tokens == [stop] and out[0][0].finished and metrics["steps"] == 0


def test_refusals(gpu_device):
    target = _target("qwen3")
    V = target.model.args.vocab_size
    with pytest.raises(ValueError, match="max_nodes"):
        beam_generate(target, [[1]], num_beams=33, max_new_tokens=2)
    with pytest.raises(ValueError, match="num_beams"):
        beam_generate(target, [[1]], num_beams=0, max_new_tokens=2)
    with pytest.raises(ValueError, match="one stop token"):
        beam_generate(target, [[1]], stop_token_ids={1, 2}, max_new_tokens=2)
    with pytest.raises(ValueError, match="max_past"):
        beam_generate(target, [[1] * 399], max_new_tokens=2)
    with pytest.raises(ValueError, match="holds a token"):
        beam_generate(target, [[1], []], max_new_tokens=2)
    with pytest.raises(ValueError, match="vocabulary"):
        beam_generate(target, [[V]], max_new_tokens=2)
    with pytest.raises(ValueError, match="positive"):
        beam_generate(target, [[1]], max_new_tokens=0)
    with pytest.raises(RuntimeError, match="start"):
        BeamDecoder(target, [[1]], 2, 3).step()
    sixteen = load_target_model(tiny_qwen3(), max_past=200)
    with pytest.raises(ValueError, match="8-bit"):
        beam_generate(sixteen, [[1]], max_new_tokens=2)


# ---- forked pools under the verify engines -------------------------------------------
def _engine(dev, kv_bits):
    cfg = tiny_qwen3()
    return Qwen3TreeModel(cfg, Qwen3Weights.random(cfg, seed=0, device=dev, norm_jitter=0.1), max_past=300,
                          kv_bits=kv_bits).engine


def _step(eng, cache, seed):
    tree = make_tree(4, eng.cfg.vocab_size, seed=seed)
    P = cache.offset
    return eng.verify(cache, tree.tokens, tree.positions(P), tree.parents, use_graph=True)


@pytest.mark.parametrize("kv_bits", [16, 8])
def test_forked_prompts_verify_like_caches_of_their_own(gpu_device, kv_bits):
    """A prompt in three candidates, each verified on by itself, and forked again: the same
    kernels on the same values, so the same results, bit for bit."""
    eng = _engine(gpu_device, kv_bits)
    prompt = random_prefix(150, eng.cfg.vocab_size, seed=3)
    own = [eng.new_cache() for _ in range(3)]
    for c in own:
        eng.prefill(c, prompt)
    pool = eng.new_pool(3, num_pages=20)
    pool.start([150])
    eng.prefill(pool.sequence(0), prompt)
    assert pool.lengths == [150, 0, 0]
    pool.fork([0, 0, 0], rows=eng.max_nodes)
    assert int((pool.refs == 3).sum()) == 2  # whole pages of the prompt
    lens = []
    for i in range(3):
        for k in range(2):
            a, b = _step(eng, pool.sequence(i), 10 + i), _step(eng, own[i], 10 + i)
            assert (a.accepted, a.bonus_token, a.posterior) == (b.accepted, b.bonus_token, b.posterior)
            if k == 0:
                pool.fork(None, rows=eng.max_nodes)
        lens.append(own[i].offset)
    assert pool.lengths == lens
    pool.fork([2, 0, 2], rows=eng.max_nodes)
    assert pool.lengths == [lens[2], lens[0], lens[2]]
    for i, j in ((1, 0), (0, 2)):
        a, b = _step(eng, pool.sequence(i), 20 + i), _step(eng, own[j], 20 + i)
        assert (a.accepted, a.bonus_token, a.posterior) == (b.accepted, b.bonus_token, b.posterior)
        n = own[j].offset
        for layer in range(eng.cfg.num_hidden_layers):
            assert torch.equal(pool.sequence(i).logical_keys(layer, n), own[j].logical_keys(layer, n))
            assert torch.equal(pool.sequence(i).logical_values(layer, n), own[j].logical_values(layer, n))
    # the third still holds the fork's positions
    assert torch.equal(pool.sequence(2).logical_keys(0, lens[2]), own[2].logical_keys(0, lens[2]))
    pool.fork([-1, -1, -1])
    assert int(pool.refs.sum()) == 0 and pool.lengths == [0, 0, 0]


def test_pool_refusals(gpu_device):
    eng = _engine(gpu_device, 16)
    pool = eng.new_pool(2, num_pages=4)
    pool.start([130])
    pool.sequence(0).offset = 130  # (as a prompt's run leaves it)
    with pytest.raises(RuntimeError, match="used up"):
        pool.fork([0, 0], rows=100)
    with pytest.raises(ValueError):
        pool.fork([0])
    with pytest.raises(ValueError):
        pool.fork([0, 2])
    with pytest.raises(ValueError, match="capacity"):
        pool.fork(None, rows=10_000)
    with pytest.raises(RuntimeError, match="used up"):
        pool.start([130, 130])
    with pytest.raises(ValueError):
        pool.start([1, 1, 1])
    with pytest.raises(IndexError):
        pool.sequence(2)
    with pytest.raises(ValueError, match="8-bit"):
        pool.batch(0)
    for kw in (dict(kv_bits=4), dict(num_seqs=0), dict(capacity=0), dict(head_dim=96, kv_bits=8), dict(num_pages=0, kv_bits=8)):
        args = dict(layers=1, kv_heads=1, head_dim=64, capacity=64, num_seqs=1)
        args.update(kw)
        with pytest.raises(ValueError):
            PagedKVPool(**args)
