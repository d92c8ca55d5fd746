"""The verify engines on an 8-bit KV cache (kv_bits = 8): prefill, tree steps
(eager and from a graph), compaction and generation.

The last layer's attention is recomputed in 64 bits from what the engine itself
holds after a step (the fused projection's rows, the cache, the lengths), with
the tolerance of test_gpu_kv_q8; its cached rows have to be the definition's
bytes. Runs of the same engine that take other paths (one token at a time, a
prompt in pieces) agree within the 2e-2 of the row maximum that the engines'
other tests grant."""
import ctypes as C

import numpy as np
import pytest
import torch

from dtree_hip import Qwen3TreeModel, Qwen3Weights, Qwen35TreeModel, Qwen35Weights, tiny_qwen3, tiny_qwen35
from dtree_hip import _native as N
from dtree_hip.adapters import load_target_model
from dtree_hip.cache import PagedKVCacheQ8, quantise_q8
from dtree_hip.dtree_runtime import dtree_generate
from dtree_hip.synthetic import random_prefix
from dtree_hip.weights import W_TILED_F16

from gpu_util import random_tree
from test_gpu_generate import BLOCK, ScriptedDrafter, _gpu_sequential_greedy
from test_gpu_kv_q8 import FP16, PAIR, Batch, check, norm_rope

pytestmark = pytest.mark.gpu
TOL = 2e-2


def _engine(dev, family, max_past=400, max_nodes=32, layer_ids=(0, 1)):
    if family == "qwen3":
        cfg = tiny_qwen3()
        w = Qwen3Weights.random(cfg, seed=0, device=dev, norm_jitter=0.1)
        return Qwen3TreeModel(cfg, w, max_past=max_past, max_nodes=max_nodes, layer_ids=layer_ids, kv_bits=8).engine
    cfg = tiny_qwen35()
    w = Qwen35Weights.random(cfg, seed=0, device=dev, norm_jitter=0.1)
    return Qwen35TreeModel(cfg, w, max_past=max_past, max_nodes=max_nodes, layer_ids=layer_ids, kv_bits=8).engine


def _kv(eng, cache):
    """(8-bit cache, its last layer, that layer's weights)."""
    kv = cache if isinstance(cache, PagedKVCacheQ8) else cache.kv
    li = eng.cfg.num_hidden_layers - 1
    return kv, kv.layers - 1, eng.w.layers[li]


def _reference(eng, cache, qkv, cos, sin, past, n, parents):
    """Batch.reference over the engine's own buffers."""
    c = eng.cfg
    kv, layer, lw = _kv(eng, cache)
    gated = hasattr(c, "rope_dims")
    b = Batch.__new__(Batch)
    b.dev, b.past, b.rows, b.starts, b.total = kv.k_pages.device, [past], [n], [0], qkv.shape[0]
    b.hq, b.hkv, b.d, b.gated = c.num_attention_heads, c.num_key_value_heads, c.head_dim, gated
    b.rd = c.rope_dims if gated else c.head_dim
    b.qkv, b.q_norm, b.cos, b.sin = qkv, lw.q_norm, cos, sin
    one = PagedKVCacheQ8.__new__(PagedKVCacheQ8)  # the last layer as layer 0
    one.__dict__.update(kv.__dict__)
    one.k_pages, one.v_pages = kv.k_pages[layer:], kv.v_pages[layer:]
    one.k_scales, one.v_scales = kv.k_scales[layer:], kv.v_scales[layer:]
    b.cache = one
    want, tol = b.reference(parents=parents)
    want[n:] = 0
    # the cached rows are the projection's, by the definition
    x = qkv[:n, qkv.shape[1] - 2 * b.hkv * b.d:].double().view(n, 2, b.hkv, b.d)
    k, v = norm_rope(x[:, 0], lw.k_norm, cos[:n], sin[:n], b.rd), x[:, 1]
    for got, rows in ((one.logical_keys(0, past + n)[past:], k), (one.logical_values(0, past + n)[past:], v)):
        q, scale = quantise_q8(rows)
        assert torch.equal(got, q.float() * scale[..., None])
    return want, tol


def _attn_rows(eng, attn, rows, width):
    """The attention buffer (the weights' layout) as rows, and its rounding."""
    at = torch.arange(rows, device=attn.device)[:, None], torch.arange(width, device=attn.device)[None]
    r, k = at
    i = ((((r >> 5) * (width >> 6) + (k >> 6)) * 4 + ((k & 31) >> 3)) * 512 + ((r & 31) + 32 * ((k & 63) >> 5)) * 8
         + (k & 7))
    f = [p.reshape(-1)[i].double() for p in attn]
    return (f[0], FP16) if eng.w.layout == W_TILED_F16 else (f[0] + f[1], PAIR)


@pytest.mark.parametrize("family", ["qwen3", "qwen3_5"])
@pytest.mark.parametrize("past,nodes", [(0, 5), (70, 25), (300, 32)])
def test_tree_step_attends_over_its_8_bit_rows(gpu_device, family, past, nodes):
    eng = _engine(gpu_device, family)
    cache = eng.new_cache()
    if past:
        eng.prefill(cache, random_prefix(past, eng.cfg.vocab_size, seed=past))
    parents = random_tree(nodes, seed=nodes)
    depth = [0] * nodes
    for i in range(1, nodes):
        depth[i] = depth[parents[i]] + 1
    toks = random_prefix(nodes, eng.cfg.vocab_size, seed=1)
    eng.forward_only(cache, toks, [past + d for d in depth], parents)
    torch.cuda.synchronize()
    want, tol = _reference(eng, cache, eng.qkv, eng.rope_cos, eng.rope_sin, past, nodes, parents)
    got, rounding = _attn_rows(eng, eng.attn, eng.MP, eng.cfg.q_dim)
    check(got, want, tol + 2.0 ** -25, rounding, family)


@pytest.mark.parametrize("family", ["qwen3", "qwen3_5"])
@pytest.mark.parametrize("head,tokens,segment", [(0, 200, 1024), (70, 300, 128)])
def test_prefill_attends_over_its_8_bit_rows(gpu_device, family, head, tokens, segment):
    eng = _engine(gpu_device, family)
    eng.PREFILL_SEGMENT = segment
    cache = eng.new_cache()
    toks = random_prefix(head + tokens, eng.cfg.vocab_size, seed=tokens)
    if head:
        eng.prefill(cache, toks[:head])  # under 128 tokens: chains of tree steps
    eng.prefill_long(cache, toks[head:])
    torch.cuda.synchronize()
    assert cache.offset == head + tokens
    n = (tokens - 1) % segment + 1  # the last segment
    pf = eng._pf
    past = head + tokens - n
    want, tol = _reference(eng, cache, pf["qkv"][:n], pf["cos"][:n], pf["sin"][:n], past, n, None)
    got, rounding = _attn_rows(eng, pf["attn"], 128 * ((n + 127) // 128), eng.cfg.q_dim)
    assert bool((got[n:] == 0).all())
    check(got[:n], want, tol + 2.0 ** -25, rounding, family)


@pytest.mark.parametrize("family", ["qwen3", "qwen3_5"])
def test_verify_from_a_graph_commits_what_the_eager_step_does(gpu_device, family):
    """Several steps, the same tree shapes eager and captured: equal results, equal caches."""
    runs = []
    for use_graph in (False, True):
        eng = _engine(gpu_device, family)
        cache = eng.new_cache()
        toks = random_prefix(150, eng.cfg.vocab_size, seed=2)
        eng.prefill(cache, toks)
        seen = []
        for step in range(4):
            nodes = 6 + 5 * step
            parents = random_tree(nodes, seed=step)
            depth = [0] * nodes
            for i in range(1, nodes):
                depth[i] = depth[parents[i]] + 1
            P = cache.offset
            ids = random_prefix(nodes, eng.cfg.vocab_size, seed=10 + step)
            for i in range(3):  # the tree follows the target for a few nodes, so that paths are accepted
                res = eng.verify(cache, ids, [P + d for d in depth], parents, use_graph=use_graph, commit=False)
                last = res.accepted[-1]
                child = next((j for j in range(nodes) if parents[j] == last), None)
                if child is None:
                    break
                ids[child] = res.bonus_token
            res = eng.verify(cache, ids, [P + d for d in depth], parents, use_graph=use_graph)
            assert cache.offset == P + len(res.accepted)
            seen.append((res.accepted, res.bonus_token))
        kv, layer, _ = _kv(eng, cache)
        runs.append((seen, cache.offset, kv.logical_keys(layer, cache.offset).clone(),
                     kv.logical_values(0, cache.offset).clone()))
    assert runs[0][:2] == runs[1][:2]
    assert torch.equal(runs[0][2], runs[1][2]) and torch.equal(runs[0][3], runs[1][3])
    assert max(len(a) for a, _ in runs[0][0]) > 1, runs[0][0]


@pytest.mark.parametrize("family", ["qwen3", "qwen3_5"])
def test_generate_on_an_8_bit_cache_is_its_own_greedy_run(gpu_device, monkeypatch, family):
    monkeypatch.setenv("DTREE_QWEN35_TREE_MODE", "full_tree")
    cfg = tiny_qwen3() if family == "qwen3" else tiny_qwen35()
    target = load_target_model(cfg, seed=0, max_past=256, device="cuda", layer_ids=[0, 1],
                               norm_jitter=0.0 if family == "qwen3" else 0.1, kv_bits=8)
    assert target.model.engine.kv_bits == 8
    prompt = np.random.default_rng(5).integers(1, cfg.vocab_size, 40).tolist()
    n_new = 30
    plan = _gpu_sequential_greedy(target, prompt, n_new)
    out, metrics = dtree_generate(target, ScriptedDrafter(target, prompt + plan), prompt, max_new_tokens=n_new,
                                  temperature=0.0, stop_token_ids=set(), layer_ids=[0, 1], speculative_tokens=BLOCK,
                                  tree_budget=12, verify_mode="parallel-greedy-argmax", tree_topk=4)
    gen = out[len(prompt):]
    assert len(gen) == n_new and max(metrics["acceptance_lengths"]) >= 5
    # teacher-forced through the same engine, one token at a time
    eng = target.model.engine
    cache = eng.new_cache()
    eng.prefill(cache, out[:len(prompt) - 1])
    for i, tok in enumerate(out[len(prompt) - 1:-1]):
        P = cache.offset
        eng.forward_only(cache, [tok], [P], [-1])
        st = eng.stream_handle()
        eng.launch_lm_head(st, want_logits=True)
        eng.launch_walk(st)
        eng.launch_compact(cache, st)
        eng.read_result()
        eng._keep_commit(cache, P, 1)
        row = eng.logits[0]
        assert float(row[gen[i]]) >= float(row.max()) - TOL * float(row.abs().max()), i


def test_8_bit_prefill_is_near_the_bf16_cache(gpu_device):
    """A whole prompt's logits, 8-bit against bf16 cache: quantisation moves a K or V
    row by at most amax / 254 per element, so by no more than a few percent of the
    logits' range; another kind of error (a wrong scale, page or head) is far larger."""
    cfg = tiny_qwen3()
    w = Qwen3Weights.random(cfg, seed=0, device=gpu_device, norm_jitter=0.1)
    toks = random_prefix(300, cfg.vocab_size, seed=4)
    logits = []
    for bits in (16, 8):
        eng = Qwen3TreeModel(cfg, w, max_past=364, kv_bits=bits).engine
        logits.append(eng.prefill_long(eng.new_cache(), toks)[0][0, 0])
    assert float((logits[0] - logits[1]).abs().max()) <= 5e-2 * float(logits[0].abs().max())


def test_caches_of_the_other_kind_are_refused(gpu_device):
    cfg = tiny_qwen3()
    w = Qwen3Weights.random(cfg, seed=0, device=gpu_device)
    eight = Qwen3TreeModel(cfg, w, max_past=100, kv_bits=8).engine
    full = Qwen3TreeModel(cfg, w, max_past=100).engine
    for eng, other in ((eight, full), (full, eight)):
        cache = other.new_cache()
        with pytest.raises(TypeError):
            eng.forward_only(cache, [1], [0], [-1])
        with pytest.raises(TypeError):
            eng.launch_compact(cache, eng.stream_handle())
    with pytest.raises(ValueError):
        Qwen3TreeModel(cfg, w, max_past=100, kv_bits=4)


@pytest.mark.parametrize("family", ["qwen3", "qwen35"])
def test_prefill_and_steps_refuse_the_other_kind(gpu_device, family):
    cfg, cls, wcls = ((tiny_qwen3(), Qwen3TreeModel, Qwen3Weights) if family == "qwen3" else
                      (tiny_qwen35(), Qwen35TreeModel, Qwen35Weights))
    w = wcls.random(cfg, seed=0, device=gpu_device)
    engines = [cls(cfg, w, max_past=256, kv_bits=bits).engine for bits in (8, 16)]
    for eng, other in (engines, engines[::-1]):
        cache = other.new_cache()
        with pytest.raises(TypeError):
            eng.prefill_long(cache, list(range(1, 129)))
        with pytest.raises(TypeError):
            eng.forward_only(cache, [1], [0], [-1])


def test_a_cache_of_several_sequences_is_refused(gpu_device):
    cfg = tiny_qwen3()
    eng = Qwen3TreeModel(cfg, Qwen3Weights.random(cfg, seed=0, device=gpu_device), max_past=100, kv_bits=8).engine
    cache = PagedKVCacheQ8(cfg.num_hidden_layers, cfg.num_key_value_heads, cfg.head_dim, 256, num_seqs=2,
                           device=gpu_device)
    for call in (lambda: eng.forward_only(cache, [1], [0], [-1]), lambda: eng.prefill_long(cache, list(range(1, 129))),
                 lambda: eng.launch_compact(cache, eng.stream_handle())):
        with pytest.raises(ValueError):
            call()


def test_first_step_from_a_captured_graph(gpu_device):
    """A graph captured before any eager step allocates nothing, and replays as the eager step."""
    cfg = tiny_qwen3()
    w = Qwen3Weights.random(cfg, seed=0, device=gpu_device)
    got = []
    for use_graph in (True, False):
        eng = Qwen3TreeModel(cfg, w, max_past=100, kv_bits=8).engine
        cache = eng.new_cache()
        res = [eng.verify(cache, [5, 6, 7], [0, 1, 2], [-1, 0, 1], use_graph=use_graph, commit=False)
               for _ in range(3)]
        got.append([(list(r.accepted), r.bonus_token) for r in res])
    assert got[0] == got[1]
