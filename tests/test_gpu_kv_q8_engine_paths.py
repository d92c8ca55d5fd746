"""What an engine takes, refuses and allocates beside the ordinary step, with
either kind of KV cache."""
import pytest
import torch

from dtree_hip import Qwen3TreeModel, Qwen3Weights, Qwen35TreeModel, Qwen35Weights, tiny_qwen3, tiny_qwen35
from dtree_hip.cache import PagedKVCache
from dtree_hip.synthetic import random_prefix

pytestmark = pytest.mark.gpu
TOL = 2e-2  # of the row maximum, as the engines' other tests grant


def _engine(dev, family, kv_bits, **kw):
    cfg, model, weights = ((tiny_qwen3(), Qwen3TreeModel, Qwen3Weights) if family == "qwen3" else
                           (tiny_qwen35(), Qwen35TreeModel, Qwen35Weights))
    return model(cfg, weights.random(cfg, seed=0, device=dev, norm_jitter=0.1), kv_bits=kv_bits, **kw).engine


class OwnCache:
    """A caller's own cache: what the bf16 engines read of one, and no more."""
    k_ptr, v_ptr, layer_stride = PagedKVCache.k_ptr, PagedKVCache.v_ptr, PagedKVCache.layer_stride

    def __init__(self, c, fields):
        for f in ("k_pages", "v_pages", "page_table", "n_pages", "kv_heads", "head_dim", "capacity", "offset", *fields):
            setattr(self, f, getattr(c, f))


@pytest.mark.parametrize("family", ["qwen3", "qwen35"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_a_bf16_engine_takes_a_cache_of_another_class(gpu_device, family, use_graph):
    """Prefill, step and compaction on it give what they give on PagedKVCache."""
    got = []
    for own in (False, True):
        eng = _engine(gpu_device, family, 16, max_past=300)
        cache = eng.new_cache()
        if own and family == "qwen3":
            cache = OwnCache(cache, ())
        elif own:
            cache.kv = OwnCache(cache.kv, ("layers",))
        eng.prefill_long(cache, random_prefix(150, eng.cfg.vocab_size, seed=3))
        P = cache.offset
        res = [eng.verify(cache, [5, 6, 7, 8], [P, P + 1, P + 1, P + 2], [-1, 0, 0, 2], use_graph=use_graph)
               for _ in range(2)]
        eng.launch_compact(cache, eng.stream_handle())
        kv = cache if family == "qwen3" else cache.kv
        got.append(([(r.accepted, r.bonus_token, r.posterior) for r in res], cache.offset, kv.k_pages, kv.v_pages))
    assert got[0][:2] == got[1][:2]
    assert torch.equal(got[0][2], got[1][2]) and torch.equal(got[0][3], got[1][3])


def test_a_step_moves_its_own_layers_rows_alone(gpu_device):
    """A cache with more layers than the model: compaction leaves the others as they are."""
    eng = _engine(gpu_device, "qwen3", 16, max_past=100)
    c = eng.cfg
    cache = PagedKVCache(c.num_hidden_layers + 1, c.num_key_value_heads, c.head_dim, 100 + eng.max_nodes,
                         device=gpu_device)
    cache.k_pages[-1].normal_()
    cache.v_pages[-1].normal_()
    k, v = cache.k_pages[-1].clone(), cache.v_pages[-1].clone()
    eng.set_step([5, 6, 7, 8], [0, 1, 1, 2], [-1, 0, 0, 2], 0, accepted=[0, 2, 3])
    eng.launch_compact(cache, eng.stream_handle(), select_hidden=False)
    torch.cuda.synchronize()
    assert torch.equal(cache.k_pages[-1], k) and torch.equal(cache.v_pages[-1], v)


@pytest.mark.parametrize("family", ["qwen3", "qwen35"])
def test_attention_without_a_cache_write_is_refused_in_8_bits(gpu_device, family):
    """The 8-bit attention reads a step's own rows from the cache."""
    eng = _engine(gpu_device, family, 8, max_past=100)
    cache = eng.new_cache()
    kv = cache if family == "qwen3" else cache.kv
    li = eng.cfg.num_hidden_layers - 1
    eng.set_step([5, 6], [0, 1], [-1, 0], 0)
    with pytest.raises(NotImplementedError):
        eng._attention(li, cache, eng.stream_handle(), write_cache=False)
    torch.cuda.synchronize()
    assert not kv.k_pages.any() and not kv.k_scales.any()


@pytest.mark.parametrize("family", ["qwen3", "qwen35"])
def test_a_prompt_allocates_its_8_bit_workspace_before_its_first_row(gpu_device, monkeypatch, family):
    """Segments over a growing prefix want more of it: had before the first of them."""
    eng = _engine(gpu_device, family, 8, max_past=1400)
    eng.PREFILL_SEGMENT = 128
    toks = random_prefix(1300, eng.cfg.vocab_size, seed=5)
    empty, attention, inside = torch.empty, eng._prefill_attention_q8, [False]

    def guarded(*a, **kw):
        if inside[0]:
            raise torch.cuda.OutOfMemoryError("no room")
        return empty(*a, **kw)

    def layer(*a, **kw):
        inside[0] = True
        try:
            return attention(*a, **kw)
        finally:
            inside[0] = False

    monkeypatch.setattr(torch, "empty", guarded)
    monkeypatch.setattr(eng, "_prefill_attention_q8", layer)
    cache = eng.new_cache()
    eng.prefill_long(cache, toks)
    torch.cuda.synchronize()
    assert cache.offset == 1300 and eng._pf["q8_ws"].numel() > 16


@pytest.mark.parametrize("family", ["qwen3", "qwen35"])
def test_a_prompt_runs_without_room_for_its_8_bit_workspace(gpu_device, monkeypatch, family):
    """Fewer key ranges, the same answer."""
    logits = []
    for full in (False, True):
        eng = _engine(gpu_device, family, 8, max_past=1400)
        toks = random_prefix(1300, eng.cfg.vocab_size, seed=5)
        cache = eng.new_cache()
        eng.prefill_long(cache, toks[:1100])
        eng._pf = None
        empty = torch.empty

        def short(*a, **kw):
            if kw.get("dtype") == torch.uint8:
                raise torch.cuda.OutOfMemoryError("no room")
            return empty(*a, **kw)

        with monkeypatch.context() as m:
            if full:
                m.setattr(torch, "empty", short)
            logits.append(eng.prefill_long(cache, toks[1100:])[0][0, 0].clone())
        assert cache.offset == 1300 and (eng._pf["q8_ws"] is None) == full
    assert float((logits[0] - logits[1]).abs().max()) <= TOL * float(logits[0].abs().max())


@pytest.mark.parametrize("family", ["qwen3", "qwen35"])
def test_an_8_bit_engine_holds_no_bf16_attention_workspace(gpu_device, family):
    eng = _engine(gpu_device, family, 8, max_past=300)
    assert eng.attn_ws is None
    cache = eng.new_cache()
    eng.prefill_long(cache, random_prefix(140, eng.cfg.vocab_size, seed=6))
    assert "attn_ws" not in eng._pf
    eng.verify(cache, [5, 6], [140, 141], [-1, 0])
    assert _engine(gpu_device, family, 16, max_past=300).attn_ws.numel() > 0


@pytest.mark.parametrize("family", ["qwen3", "qwen35"])
@pytest.mark.parametrize("kv_bits", [8, 16])
def test_a_prompt_in_segments_of_any_length(gpu_device, family, kv_bits):
    """Buffers that grow between a prompt's segments: the same logits."""
    logits = []
    for segment in (1024, 200):
        eng = _engine(gpu_device, family, kv_bits, max_past=700)
        eng.PREFILL_SEGMENT = segment
        cache = eng.new_cache()
        logits.append(eng.prefill_long(cache, random_prefix(600, eng.cfg.vocab_size, seed=8))[0][0, 0].clone())
        assert cache.offset == 600
    assert float((logits[0] - logits[1]).abs().max()) <= TOL * float(logits[0].abs().max())
