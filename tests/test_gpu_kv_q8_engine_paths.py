"""What an engine takes, refuses and allocates beside the ordinary step, with
either kind of KV cache."""
import pytest
import torch

from dtree_hip import Qwen3TreeModel, Qwen3Weights, Qwen35TreeModel, Qwen35Weights, tiny_qwen3, tiny_qwen35
from dtree_hip.cache import PagedKVCache
from dtree_hip.synthetic import random_prefix

pytestmark = pytest.mark.gpu


def _engine(dev, family, kv_bits, **kw):
    cfg, model, weights = ((tiny_qwen3(), Qwen3TreeModel, Qwen3Weights) if family == "qwen3" else
                           (tiny_qwen35(), Qwen35TreeModel, Qwen35Weights))
    return model(cfg, weights.random(cfg, seed=0, device=dev, norm_jitter=0.1), kv_bits=kv_bits, **kw).engine


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
