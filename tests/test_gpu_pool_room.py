"""Steps that a pool's sequence has no room for are refused by the engines, and leave every
sequence's rows as they are."""
import numpy as np
import pytest
import torch

from dtree_hip import BeamDecoder
from dtree_hip.adapters import load_target_model
from dtree_hip.config import tiny_qwen3
from dtree_hip.synthetic import make_tree, random_prefix

pytestmark = pytest.mark.gpu


def _target(kv_bits):
    return load_target_model(tiny_qwen3(), seed=0, max_past=300, norm_jitter=0.1, kv_bits=kv_bits)


def _tree(eng, P, seed=1, budget=4):
    tree = make_tree(budget, eng.cfg.vocab_size, seed=seed)
    return tree.tokens, tree.positions(P), tree.parents


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("kv_bits", [16, 8])
def test_steps_without_room(gpu_device, kv_bits, use_graph):
    target = _target(kv_bits)
    eng = target.model.engine
    pool = eng.new_pool(3, num_pages=20)
    prompt = random_prefix(150, eng.cfg.vocab_size, seed=3)
    a, b, c = (pool.sequence(i) for i in range(3))
    with pytest.raises(ValueError, match="no room"):  # not started
        eng.prefill(a, prompt)
    pool.start([120])
    with pytest.raises(ValueError, match="room"):  # started for fewer
        eng.prefill(a, prompt)
    pool.start([150])
    eng.prefill(a, prompt)

    def verify(cache):
        return eng.verify(cache, *_tree(eng, cache.offset), use_graph=use_graph, commit=False)

    def logits():
        return torch.randn(4, eng.cfg.vocab_size, device=gpu_device)

    pool.fork([0, 0, 0])  # the last page is shared, there is none behind it
    rows = [t.clone() for t in pool.pools]
    for seq in (a, b, c):
        with pytest.raises(ValueError, match="no room"):
            verify(seq)
        with pytest.raises(ValueError, match="no room"):
            eng.verify_from_logits(seq, logits(), 4, None, 1, use_graph=use_graph)
        with pytest.raises(ValueError, match="no room"):
            eng.prefill(seq, prompt[:3])
        with pytest.raises(ValueError, match="no room"):
            target.forward_with_hidden_states(torch.tensor([prompt[:128]]), seq, [])
        tokens, positions, parents = _tree(eng, 150)
        L = len(tokens)
        mask = np.zeros((L, 150 + L), bool)
        mask[:, :150] = True
        for i in range(L):
            j = i
            while j >= 0:
                mask[i, 150 + j] = True
                j = parents[j]
        with pytest.raises(ValueError, match="no room"):
            target.forward_tree_with_hidden_states(tokens, seq, [], parents, positions, mask)
        assert seq.offset == 150
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(pool.pools, rows))

    pool.fork(None, rows=5)
    assert [s.room for s in (a, b, c)] == [(128, 192)] * 3
    want = eng.new_cache()
    eng.prefill(want, prompt)
    r, w = verify(b), verify(want)
    assert (r.accepted, r.posterior) == (w.accepted, w.posterior)
    eng.verify_from_logits(b, logits(), 31, None, 1, use_graph=use_graph, commit=False)  # 150 + 32 <= 192
    b.offset = 161
    with pytest.raises(ValueError, match="128 .. 191"):
        eng.verify_from_logits(b, logits(), 31, None, 1, use_graph=use_graph, commit=False)
    b.offset = 127  # taken back into a page that the others hold
    with pytest.raises(ValueError, match="128 .. 191"):
        verify(b)


@pytest.mark.parametrize("kv_bits", [16, 8])
def test_a_tree_committed_behind_a_fork(gpu_device, kv_bits):
    """A forward's rows, forked before they are compacted, are the others' too."""
    target = _target(kv_bits)
    eng = target.model.engine
    pool = eng.new_pool(2, num_pages=12)
    pool.start([60])
    a = pool.sequence(0)
    eng.prefill(a, random_prefix(60, eng.cfg.vocab_size, seed=4))
    pool.fork([0, -1], rows=8)
    tokens, positions, parents = [5, 6, 7], [60, 61, 61], [-1, 0, 0]
    mask = np.ones((3, 63), bool)
    mask[:, 60:] = np.array([[1, 0, 0], [1, 1, 0], [1, 0, 1]], bool)
    target.forward_tree_with_hidden_states(tokens, a, [], parents, positions, mask)
    assert a.offset == 63
    pool.fork([0, 0])
    with pytest.raises(ValueError, match="no room"):
        target.compact_kv_caches(a, 60, [0, 2])
    pool.fork(None, rows=1)  # (the first copies its last page, the other keeps it)
    target.compact_kv_caches(a, 60, [0, 2])
    assert a.offset == 62
    for t in (a.logical_keys(0, 63), a.logical_values(0, 63)):
        assert not torch.equal(t[61], t[60])
    b = pool.sequence(1)
    assert torch.equal(a.logical_keys(0, 62)[61], b.logical_keys(0, 63)[62])
    assert not torch.equal(b.logical_keys(0, 63)[61], b.logical_keys(0, 63)[62])


@pytest.mark.parametrize("kv_bits", [16, 8])
def test_pages_used_up_leave_no_room(gpu_device, kv_bits):
    target = _target(kv_bits)
    eng = target.model.engine
    pool = eng.new_pool(2, num_pages=4)
    pool.start([130])
    a = pool.sequence(0)
    eng.prefill(a, random_prefix(130, eng.cfg.vocab_size, seed=5))
    with pytest.raises(RuntimeError, match="used up"):
        pool.fork([0, 0], rows=100)
    for s in (a, pool.sequence(1)):
        with pytest.raises(ValueError, match="no room"):
            eng.verify(s, *_tree(eng, s.offset), use_graph=False)
    with pytest.raises(ValueError, match="pages"):
        pool.fork([0, 0], rows=1)
    pool.start([4])
    eng.prefill(a, [1, 2, 3, 4])


def test_a_decoders_pages_are_its_own(gpu_device):
    """Behind the prompts the device forks a decoder's pool: the host has no room in it."""
    target = _target(8)
    d = BeamDecoder(target, [[3, 4, 5]], 3, 6)
    d.start()
    for i in range(3):
        with pytest.raises(ValueError, match="no room"):
            target.model.engine.prefill(d.cache.pool.sequence(i), [1, 2])
    d.step()
