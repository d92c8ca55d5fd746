"""Where a pool's sequences may be written: behind start(). CPU only (nothing is launched;
forks are in test_gpu_pool_room.py)."""
import pytest
import torch

from dtree_hip import PagedKVCache, PagedKVPool
from dtree_hip.cache import check_room


def _pool(kv_bits):
    return PagedKVPool(2, 2, 64, 256, 3, kv_bits=kv_bits, device="cpu")


@pytest.mark.parametrize("kv_bits", [16, 8])
def test_a_started_sequence_is_written_on_its_pages_alone(kv_bits):
    pool = _pool(kv_bits)
    early = pool.sequence(0)
    rows = torch.ones(1, 2, 64)
    with pytest.raises(ValueError, match="no room"):
        early.write_logical(0, rows, rows)
    pool.start([100, 1])
    before = [t.clone() for t in pool.pools]
    assert [pool.sequence(i).room for i in range(3)] == [(0, 128), (0, 64), (0, 0)]
    for i, at in ((0, 128), (0, 250), (1, 64), (2, 0)):
        with pytest.raises(ValueError, match="room"):
            pool.sequence(i).write_logical(0, rows, rows, start=at)
    with pytest.raises(ValueError, match="room"):
        pool.sequence(0).write_logical(0, rows.expand(2, 2, 64), rows.expand(2, 2, 64), start=127)
    assert all(torch.equal(a, b) for a, b in zip(pool.pools, before))
    pool.sequence(0).write_logical(1, rows, rows, start=127)
    assert torch.equal(early.logical_keys(1, 128)[127].float(), rows[0])
    pool.start([])
    with pytest.raises(ValueError, match="no room"):
        early.write_logical(0, rows, rows)


def test_other_caches_are_their_own_throughout():
    c = PagedKVCache(1, 2, 64, 128, device="cpu")
    check_room(c, 0, 128)
    check_room(object(), 5, 5)  # (any class with an engine's fields)
    c.write_logical(0, torch.ones(128, 2, 64), torch.ones(128, 2, 64))


def test_a_length_without_pages_is_not_forked():
    pool = _pool(16)
    pool.start([100])
    pool.sequence(0).offset = 129
    with pytest.raises(ValueError, match="pages"):
        pool.fork(None, rows=1)
