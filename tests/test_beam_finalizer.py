"""A decoder's finalizer, which may run at any point, waits for nothing and destroys
nothing: its captured steps go to the engine, which destroys them between launches."""
from types import SimpleNamespace

import torch

from dtree_hip import BeamDecoder


def _decoder(destroyed):
    d = BeamDecoder.__new__(BeamDecoder)
    lib = SimpleNamespace(dtree_graph_destroy=lambda g: destroyed.append(g.value))
    d.eng = SimpleNamespace(_dead_graphs=[], dev=None, lib=lib)
    d._graphs = {0: 11, 1: 12}
    return d


def test_finalizer_hands_the_graphs_over(monkeypatch):
    waits, destroyed = [], []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: waits.append(a))
    d = _decoder(destroyed)
    eng = d.eng
    del d
    assert not waits and not destroyed and sorted(eng._dead_graphs) == [11, 12]
    BeamDecoder.__new__(BeamDecoder)  # (one whose arguments were refused has nothing)


def test_release_destroys_at_once(monkeypatch):
    waits, destroyed = [], []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: waits.append(a))
    d = _decoder(destroyed)
    eng = d.eng
    d.release()
    assert len(waits) == 1 and sorted(destroyed) == [11, 12]
    del d
    assert eng._dead_graphs == [] and len(destroyed) == 2
