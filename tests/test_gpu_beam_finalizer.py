"""A decoder that dies during another capture."""
import ctypes as C
import gc

import pytest
import torch

from dtree_hip import BeamDecoder, _native as N
from dtree_hip.adapters import load_target_model
from dtree_hip.config import tiny_qwen3

pytestmark = pytest.mark.gpu


def test_a_decoder_dies_during_a_capture(gpu_device):
    target = load_target_model(tiny_qwen3(), seed=0, max_past=200, norm_jitter=0.1, kv_bits=8)
    eng = target.model.engine

    def decoder():
        d = BeamDecoder(target, [[3, 4, 5]], 3, 8)
        d.start()
        return d

    d, other = decoder(), decoder()
    for _ in range(4):
        d.step()
    n = len(d._graphs)
    assert n >= 2 and not eng._dead_graphs
    gc.collect()  # (whatever else is garbage, other tests' engines among it, goes before the capture)
    torch.cuda.synchronize()
    lib, side = N.lib(), torch.cuda.Stream()
    N.check(lib.dtree_graph_begin(side.cuda_stream), "begin")
    del d
    gc.collect()
    N.check(lib.dtree_rope_table(eng.desc.data_ptr(), eng.MP, eng.cfg.head_dim, eng.cfg.rope_theta, eng.rope_cos.data_ptr(),
                                 eng.rope_sin.data_ptr(), side.cuda_stream), "rope table")
    ex = C.c_void_p()
    N.check(lib.dtree_graph_end(side.cuda_stream, C.byref(ex)), "end")
    assert len(eng._dead_graphs) == n
    N.check(lib.dtree_graph_launch(ex, side.cuda_stream), "launch")
    torch.cuda.synchronize()
    lib.dtree_graph_destroy(ex)
    for _ in range(3):
        other.step()
    assert not eng._dead_graphs  # destroyed before the other's capture
    ref = decoder()
    ref.use_graph = False
    for _ in range(3):
        ref.step()
    assert [h.tokens for h in other.hypotheses()[0]] == [h.tokens for h in ref.hypotheses()[0]]
