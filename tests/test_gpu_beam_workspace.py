"""Where dtree_beam_select keeps the maxima of every 32 logits: its second kernel reads
them 16 bytes at a time."""
import ctypes as C

import pytest
import torch

from dtree_hip import _native as N

from test_gpu_beam_select import Select, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("G,K", [(1, 1), (3, 1), (1, 2)])
def test_segment_maxima_are_aligned(gpu_device, G, K):
    """An odd number of blocks of 4096 logits, and an even one."""
    V = 4096
    x = rows(gpu_device, G * K, V, seed=51)
    s = Select(gpu_device, G, K, 2, V, x, [0.0] * (G * K))
    s.run()
    s.check()
    want = x.view(G * K, V // 32, 32).amax(-1).contiguous().cpu().numpy().tobytes()
    at = s.ws.cpu().numpy().tobytes().find(want)
    assert at >= 0 and at % 16 == 0


@pytest.mark.parametrize("vocab,beams", [(1, 1), (4097, 3), (8192, 1), (20000, 5)])
def test_size_is_a_multiple_of_16(gpu_device, vocab, beams):
    a = N.BeamArgs()
    a.type = N.T_F32; a.ld_logits = a.vocab = vocab; a.groups = 1; a.beams = beams; a.num_select = 1
    need = N.lib().dtree_beam_select_workspace_bytes(C.byref(a))
    assert need > 0 and need % 16 == 0
