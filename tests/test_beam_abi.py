"""Refusals of the selection, fork, copy and batch entries (nothing is launched),
and the oracle's own properties. CPU only."""
import ctypes as C

import numpy as np
import pytest

from dtree_hip import _native as N
from oracle import beam as ob


def record(cls, base, kw):
    r = cls()
    for k, v in {**base, **kw}.items():
        if isinstance(v, (list, tuple)):
            for i, x in enumerate(v):
                getattr(r, k)[i] = x
        else:
            setattr(r, k, v)
    return r


def refused(rc, word, code=N.E_ARG):
    assert rc == code
    msg = N.lib().dtree_last_error().decode()
    assert word in msg, msg


BEAM = dict(logits=4096, type=N.T_F32, ld_logits=1000, vocab=1000, groups=2, beams=4, num_select=4, scores=4096,
            eos_token=-1, pad_token=0, scores_out=8192, tokens_out=8192, parents_out=8192, workspace=4096,
            workspace_bytes=1 << 20)


@pytest.mark.parametrize("kw,word", [
    (dict(logits=None), "null"), (dict(scores_out=None), "null"), (dict(tokens_out=None), "null"),
    (dict(parents_out=None), "null"), (dict(type=2), "type"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 20) + 1, ld_logits=1 << 21), "vocab"), (dict(beams=0), "beams"), (dict(beams=65), "beams"),
    (dict(num_select=0), "num_select"), (dict(num_select=65), "num_select"), (dict(groups=0), "groups"),
    (dict(groups=-1), "groups"), (dict(groups=1 << 22), "groups"), (dict(ld_logits=999), "ld_logits"),
    (dict(logits=4098), "aligned"), (dict(logits=4097, type=N.T_BF16), "aligned"), (dict(eos_token=-2), "eos_token"),
    (dict(eos_token=1000), "eos_token"), (dict(pad_token=-1), "pad_token"), (dict(pad_token=1000), "pad_token"),
    (dict(length_penalty=float("nan")), "length_penalty"), (dict(length_penalty=float("inf")), "length_penalty"),
    (dict(length_penalty=17.0), "length_penalty"), (dict(workspace=None), "workspace"), (dict(workspace=4104), "workspace"),
    (dict(scores_out=4096, num_select=3), "num_select"), (dict(lengths=64, lengths_out=64, num_select=3), "num_select"),
    (dict(finished=64, finished_out=64, num_select=8), "num_select"),
])
def test_select_refusals(kw, word):
    a = record(N.BeamArgs, BEAM, kw)
    refused(N.lib().dtree_beam_select(C.byref(a), None), word)


def test_select_workspace():
    lib = N.lib()
    a = record(N.BeamArgs, BEAM, {})
    need = lib.dtree_beam_select_workspace_bytes(C.byref(a))
    assert need > 0 and need % 16 == 0
    a.workspace_bytes = need - 1
    refused(lib.dtree_beam_select(C.byref(a), None), "workspace", N.E_WORKSPACE)
    refused(lib.dtree_beam_select(None, None), "null")
    assert lib.dtree_beam_select_workspace_bytes(None) == 0
    assert lib.dtree_beam_select_workspace_bytes(C.byref(record(N.BeamArgs, BEAM, dict(beams=65)))) == 0


FORK = dict(refs=4096, num_pages=16, num_seqs=4, ld_tables=8, tables=1 << 16, tables_out=1 << 17, lengths=4096,
            lengths_out=8192, parents=4096, absent=-1)


@pytest.mark.parametrize("kw,word", [
    (dict(refs=None), "null"), (dict(tables=None), "null"), (dict(tables_out=None), "null"), (dict(lengths=None), "null"),
    (dict(lengths_out=None), "null"), (dict(num_seqs=0), "num_seqs"), (dict(num_seqs=1025), "num_seqs"),
    (dict(num_pages=0), "num_pages"), (dict(ld_tables=0), "ld_tables"), (dict(ld_tables=(1 << 22) + 1), "ld_tables"),
    (dict(num_seqs=1024, ld_tables=1 << 22), "entries"), (dict(rows=-1), "rows"), (dict(advance=-1), "rows"),
    (dict(rows=1), "copies"), (dict(absent=-2), "absent"), (dict(absent=16), "absent"), (dict(tables_out=1 << 16), "in place"),
    (dict(tables_out=(1 << 16) + 64), "overlap"), (dict(lengths_out=4100), "overlap"),
])
def test_fork_refusals(kw, word):
    refused(N.lib().dtree_pages_fork(C.byref(record(N.PagesFork, FORK, kw)), None), word)


COPY = dict(copies=4096, max_copies=4, num_pages=16, num_heads=2, layers=2, pools=[4096, 8192], block_bytes=[4096, 256])


@pytest.mark.parametrize("kw,word", [
    (dict(copies=None), "null"), (dict(max_copies=0), "max_copies"), (dict(max_copies=1025), "max_copies"),
    (dict(num_pages=0), "num_pages"), (dict(num_heads=0), "num_heads"), (dict(layers=0), "layers"),
    (dict(layers=1 << 16, num_heads=32), "2^20"), (dict(pools=[None, None]), "no pool"), (dict(pools=[4104]), "aligned"),
    (dict(block_bytes=[0]), "block_bytes"), (dict(block_bytes=[4096, 48]), "block_bytes"),
])
def test_copy_refusals(kw, word):
    refused(N.lib().dtree_pages_copy(C.byref(record(N.PagesCopy, COPY, kw)), None), word)


def test_null_records():
    lib = N.lib()
    refused(lib.dtree_pages_fork(None, None), "null")
    refused(lib.dtree_pages_copy(None, None), "null")
    refused(lib.dtree_gdn_layer_batch(None, None, 1, None), "null")


GDN = dict(rows_padded=32, num_k_heads=2, num_v_heads=4, head_k_dim=128, head_v_dim=128, conv_keep=3, proj=4096,
           ld_proj=2048, window=1 << 20, conv_w=4096, A_log=4096, dt_bias=4096, state=1 << 24, norm_w=4096, eps=1e-6,
           out=4096, out_layout=N.W_ROWMAJOR, ld_out=512, window_out=2 << 20, state_out=2 << 24)


@pytest.mark.parametrize("kw,seqs,word", [
    (dict(rows_padded=1 << 16, num_v_heads=128), 4, "2^23"), ({}, 0, "num_seqs"), ({}, 33, "num_seqs"), (dict(rows_padded=1 << 17), 4, "num_seqs"), (dict(num_k_heads=0), 4, "heads"),
    (dict(num_v_heads=5), 4, "heads"), (dict(num_v_heads=512), 4, "heads"), (dict(head_k_dim=64), 4, "dims"),
    (dict(head_v_dim=256), 4, "dims"), (dict(conv_keep=0), 4, "conv_keep"), (dict(conv_keep=8), 4, "conv_keep"),
    (dict(ld_proj=1540), 4, "ld_proj"), (dict(ld_proj=2049), 4, "ld_proj"), (dict(proj=4100), 4, "aligned"),
    (dict(state=4100), 4, "aligned"), (dict(window_out=(2 << 20) + 8), 4, "aligned"), (dict(out=4100), 4, "aligned"),
    (dict(ld_out=510), 4, "out layout"), (dict(out_layout=N.W_Q4G64), 4, "out layout"),
    (dict(out_layout=N.W_TILED, rows_padded=33), 4, "out layout"), (dict(state_out=1 << 24), 4, "own"),
    (dict(window_out=(1 << 20) + 1024), 4, "own"),
    *[({k: None}, 4, "null") for k in ("proj", "window", "conv_w", "A_log", "dt_bias", "state", "norm_w", "out", "window_out",
                                      "state_out")],
])
def test_batch_refusals(kw, seqs, word):
    refused(N.lib().dtree_gdn_layer_batch(C.byref(record(N.GdnArgs, GDN, kw)), None, seqs, None), word)


def test_oracle_selection_by_hand():
    x = np.log(np.array([[0.5, 0.3, 0.2], [0.6, 0.3, 0.1]]))
    o = ob.select(x, np.log([0.4, 0.6]), [1, 1], [0, 0], 1, 2, 4, 0, 0, 0.0)
    assert o["tokens"].tolist() == [[0, 0, 1, 1]] and o["parents"].tolist() == [[1, 0, 1, 0]]
    assert np.allclose(np.exp(o["scores"]), [[0.36, 0.2, 0.18, 0.12]])
    assert o["finished"].tolist() == [[1, 1, 0, 0]] and o["sources"].tolist() == [[-1, -1, 1, 0]]
    o = ob.select(x, np.log([0.9, 0.6]), [3, 1], [1, 0], 1, 2, 2, -1, 2, 1.0)  # a finished beam, ranked by its mean
    assert o["tokens"].tolist() == [[2, 0]] and o["lengths"].tolist() == [[3, 2]] and o["finished"].tolist() == [[1, 0]]


def test_oracle_fork_by_hand():
    refs, tables, lengths, copies, missing = ob.fork([1, 1, 0, 0, 0, 0], [[0, 1, -1], [-1, -1, -1], [-1, -1, -1]],
                                                     [100, 0, 0], [0, 0, -1], 0, 1)
    assert tables.tolist() == [[0, 2, -1], [0, 1, -1], [3, -1, -1]] and copies == [(1, 2, 36)]
    assert refs.tolist() == [2, 1, 1, 1, 0, 0] and lengths.tolist() == [100, 100, 0] and missing == 0


def test_kernels_use_no_scratch():
    from test_kernel_scratch import _code_objects, _kernels

    if not N.LIB_PATH.exists():
        pytest.skip("library not built")
    names = ("beam_scan", "beam_pick", "pages_share", "pages_take", "pages_copy", "gdn_batch")
    mine = [k for o in _code_objects(N.LIB_PATH.read_bytes()) for k in _kernels(o) if any(n in k[".name"] for n in names)]
    assert len(mine) == 4 + 1 + 2 + 1 + 7
    assert [k[".name"] for k in mine if k[".private_segment_fixed_size"]] == []
