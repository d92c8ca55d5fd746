"""The 8-bit cache's rounding rule and the bounds its records are held to, on
the host. CPU only."""
import ctypes as C

import pytest
import torch

from dtree_hip import _native as N
from dtree_hip import tiny_qwen35
from dtree_hip.cache import PagedKVCache, PagedKVCacheQ8, Qwen35Cache, quantise_q8

from test_kv_q8_abi import attn, cache, refused


def tie_rows(dim, scales, seed=0):
    """Rows whose scale is exactly s (max |x| = 127 s) and whose other elements
    lie halfway between two integers: ([rows, dim] fp32, [rows, dim] integers)."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(-126, 126, (len(scales), dim), generator=g)  # x / s = k + 1 / 2
    s = torch.tensor(scales, dtype=torch.float64)[:, None]
    x = (2 * k + 1).double() * (s / 2)
    q = torch.where(k % 2 == 0, k, k + 1)  # to even
    x[:, 5], q[:, 5] = 127 * s[:, 0], 127
    assert torch.equal(x.float().double(), x)  # 24 bits hold them all
    return x.float(), q


SCALES = [49, 3, 7, 11, 13, 41, 107, 257, 1021, 8191, 32771, 65535, 49 * 2.0 ** -30, 41 * 2.0 ** 60, 0.75, 1.0, 64.0]


def test_ties_go_to_even_whatever_the_scale():
    x, want = tie_rows(128, SCALES)
    q, scale = quantise_q8(x)
    assert torch.equal(scale.double(), torch.tensor(SCALES, dtype=torch.float64))
    assert torch.equal(q.long(), want)


def test_ties_of_one_row_worked_by_hand():
    q, scale = quantise_q8(torch.tensor([6223.0, 73.5, 171.5, -122.5]))
    assert float(scale) == 49.0 and q.tolist() == [127, 2, 4, -2]  # 1.5, 3.5, -2.5


@pytest.mark.parametrize("bits", [0, 4, 32, None, "8"])
def test_hybrid_cache_refuses_other_widths(bits):
    with pytest.raises(ValueError):
        Qwen35Cache(tiny_qwen35(), 64, device="cpu", kv_bits=bits)


def test_hybrid_cache_of_either_width():
    assert type(Qwen35Cache(tiny_qwen35(), 64, device="cpu").kv) is PagedKVCache
    assert type(Qwen35Cache(tiny_qwen35(), 64, device="cpu", kv_bits=8).kv) is PagedKVCacheQ8


# Work items of a launch are counted in 32 bits: 2^24 workgroups of 256 threads are one too many.
WIDE = dict(num_kv_heads=256, num_seqs=65536, max_rows=1, total_rows=65536, max_past_length=0, ld_page_table=1)


def test_launches_of_2_to_the_32_threads_are_refused():
    lib = N.lib()
    r = cache(**WIDE)
    width = 256 * 128
    refused(lib.dtree_kv_q8_append(C.byref(r), 4096, 4096, N.T_F32, width, width, None, 0.0, None, None, 0, None),
            "too large")
    refused(lib.dtree_kv_q8_read(C.byref(r), 4096, 4096, N.T_F32, width, width, None), "too large")
    a = attn(num_heads=256, ld_q=width, ld_out=width)
    refused(lib.dtree_attention_q8(C.byref(r), C.byref(a), None), "too large")
