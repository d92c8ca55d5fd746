"""Rules of the 8-bit cache that ordinary random rows do not meet."""
import ctypes as C

import pytest
import torch

from dtree_hip import _native as N
from dtree_hip.cache import PagedKVCacheQ8, _block_index_q8

from gpu_util import stream
from test_gpu_kv_q8 import PAIR, Batch, check, i32
from test_kv_q8_rules import SCALES, tie_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_takes_ties_to_even_whatever_the_scale(gpu_device, d):
    """x / scale halfway between two integers, the scale no power of two: exact
    in fp32, so the stored integer is determined. K without norm or rotation."""
    dev = gpu_device
    n, hkv = len(SCALES), 2
    x, q = zip(*(tie_rows(d, SCALES, seed) for seed in range(2 * hkv)))
    rows = torch.stack(x, 1).reshape(n, 2 * hkv * d).to(dev).contiguous()  # [k heads | v heads]
    c = PagedKVCacheQ8(1, hkv, d, n + 3, device=dev)
    past, count = i32([3], dev), i32([n], dev)
    rec = c.record(0, past, count, 3, n, n)
    N.check(N.lib().dtree_kv_q8_append(C.byref(rec), rows.data_ptr(), rows.data_ptr() + 4 * hkv * d, N.T_F32, 2 * hkv * d,
                                       2 * hkv * d, None, 0.0, None, None, 0, stream()), "append")
    slot = torch.arange(3, 3 + n)
    for which, pages, scales, j in (("k", c.k_pages, c.k_scales, 0), ("v", c.v_pages, c.v_scales, hkv)):
        at = _block_index_q8(d, which)[slot].to(dev)
        for h in range(hkv):
            assert torch.equal(scales[0, 0, h, slot].cpu().double(), torch.tensor(SCALES, dtype=torch.float64))
            assert torch.equal(pages[0, 0, h][at].cpu().long(), q[j + h]), (which, h)


@pytest.mark.parametrize("heads", ["128", "256g", "64", "mqa"])
@pytest.mark.parametrize("past,rows,workspace", [([100], [1], True), ([1500], [1], True), ([100], [60], True),
                                                 ([2500], [70], True), ([2500], [70], False)])
@pytest.mark.parametrize("size,typ", [(1e9, torch.float32), (1e30, torch.float32), (1e12, torch.bfloat16)])
def test_a_query_far_larger_than_its_neighbours(gpu_device, heads, past, rows, workspace, size, typ):
    """One (row, head) beyond the others by more than fp16's exponents span: each
    keeps its own bits, without a q_norm that would bring them together."""
    b = Batch(gpu_device, heads, past, rows, typ=typ, seed=41, norm=False)
    b.append()
    at = (2 * b.d if b.gated else b.d)
    b.qkv[rows[0] // 2, at:at + b.d] *= size  # head 1
    if rows[0] > 1:  # beside them a query of zeros and one that is not finite
        b.qkv[3, :b.d] = 0.0
        b.qkv[5, 0] = float("inf")
    want, tol = b.reference()
    check(b.attend(pair=True, workspace=workspace), want, tol, PAIR)
