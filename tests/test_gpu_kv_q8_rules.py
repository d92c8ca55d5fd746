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


@pytest.mark.parametrize("heads", ["128", "256g", "64"])
@pytest.mark.parametrize("rows", [1, 60])
def test_a_query_near_the_end_of_fp32(gpu_device, heads, rows):
    """Its logits are finite, its products with the cached integers are not: those are
    larger by 127 / max |k|. Beside ordinary queries, and all of them so."""
    for all_of_them in (False, True):
        b = Batch(gpu_device, heads, [300], [rows], seed=42, norm=False)
        b.append()
        for h in range(b.hq if all_of_them else 1):
            at = ((h + 1) % b.hq) * (2 * b.d if b.gated else b.d)
            b.qkv[(slice(None) if all_of_them else rows // 2), at:at + b.d] *= 2e37
        want, tol = b.reference()
        check(b.attend(pair=True), want, tol, PAIR, all_of_them)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_whose_scale_is_subnormal(gpu_device, d):
    """Multiples of fp32's smallest number, ties among them."""
    dev, unit = gpu_device, 2.0 ** -149
    scales = [2 * unit, 6 * unit, 98 * unit, 65534 * unit]
    x, q = tie_rows(d, scales, seed=9)
    rows = torch.cat([x, x], 1).to(dev).contiguous()
    c = PagedKVCacheQ8(1, 1, d, len(scales), device=dev)
    past, count = i32([0], dev), i32([len(scales)], dev)
    rec = c.record(0, past, count, 0, len(scales), len(scales))
    N.check(N.lib().dtree_kv_q8_append(C.byref(rec), rows.data_ptr(), rows.data_ptr() + 4 * d, N.T_F32, 2 * d, 2 * d, None,
                                       0.0, None, None, 0, stream()), "append")
    at = [_block_index_q8(d, which)[:len(scales)].to(dev) for which in "kv"]
    for pages, s, i in ((c.k_pages, c.k_scales, at[0]), (c.v_pages, c.v_scales, at[1])):
        assert torch.equal(s[0, 0, 0, :len(scales)].cpu().double(), torch.tensor(scales, dtype=torch.float64))
        assert torch.equal(pages[0, 0, 0][i].cpu().long(), q)
    k = torch.zeros(len(scales), d, device=dev)
    N.check(N.lib().dtree_kv_q8_read(C.byref(rec), k.data_ptr(), None, N.T_F32, d, 0, stream()), "read")
    assert torch.equal(k.cpu().double(), q.double() * torch.tensor(scales, dtype=torch.float64)[:, None])
