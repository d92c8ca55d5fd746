"""dtree_beam_select where whole chunks of a row, or whole rows, lie far from zero: tokens
masked with a large finite number, and rows whose logits have any magnitude. Against the
selection in 64 bits, within test_gpu_beam_select's tolerance: its derivation counts
|x - m| 2^-23 a term, whichever way the exponent is formed."""
import numpy as np
import pytest
import torch

from test_gpu_beam_select import Select, rows, scores_of

pytestmark = pytest.mark.gpu

CHUNK = 4096  # logits whose sum is taken together


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [-1e5, -1048576.0, -3e6, -1e9, -5e9, -1e10, -1e15, -1e20, -9e29, -1.1e30, -3e38])
def test_chunks_masked_by_a_finite_number(gpu_device, value, dtype):
    """Some beams of a group have a chunk of masked tokens alone: its weight is 0 beside the
    rest of the row, and the beam's sums are what they are without it."""
    G, K, M, V = 2, 4, 10, 3 * CHUNK + 100
    x = rows(gpu_device, G * K, V, dtype, seed=41)
    x[1, CHUNK:2 * CHUNK] = value
    x[2, 3 * CHUNK:] = value
    x[3, :3 * CHUNK] = value
    x[6, :CHUNK] = value
    x[6, CHUNK:2 * CHUNK] = value * 0.5
    s = Select(gpu_device, G, K, M, V, x, scores_of(G * K, 42))
    s.run()
    s.check()
    assert {1, 2, 3} & set(s.out["parents"][0].tolist())  # (masked rows take part)


@pytest.mark.parametrize("centre", [2.0 ** 19, 2.0 ** 20, 2.0 ** 21, 3e6, 1e8, 5e9, 1e10, 1e20, 9e29])
@pytest.mark.parametrize("sign", [1, -1])
def test_rows_around_a_large_number(gpu_device, centre, sign):
    """Rows of a few fp32 steps around the number, beside ordinary ones: the differences
    decide, which are exact."""
    G, K, M, V = 1, 6, 24, 2 * CHUNK + 77
    x = rows(gpu_device, G * K, V, seed=43)
    step = float(np.spacing(np.float32(centre)))
    far = torch.round(x[:3] * (1.0 if step > 1 else 1.0 / step)) * step
    x[:3] = sign * centre + far
    x[2, CHUNK:] -= 64 * step  # (chunks of unlike maxima)
    s = Select(gpu_device, G, K, M, V, x, [-2.0, -1.0, 0.0, -2.0, -1.0, 0.0])
    s.run()
    s.check()
    b = Select(gpu_device, G, K, M, V, x.bfloat16(), [-2.0, -1.0, 0.0, -2.0, -1.0, 0.0])
    b.run()
    b.check()
