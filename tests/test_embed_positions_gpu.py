"""The gradient of the position rows: sums over the sequences, eight of them at a time by themselves in pairs, so that B of
them pass through at most 3 + B / 8 + B mod 8 roundings, and one for what is there."""
import numpy as np
import pytest

import test_embed_sorted_gpu as sorted_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("B,T,C", [(64, 5, 8), (64, 5, 7), (64, 40, 8), (61, 40, 7), (257, 6, 4), (7, 3, 4), (8, 200, 1)])
def test_one_large_row_and_many_small_ones(rt, B, T, C, accumulate):
    """2^24 and ones: a chain would drop every one of them."""
    g = np.ones((B, T, C), np.float32)
    g[0] = 2.0 ** 24
    before = np.ones((T, C), np.float32)
    _, dP = sorted_gpu.gather(rt, g, np.zeros((B, T), np.float32), 1.0, np.zeros((3, C), np.float32), before, accumulate)
    want = 2.0 ** 24 + B - 1 + accumulate
    tol = (3 + B // 8 + B % 8 + accumulate) * sorted_gpu.U * want
    sorted_gpu.close("dP", dP, np.full((T, C), want), tol)
