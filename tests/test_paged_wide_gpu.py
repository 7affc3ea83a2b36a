"""Attention over pages where enough workgroups take many rows each that the waves of fp32 pages hold two groups of 16
rows (384 workgroups, csrc/paged_attn_wide.hip): every head size's tile, whole and ragged rows, cut and uncut keys.

Tolerances: those of test_paged_gpu.py.  They are checked for every row.
"""
import ctypes

import numpy as np
import pytest
import torch

import gptc
from test_paged import schedule
from test_paged_gpu import U, Pool

pytestmark = pytest.mark.gpu

TWO_GROUPS = 384  # workgroups from which a wave takes two groups


def attention(q, kv, past):
    """test_paged_gpu.attention, a head at a time: q (n, H, D); y, and the bound on its error."""
    k, v = kv
    n, H, D = q.shape
    y, bound = np.zeros((n, H, D)), np.zeros((n, H, 1))
    hidden = np.arange(past + n) > past + np.arange(n)[:, None]
    for h in range(H):
        kk, vv = k[:, h * k.shape[1] // H], v[:, h * k.shape[1] // H]
        t = np.where(hidden, -np.inf, q[:, h] @ kk.T / np.sqrt(D))
        p = np.exp(t - t.max(1, keepdims=True))
        y[:, h] = p @ vv / p.sum(1, keepdims=True)
        dt = (D + 2) * U * np.where(hidden, 0, np.abs(q[:, h]) @ np.abs(kk).T).max(1) / np.sqrt(D)
        bound[:, h, 0] = np.abs(vv).max() * (2 * dt + 128 * U)
    return y, bound


def workgroups(lib, past, fresh, H, KV, dtype, D):
    """Those that take wide items, and how many of the items are parts."""
    n, items = schedule(lib, past, fresh, H, KV, dtype, 1 << 14, D)
    assert n >= 0
    wide = items[items[:, 7] == 1]
    return len(wide) * KV, int((wide[:, 6] >= 0).sum())


STEPS = [
    # past, fresh, H, KV; some items uncut, some cut
    ([0, 700, 33, 5, 300, 0, 128, 64], [260, 130, 300, 257, 129, 384, 200, 140], 16, 16),
    ([0, 65, 900, 1, 17, 500], [70, 129, 64, 200, 191, 128], 36, 12),
]


@pytest.mark.parametrize("D", [64, 40, 33, 96, 80, 72, 95, 128, 104, 127])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_two_groups_a_wave(rt, step, D):
    past, fresh, H, KV = STEPS[step]
    n, parts = workgroups(rt.lib, past, fresh, H, KV, gptc.F32, D)
    assert n >= TWO_GROUPS and parts > 0
    pool = Pool(rt, past, fresh, H, KV, D, 32, gptc.F32, seed=D)
    kept = pool.fill([p + f for p, f in zip(past, fresh)])
    pool.set()
    N = sum(fresh)
    q = pool.normal(N, H, D)
    tq, out = rt.from_numpy(q.reshape(N, -1)), rt.empty((N, H * D))
    pool.plan.attention(0, tq, out)
    got, row = rt.to_numpy(out).reshape(N, H, D), 0
    for s, (p, f) in enumerate(zip(past, fresh)):
        want, bound = attention(q[row:row + f].astype(np.float64), kept[s], p)
        err = np.abs(got[row:row + f] - want)
        assert (err <= bound).all(), (s, float((err / bound).max()))
        row += f
    pool.free()
    rt.free(tq)
    rt.free(out)


@pytest.mark.parametrize("D", [64, 33, 96, 80, 128, 127])
def test_two_groups_hide_what_is_not_finite(rt, D):
    """A later token's values that are no finite bf16 sums: the rows before it are what they are without."""
    past, fresh, H, KV = STEPS[0]
    pool = Pool(rt, past, fresh, H, KV, D, 32, gptc.F32, seed=D + 1)
    kept = pool.fill([p + f for p, f in zip(past, fresh)])
    bad = [(0, 150, 0, np.inf), (1, 70, D - 1, np.nan), (2, 299, 5, float(np.finfo(np.float32).max)), (5, 127, 9, -np.inf),
           (5, 128, 9, -float(np.finfo(np.float32).max))]
    for s, i, d, x in bad:
        page, slot = pool.rows(s, past[s] + i, past[s] + i + 1)
        pool.v[0][page[0], :, slot[0], d] = x
    torch.cuda.synchronize()
    pool.set()
    N = sum(fresh)
    q = pool.normal(N, H, D)
    tq, out = rt.from_numpy(q.reshape(N, -1)), rt.empty((N, H * D))
    pool.plan.attention(0, tq, out)
    got, row = rt.to_numpy(out).reshape(N, H, D), 0
    for s, (p, f) in enumerate(zip(past, fresh)):
        want, bound = attention(q[row:row + f].astype(np.float64), kept[s], p)
        seen = np.zeros((f, 1, D), bool)
        for at, i, d, _ in bad:
            if at == s:
                seen[i:, 0, d] = True
        assert ((np.abs(got[row:row + f] - want) <= bound) | seen).all(), s
        row += f
    pool.free()
    rt.free(tq)
    rt.free(out)
