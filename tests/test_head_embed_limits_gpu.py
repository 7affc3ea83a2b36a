"""The two ends of a GPT at sizes whose launches or whole numbers end.  Of the tables, values are whole numbers, whose sums
and products are exact in fp32."""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

import test_embed_sorted_gpu as sorted_gpu
import test_head_loss_gpu as head

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("positions", [False, True])
def test_lookup_of_more_ids_than_a_launch_has_waves(rt, positions):
    """2^26 rows, a wave each, are 2^32 threads."""
    shape = (4097, 16384)
    ids = (np.arange(shape[0] * shape[1], dtype=np.int64) * 7 % 41).astype(np.float32).reshape(shape)
    W = np.arange(37, dtype=np.float32)[:, None] - 11
    P = np.arange(16384, dtype=np.float32)[:, None] if positions else None
    got = sorted_gpu.lookup(rt, W, P, ids, 3.0)[..., 0]
    table = np.append(3 * W[:, 0], np.full(4, np.nan, np.float32))
    for b in (0, 1, 2048, 4094, 4095, 4096):
        want = table[ids[b].astype(int)]
        assert np.array_equal(got[b], want + P[:, 0] if positions else want, equal_nan=True), b
    assert np.array_equal(np.isnan(got), ids >= 37)


def test_gradient_of_as_many(rt):
    shape = (4097, 16384)
    ids = (np.arange(shape[0] * shape[1], dtype=np.int64) * 7 % 41).astype(np.float32).reshape(shape)
    g = np.ones((*shape, 1), np.float32)
    dW, dP = sorted_gpu.gather(rt, g, ids, 1.0, np.full((37, 1), np.nan, np.float32),
                               np.full((16384, 1), np.nan, np.float32))
    assert np.array_equal(dW[:, 0], np.bincount(ids.ravel().astype(np.int64), minlength=41)[:37].astype(np.float32))
    assert (dP == 4097).all()


def test_gradient_of_too_many_is_refused():
    """2^31 - 1 ids, whose parts' count may not wrap."""
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import gptc
        rt = gptc.Runtime(gptc.load())
        rt.init()
        n = (1 << 31) - 1
        g, ids, dW = rt.empty((n, 1)), rt.empty((n,)), rt.empty((5, 1))
        print("made", flush=True)
        rt.lib.gptc_embedding_backward_sorted_cuda(g, ids, 1.0, dW, None, 0)
        print("returned")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1 and "made" in r.stdout and "Too many rows" in r.stderr and "returned" not in r.stdout, r.stderr


@pytest.mark.parametrize("R", [5, 70])
def test_as_many_features_as_there_may_be(rt, R):
    """All but 200 of 2^22 - 1 features are zero in x and W: the reference has those alone."""
    C, rng = (1 << 22) - 1, np.random.default_rng(R)
    at = np.sort(rng.choice(C - 2, 198, replace=False))
    at = np.concatenate([at, [C - 2, C - 1]])
    x, W, t, w = head.inputs(R, 3, 200, weights=True)
    ref = head.Exact(x, W, t, w)
    wide = [np.zeros((len(a), C), np.float32) for a in (x, W)]
    for a, b in zip(wide, (x, W)):
        a[:, at] = b
    got = head.Call(rt, *wide, t, w)
    got.dx, dx, got.dW, dW = got.dx[:, at], got.dx, got.dW[:, at], got.dW
    head.agree(got, ref)
    assert np.count_nonzero(dx) == np.count_nonzero(got.dx) and np.count_nonzero(dW) == np.count_nonzero(got.dW)
    head.agree(head.Call(rt, *wide, t, w, dx=False, dW=False), ref)
