"""The cross entropy without logits on either side of where W is laid out, every kind of call, and across its pieces of rows,
with the reference, inputs and tolerances of test_head_loss_gpu.py.  (The sizes of test_head_embed_sizes_gpu.py that are named
after this line lie on either side of an earlier one.)"""
import numpy as np
import pytest

import test_head_loss_gpu as head

pytestmark = pytest.mark.gpu

KINDS = {"loss": dict(dx=False, dW=False), "both": {}, "dx": dict(dW=False), "dW": dict(dx=False)}


def as_it_comes(R, V, C, grad):
    """Whether W is read as it comes (few_rows of head_loss.hip)."""
    read = -(-R // 128) * 128
    if R > 4096 or R * C >= 1 << 28:
        return False
    if not grad:
        return read <= 512 + 5000000000 // (V * (C + 4))
    return R <= 128 or (read <= 240 + 1600000000 // (V * (C + 500)) and R * C <= 1 << 21)


SIDES = [(kind, V, C, R) for kind, V, C, R in [
    ("loss", 50257, 70, 1792), ("loss", 50257, 320, 768), ("loss", 5003, 300, 3712), ("loss", 300, 33, 4096),
    ("loss", 130000, 500, 512), ("both", 50257, 70, 256), ("both", 50257, 700, 256), ("both", 5003, 100, 768),
    ("both", 1000, 70, 2944), ("both", 300, 768, 2730), ("both", 130, 1000, 2097), ("both", 300, 33, 4096),
    ("dx", 5003, 100, 768), ("dx", 50257, 70, 256), ("dW", 5003, 100, 768), ("dW", 50257, 70, 256), ("dx", 130, 1000, 2097),
    ("dW", 130, 1000, 2097)]]


@pytest.mark.parametrize("over", [0, 1])
@pytest.mark.parametrize("kind,V,C,R", SIDES)
def test_either_side_of_where_w_is_laid_out(rt, kind, V, C, R, over):
    assert as_it_comes(R, V, C, kind != "loss") and not as_it_comes(R + 1, V, C, kind != "loss")
    a = head.inputs(R + over, V, C, seed=20, weights=True)
    head.agree(head.Call(rt, *a, **KINDS[kind]), head.Exact(*a))


@pytest.mark.parametrize("accumulate", [False, True])
def test_gpt2_vocabulary_in_two_pieces(rt, accumulate):
    """3500 rows of 50257 tokens are pieces of 3328 and 172; rows of weight 0 in both hold NaN."""
    R, V, C = 3500, 50257, 100
    x, W, t, w = head.inputs(R, V, C, seed=21, weights=True)
    w[[0, 3327, 3328, 3400, 3499]] = 0
    w[3498] = 1
    clean = np.where(w[:, None] == 0, 0, x)
    dead = w == 0
    x[dead], t[dead] = np.nan, -3
    ref = head.Exact(clean, W, np.where(dead, 0, t), w)
    before = np.random.default_rng(22).standard_normal((V, C)).astype(np.float32) if accumulate else None
    got = head.Call(rt, x, W, t, w, accumulate=before)
    dW = got.dW
    got.dW = None
    head.agree(got, ref)
    assert not got.dx[dead].any() and not got.losses[dead].any()
    # The second piece's sum is added to the first one's, and that to what was there: a rounding each.
    want, tol = ref.dW, ref.dW_tol
    first = head.Exact(clean[:3328], W, np.where(dead, 0, t)[:3328], w[:3328]).dW.abs() * (3328 / R)
    if accumulate:
        want, tol = want + head.dev(before), tol + head.U * (head.dev(before).abs() + first)
    head.check("dW", dW, want, tol + head.U * (first + want.abs()))
    head.agree(head.Call(rt, x, W, t, w, dx=False, dW=False), ref)


@pytest.mark.parametrize("kw", [dict(dW=False), dict(dx=False)])
def test_one_gradient_in_two_pieces(rt, kw):
    a = head.inputs(3457, 50257, 70, seed=23, weights=True)
    head.agree(head.Call(rt, *a, **kw), head.Exact(*a))
