"""The cross entropy without logits on either side of where W is laid out, every kind of call,
with the reference, inputs and tolerances of test_head_loss_gpu.py.  (The sizes of test_head_embed_sizes_gpu.py that are named
after this line lie on either side of an earlier one.)"""
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
