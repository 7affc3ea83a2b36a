"""The softmax of gptc_linear_cross_entropy_cuda apart from its products: logits that are exact in fp32.

x = (1, K) and W = (a_j, 1) with a_j a multiple of 1/16 and K whole: the logits a_j + K, their largest one m, and l - m are
exact, in the two fp16 parts and in every sum.  So a row's loss and gradients may not depend on K at all, and what is
left are the roundings of the softmax.  With u = 2^-24, V tokens:
  e = exp(l - m) comes as exp2 of (l - m) times log2(e) in fp32: off by 1.3 u of its argument, 2 u for exp2; where a part's
    sum moves to another largest value, that splits into distances which add up to l - m, each with 3 u more.
  s, the sum: at most V - 1 additions of positive values that are not 0, of which no chain has more than 75 + V / 2048, in
    at most ceil(V / 32), 12, moves:  S = (min(V - 1, 75 + V / 2048) + 3 min(ceil(V / 32), 12)) u + 2 u sum p |l - m|.
  loss = log s - (l_t - m): S, 4 u of log s and 2 u of the loss and its larger term.
  p = e / s: 2 u |l - m| + 6 u + S of p;  d = p - [j = t]: 2 u |d| more, and 2^-39 where its parts end.
  dx, dW: those times the other operand, and of the products' |terms| (4 + min(n, 64) + n / 32) u for n terms.
"""
import numpy as np
import pytest

import test_head_loss_gpu as head

pytestmark = pytest.mark.gpu

U, END = head.U, head.END
MANY = 4225  # rows past 4096: W is laid out


def tokens(kind, V):
    rng = np.random.default_rng([7, V])
    if kind == "confident":  # one token 11 above the others: their shares are 1e-5 and less
        a = rng.integers(0, 33, V) / 16
        a[V // 2] = 13
    elif kind == "equal":
        a = np.full(V, 3.0)
    else:
        a = rng.integers(-128, 129, V) / 16
    return a


def problem(kind, R, V, far):
    """Rows in pairs of one target, the second of each by K away."""
    rng = np.random.default_rng([8, R, V])
    a = tokens(kind, V)
    t = np.where(rng.random(R) < 0.5, int(a.argmax()), rng.integers(0, V, R))
    t[1::2] = t[0:2 * (R // 2):2]
    K = rng.integers(far // 2, far + 1, R) * rng.choice([-1, 1], R)
    K[0::2] = 0
    x = np.stack([np.ones(R), K], 1).astype(np.float32)
    W = np.stack([a, np.ones(V)], 1).astype(np.float32)
    return x, W, t.astype(np.float32), a


def bounds(x, W, t, a):
    """(losses, bound), (dx, bound), (dW, bound) in 64 bits; the logits of all rows differ by K alone."""
    R, V = len(x), len(a)
    t = t.astype(int)
    far = a - a.max()
    e = np.exp(far)
    s = e.sum()
    p = e / s
    S = (min(V - 1, 75 + V / 2048) + 3 * min(-(-V // 32), 12)) * U + 2 * U * (p * -far).sum()
    losses = np.log(s) - far[t]
    losses_tol = S + 4 * U * np.log(s) + 2 * U * (losses + np.abs(far[t]))
    d = np.repeat(p[None], R, 0)
    d[np.arange(R), t] -= 1
    Ed = (p * (2 * U * -far + 6 * U + S))[None] + 2 * U * np.abs(d) + END
    aW, ax = np.abs(W).astype(np.float64), np.abs(x).astype(np.float64)
    dx = d @ W.astype(np.float64) / R
    dx_tol = (Ed @ aW + (4 + min(V, 64) + V / 32) * U * (np.abs(d) @ aW)) / R
    dW = d.T @ x.astype(np.float64) / R
    dW_tol = (Ed.T @ ax + (4 + min(R, 64) + R / 32) * U * (np.abs(d).T @ ax) + END * R * ax.max(0)) / R
    return (losses, losses_tol), (dx, dx_tol), (dW, dW_tol)


def close(name, got, want, tol):
    err = np.abs(got.astype(np.float64) - want)
    print(f"  {name}: error at most {(err / tol).max():.3f} of its bound, largest {err.max():.2e}", flush=True)
    assert (err <= tol).all(), name


CASES = [(kind, R, V) for R in (2, 5, 31, 100, 300, MANY) for kind, V in
         (("confident", 5), ("confident", 40), ("confident", 600), ("spread", 40), ("spread", 600), ("equal", 4),
          ("equal", 333))]


@pytest.mark.parametrize("far", [128, 4000])
@pytest.mark.parametrize("kind,R,V", CASES)
def test_losses_of_exact_logits(rt, kind, R, V, far):
    x, W, t, a = problem(kind, R, V, far)
    got = head.Call(rt, x, W, t, dx=False, dW=False)
    close("losses", got.losses, *bounds(x, W, t, a)[0])
    pairs = R // 2 * 2
    assert np.array_equal(got.losses[0:pairs:2], got.losses[1:pairs:2])  # the same distances from the largest


@pytest.mark.parametrize("far", [128, 4000])
@pytest.mark.parametrize("kind,R,V", CASES)
def test_gradients_of_exact_logits(rt, kind, R, V, far):
    """dx of the constant feature is the sum of a row of d: 0 but for what the shares are off by together."""
    x, W, t, a = problem(kind, R, V, far)
    got = head.Call(rt, x, W, t)
    losses, dx, dW = bounds(x, W, t, a)
    close("losses", got.losses, *losses)
    close("dx", got.dx, *dx)
    close("dW", got.dW, *dW)
    pairs = R // 2 * 2
    assert np.array_equal(got.losses[0:pairs:2], got.losses[1:pairs:2])
    assert np.array_equal(got.dx[0:pairs:2], got.dx[1:pairs:2])


@pytest.mark.parametrize("R", [1, 40, 100, MANY])
@pytest.mark.parametrize("C", [33, 63, 70])
def test_a_loud_row_of_w_behind_a_quiet_one(rt, R, C):
    """Row 64 begins with values of 2^60, where x is 0.  They lie behind row 63's last features in memory, and belong to
    another 64 rows: row 63's logits, and all gradients but dx of those features, are as if they were 0."""
    x, W, t, w = head.inputs(R, 200, C, seed=12, weights=True)
    x[:, :31] = 0
    W[64:128] = 0
    t[0], w[0] = 63, 1
    ref = head.Exact(x, W, t, w)
    W[64, :31] = 2.0 ** 60
    got = head.Call(rt, x, W, t, w)
    ref.dx, ref.dx_tol, got.dx = ref.dx[:, 31:], ref.dx_tol[:, 31:], got.dx[:, 31:]
    head.agree(got, ref)
    head.agree(head.Call(rt, x, W, t, w, dx=False, dW=False), ref)


@pytest.mark.parametrize("R", [5, 90, 300, MANY])
@pytest.mark.parametrize("shift", [-118, -110, 110, 118])
def test_values_near_the_ends_of_fp32(rt, R, shift):
    """x times 2^shift and W times 2^-shift: ordinary logits, and a dx or dW of up to 2^119.  (The other one is subnormal.)"""
    x, W, t, w = head.inputs(R, 500, 70, seed=13, weights=True)
    a = np.ldexp(x, shift), np.ldexp(W, -shift), t, w
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a, dx=shift < 0, dW=shift > 0), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("R", [3, 100, MANY])
def test_unlikely_tokens(rt, R):
    """Shares are held to 2^-40: what a token's row of dW may be off by where all of them are far below 1, target or not."""
    V = 40
    a = -np.arange(V, dtype=np.float64)  # shares down to e^-39
    rng = np.random.default_rng([14, R])
    x = np.stack([np.ones(R), rng.integers(-2000, 2001, R)], 1).astype(np.float32)
    W = np.stack([a, np.ones(V)], 1).astype(np.float32)
    t = rng.integers(0, 3, R).astype(np.float32)
    got = head.Call(rt, x, W, t)
    _, dx, (dW, tol) = bounds(x, W, t, a)
    close("dx", got.dx, *dx)
    # The bound with 2^-40 of the share itself, and of x its own end 2^-40 below the column's largest.
    p = np.exp(a) / np.exp(a).sum()
    ax = np.abs(x).astype(np.float64)
    rel = (2 * -a + 6 + 3 * V + 2 * (p * -a).sum() + 4 + min(R, 64) + R / 32) * U
    tight = (2.0 ** -40 + rel * p)[3:, None] * ax.mean(0) + 2.0 ** -40 * p[3:, None] * ax.max(0)
    close("dW of unlikely tokens", got.dW[3:], dW[3:], np.minimum(tight, tol[3:]))


@pytest.mark.parametrize("R", [5, 90, 300, MANY])
@pytest.mark.parametrize("shift", [90, 100, 105])
def test_scales_that_are_subnormal(rt, R, shift):
    """Values of W of 2^-100 are held times 2^114, and come back by a factor below 2^-126; the results are ordinary."""
    x, W, t, w = head.inputs(R, 500, 70, seed=15, weights=True)
    a = np.ldexp(x, shift), np.ldexp(W, -shift), t, w
    head.agree(head.Call(rt, *a), head.Exact(*a))
