"""gptc_linear_cross_entropy_cuda on the GPU against its definition in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32, relative).
  logits: a product of C terms, each operand off by at most u and what is left out of a product by u more, the sums in
    chains of at most C / 32 sums of 32 terms:  E_l = (C / 32 + 64) u sum |x W|.  An operand's parts end 2^-39 below
    the largest value of its row, which adds 2^-39 (max|x| sum|W| + max|W| sum|x|).
  loss = lse - l[t]: 2 max E_l; the exponentials' arguments are rounded (2 u of their distance from the largest, as
    weighted by their share), sums of V shares in chains of at most V / 256 + 64; and the roundings of lse and l[t].
  d = w / R (p - [j = t]): p is off by p times twice E_l and what its exponential and 1 / sum are off, a few u of the
    rest, and 2^-39 of w / R where its parts end.
  dx = d W and dW = d^T x: |d| errors times the other operand, and (n / 32 + 64) u of the sums of |d| |W| or |d| |x|
    over n terms, with the parts' ends as above.
"""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest
import torch

import gptc

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
END = 2.0 ** -39


class Call:
    """One call on numpy inputs; results as 64-bit tensors on the GPU."""

    def __init__(self, rt, x, W, targets, weights=None, dx=True, dW=True, accumulate=None, losses=True):
        self.rt, ts = rt, []

        def put(a):
            if a is not None:
                ts.append(rt.from_numpy(a))
                return ts[-1]

        xt, wt, tt, gt = put(x), put(W), put(targets), put(weights)
        out = put(np.full(1, np.nan))
        lt = put(np.full(x.shape[:-1], np.nan)) if losses else None
        dxt = put(np.full(x.shape, np.nan)) if dx else None
        dwt = put(np.full(W.shape, np.nan) if accumulate is None else accumulate) if dW else None
        rt.lib.gptc_linear_cross_entropy_cuda(xt, wt, tt, gt, out, lt, dxt, dwt, 0 if accumulate is None else 1)
        self.loss = rt.to_numpy(out)
        self.losses, self.dx, self.dW = (None if t is None else rt.to_numpy(t) for t in (lt, dxt, dwt))
        self.losses = None if self.losses is None else self.losses.ravel()
        self.dx = None if self.dx is None else self.dx.reshape(-1, x.shape[-1])
        for t in ts:
            rt.free(t)


def dev(a):
    return torch.tensor(np.asarray(a, np.float64), device="cuda")


class Exact:
    """The definition in 64 bits, with the bounds above."""

    def __init__(self, x, W, targets, weights=None):
        x, W = dev(x).reshape(-1, W.shape[1]), dev(W)
        R, C = x.shape
        V = len(W)
        w = torch.ones(R, dtype=torch.float64, device="cuda") if weights is None else dev(weights).ravel()
        live = w != 0
        x = torch.where(live[:, None], x, 0.0)
        t = dev(targets).ravel().trunc().long()
        ok = (t >= 0) & (t < V)
        l = x @ W.t().contiguous()
        ax, aW = x.abs(), W.abs()
        El = (C / 32 + 64) * U * (ax @ aW.t().contiguous()) + END * (
            ax.amax(1)[:, None] * aW.sum(1) + ax.sum(1)[:, None] * aW.amax(1))
        Em = El.amax(1)
        m, lse = l.amax(1), torch.logsumexp(l, 1)
        p = torch.exp(l - lse[:, None])
        spread = (p * (m[:, None] - l)).sum(1)
        lt = l.gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
        self.losses = torch.where(live, torch.where(ok, lse - lt, torch.nan), 0.0)
        # What a sum of shares, its logarithm and the exponentials are off.
        share = (V / 256 + 64) * U + 2 * U * spread
        self.losses_tol = torch.where(live, 2 * Em + share + 4 * U * (lse.abs() + lt.abs() + m.abs()), 0.0)
        self.loss = (self.losses * w).sum() / R
        self.loss_tol = (self.losses_tol * w.abs()).sum() / R + 2 * U * (self.losses * w).abs().sum() / R
        d = p.clone()
        rows = torch.arange(R, device="cuda")
        d[rows[ok], t[ok]] -= 1
        f = (w / R)[:, None]
        rel = El + (2 * Em + share + 4 * U * (m.abs() + lse.abs()))[:, None] + 2 * U * (m[:, None] - l)
        Ed = torch.where(live[:, None], (p * torch.expm1(rel) + 8 * U * (d.abs() + p) + END) * f.abs(), 0.0)
        d *= f
        ad = d.abs()
        self.d = d
        self.dx = d @ W
        self.dx_tol = Ed @ aW + (V / 32 + 64) * U * (ad @ aW) + END * ad.sum(1)[:, None] * aW.amax(0)
        self.dW = d.t().contiguous() @ x
        fx = f.abs() * ax
        self.dW_tol = (Ed.t().contiguous() @ ax + (R / 32 + 64) * U * (ad.t().contiguous() @ ax) +
                       END * (ad / f.abs().clamp(min=1e-300)).sum(0)[:, None] * fx.amax(0))


def check(name, got, want, tol):
    got = dev(got).reshape(want.shape)
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaN in other places"
    err = torch.where(want.isnan(), 0.0, (got - want).abs())
    tol = torch.where(want.isnan(), 1.0, tol)
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    print(f"  {name}: error at most {worst:.3f} of its bound, largest {err.max().item():.2e}", flush=True)
    assert (err <= tol).all(), f"{name}: {worst} of the bound"


def agree(got, ref):
    check("loss", got.loss, ref.loss.reshape(1), ref.loss_tol.reshape(1))
    if got.losses is not None:
        check("losses", got.losses, ref.losses, ref.losses_tol)
    if got.dx is not None:
        check("dx", got.dx, ref.dx, ref.dx_tol)
    if got.dW is not None:
        check("dW", got.dW, ref.dW, ref.dW_tol)


def inputs(R, V, C, seed=0, weights=False, scale=1.0):
    rng = np.random.default_rng([seed, R, V, C])
    x = rng.standard_normal((R, C)).astype(np.float32)
    W = (rng.standard_normal((V, C)) * scale * 2.5 / np.sqrt(C)).astype(np.float32)
    targets = rng.integers(0, V, R).astype(np.float32)
    w = np.where(rng.random(R) < 0.3, 0.0, rng.uniform(0.1, 2.0, R)).astype(np.float32) if weights else None
    return x, W, targets, w


SIZES = [(1, 1, 1), (1, 2, 3), (3, 5, 1), (2, 4097, 31), (5, 129, 33), (63, 1000, 64), (64, 128, 32), (65, 127, 65),
         (129, 257, 100), (191, 3001, 96), (200, 5003, 100), (256, 512, 768), (333, 1000, 770), (512, 384, 64),
         (513, 700, 48), (1025, 2049, 129), (2100, 130, 36)]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("R,V,C", SIZES)
def test_loss_and_gradients(rt, R, V, C, weights):
    a = inputs(R, V, C, weights=weights)
    ref = Exact(*a)
    agree(Call(rt, *a), ref)
    agree(Call(rt, *a, dx=False, dW=False), ref)


def test_gpt2_vocabulary_in_several_pieces(rt):
    a = inputs(3000, 50257, 20, weights=True)
    agree(Call(rt, *a), Exact(*a))


def test_gpt2_width(rt):
    a = inputs(300, 50257, 768)
    agree(Call(rt, *a), Exact(*a))


@pytest.mark.parametrize("R,V,C", [(7, 50, 12), (300, 1000, 40)])
def test_parts_of_the_results(rt, R, V, C):
    """dx or dW alone, no row losses, dW added to what is there."""
    a = inputs(R, V, C, weights=True)
    ref = Exact(*a)
    whole = Call(rt, *a)
    for kw in ({"dx": False}, {"dW": False}, {"losses": False}):
        part = Call(rt, *a, **kw)
        for n in ("loss", "losses", "dx", "dW"):
            if getattr(part, n) is not None:
                assert np.array_equal(getattr(part, n), getattr(whole, n)), (kw, n)
    before = np.random.default_rng(3).standard_normal((V, C)).astype(np.float32)
    got = Call(rt, *a, accumulate=before)
    # One more rounding for every piece that is added.
    check("dW", got.dW, ref.dW + dev(before), ref.dW_tol + 2 * U * (ref.dW + dev(before)).abs() + 2 * U * dev(before).abs())


@pytest.mark.parametrize("R,V,C", [(9, 70, 8), (300, 600, 64)])
def test_padding_rows_take_no_part(rt, R, V, C):
    """Rows of weight 0 hold NaN, infinities and targets that are none; the others' results are those without them."""
    x, W, t, w = inputs(R, V, C, weights=True)
    w[:3] = [0.0, 1.0, 0.0]
    clean = Call(rt, np.where(w[:, None] == 0, 0, x), W, np.where(w == 0, 0, t), w)
    dead = np.flatnonzero(w == 0)
    x[dead[0::3]], x[dead[1::3]], x[dead[2::3]] = np.nan, np.inf, 3e38
    t[dead[0::2]], t[dead[1::2]] = -7, np.nan
    got = Call(rt, x, W, t, w)
    agree(got, Exact(np.where(w[:, None] == 0, 0, x), W, np.where(w == 0, 0, t), w))
    for n in ("loss", "losses", "dx", "dW"):
        assert np.array_equal(getattr(got, n), getattr(clean, n)), n
    assert not got.dx[dead].any() and not got.losses[dead].any()


@pytest.mark.parametrize("R", [4, 300])
def test_all_rows_padding(rt, R):
    x, W, t, _ = inputs(R, 300, 24)
    got = Call(rt, np.full_like(x, np.nan), W, t, np.zeros(R))
    assert got.loss[0] == 0 and not got.losses.any() and not got.dx.any() and not got.dW.any()
    before = np.random.default_rng(5).standard_normal(W.shape).astype(np.float32)
    assert np.array_equal(Call(rt, x, W, t, np.zeros(R), accumulate=before).dW, before)


@pytest.mark.parametrize("R", [6, 300])
def test_targets_outside_the_vocabulary(rt, R):
    """NaN losses; the gradients are the softmax's.  Targets are truncated."""
    x, W, t, _ = inputs(R, 90, 24)
    t[0], t[1], t[2], t[3] = -1, 90, 1e9, 17.9
    ref = Exact(x, W, t)
    got = Call(rt, x, W, t)
    agree(got, ref)
    assert np.isnan(got.losses[:3]).all() and np.isfinite(got.losses[3:]).all() and np.isnan(got.loss[0])
    t[0], t[1], t[2] = np.nan, np.inf, -np.inf
    again = Call(rt, x, W, t)
    assert np.array_equal(again.dx, got.dx) and np.array_equal(again.dW, got.dW) and np.isnan(again.losses[:3]).all()


@pytest.mark.parametrize("R", [5, 300])
def test_confident_and_far_logits(rt, R):
    """Logits hundreds apart: shares of exactly 0 and 1."""
    a = inputs(R, 400, 64, scale=60.0)
    ref = Exact(*a)
    got = Call(rt, *a)
    agree(got, ref)
    assert np.isfinite(got.dx).all() and np.isfinite(got.dW).all()


@pytest.mark.parametrize("R", [5, 300])
@pytest.mark.parametrize("shift", [-60, -30, 30, 50])
def test_values_far_from_one(rt, R, shift):
    """x times 2^shift and W times 2^-shift: the same logits."""
    x, W, t, w = inputs(R, 500, 70, weights=True)
    a = np.ldexp(x, shift), np.ldexp(W, -shift), t, w
    agree(Call(rt, *a), Exact(*a))


@pytest.mark.parametrize("R", [5, 300])
def test_rows_and_columns_of_other_sizes(rt, R):
    """Loud rows and features beside quiet ones."""
    x, W, t, w = inputs(R, 500, 70, weights=True)
    rng = np.random.default_rng(9)
    by_row, by_col = np.ldexp(1.0, rng.integers(-12, 4, (R, 1))), np.ldexp(1.0, rng.integers(-9, 9, 70))
    a = (x * by_row * by_col).astype(np.float32), (W / by_col).astype(np.float32), t, w
    agree(Call(rt, *a), Exact(*a))


@pytest.mark.parametrize("R", [5, 300])
def test_zeros(rt, R):
    """No difference between the tokens: loss log V, and rows that are all zero."""
    x, W, t, _ = inputs(R, 333, 50)
    agree(Call(rt, np.zeros_like(x), W, t), Exact(np.zeros_like(x), W, t))
    agree(Call(rt, x, np.zeros_like(W), t), Exact(x, np.zeros_like(W), t))


@pytest.mark.parametrize("R", [5, 300])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(rt, R, bad):
    """A row of x that holds one spoils its own loss and dx, and all of dW; no other row's."""
    x, W, t, _ = inputs(R, 200, 40)
    x[3, 7] = bad
    got, ref = Call(rt, x, W, t), Exact(np.where(np.isfinite(x), x, 0), W, t)
    others = np.arange(R) != 3
    assert not np.isfinite(got.losses[3]) and not np.isfinite(got.loss[0]) and not np.isfinite(got.dx[3]).any()
    assert not np.isfinite(got.dW).any()
    check("losses", got.losses[others], ref.losses[dev(others).bool()], ref.losses_tol[dev(others).bool()])
    check("dx", got.dx[others], ref.dx[dev(others).bool()], ref.dx_tol[dev(others).bool()])


@pytest.mark.parametrize("R,V,C", [(3, 10, 5), (300, 257, 33), (260, 512, 64)])
def test_tensors_off_16_bytes(rt, R, V, C):
    a = x, W, t, w = inputs(R, V, C, weights=True)
    ref = Exact(*a)
    # Every tensor of the call one float into its block.
    n = {"x": x, "W": W, "t": t, "w": w, "loss": np.zeros(1), "losses": np.zeros(R), "dx": np.zeros_like(x),
         "dW": np.zeros_like(W)}
    blocks = {k: torch.zeros(v.size + 9, device="cuda") for k, v in n.items()}
    for k, v in n.items():
        blocks[k][1:1 + v.size] = torch.tensor(np.asarray(v, np.float32).ravel(), device="cuda")
        blocks[k][1 + v.size:] = 77.0
    torch.cuda.synchronize()

    def wrap(k):
        tt = gptc.Tensor()
        tt.t = gptc.ctypes.cast(blocks[k].data_ptr() + 4, gptc.ctypes.POINTER(gptc.ctypes.c_float))
        tt.ndims, tt.length, tt.device = n[k].ndim, n[k].size, gptc.CUDA
        for i, s in enumerate(n[k].shape):
            tt.shape[i] = s
        return gptc.ctypes.pointer(tt)
    rt.lib.gptc_linear_cross_entropy_cuda(*(wrap(k) for k in n), 0)
    rt.sync()
    for k in ("loss", "losses", "dx", "dW"):
        got, want = blocks[k].cpu().numpy(), getattr(ref, k).reshape(n[k].shape)
        check(k, got[1:1 + n[k].size], want, getattr(ref, k + "_tol").reshape(n[k].shape))
        assert got[0] == 0 and (got[1 + n[k].size:] == 77.0).all(), k


def test_leading_dimensions(rt):
    x, W, t, w = inputs(60, 100, 16, weights=True)
    flat = Call(rt, x, W, t, w)
    got = Call(rt, x.reshape(3, 4, 5, 16), W, t.reshape(3, 4, 5), w.reshape(3, 20))
    for n in ("loss", "losses", "dx", "dW"):
        assert np.array_equal(getattr(got, n), getattr(flat, n)), n


@pytest.mark.parametrize("R,V,C", [(17, 3000, 80), (700, 3000, 80)])
def test_the_same_every_time(rt, R, V, C):
    a = inputs(R, V, C, weights=True)
    one = Call(rt, *a)
    Call(rt, *inputs(R + 9, V, C, seed=5))  # other values in the scratch
    two = Call(rt, *a)
    for n in ("loss", "losses", "dx", "dW"):
        assert np.array_equal(getattr(one, n), getattr(two, n)), n


@pytest.mark.parametrize("R", [6, 300])
def test_gradients_against_differences(rt, R):
    """(L(x + h v) - L(x - h v)) / 2h: off by h^2 / 6 of a third derivative, and by what the two losses are off over h.
    The third derivative of a row's lse is the third central moment of the logits' rates of change under the shares,
    at most 1 / (6 sqrt 3) of the cube of their spread (two values, of shares 1/2 +- 1/(2 sqrt 3))."""
    x, W, t, w = inputs(R, 150, 32, weights=True)
    got = Call(rt, x, W, t, w)
    rng = np.random.default_rng(4)
    h = 2.0 ** -5
    for name, v in (("x", rng.standard_normal(x.shape)), ("W", rng.standard_normal(W.shape) * 0.3)):
        v = v.astype(np.float32)
        ends, tol = [], 0.0
        for sign in (1, -1):
            y = ((x + np.float32(sign * h) * v) if name == "x" else x).astype(np.float32)
            Z = ((W + np.float32(sign * h) * v) if name == "W" else W).astype(np.float32)
            ends.append(float(Call(rt, y, Z, t, w, dx=False, dW=False).loss[0]))
            tol += Exact(y, Z, t, w).loss_tol.item() / (2 * h)
        rate = v.astype(np.float64) @ W.T.astype(np.float64) if name == "x" else x.astype(np.float64) @ v.T.astype(np.float64)
        spread = rate.max(1) - rate.min(1)
        tol += float((spread ** 3 * w).sum() / R) / (6 * 3 ** 0.5) * h * h / 6
        grad = got.dx if name == "x" else got.dW
        slope = float((grad.astype(np.float64) * v).sum())
        # The ends themselves are rounded: u of each value on either side.
        tol += float((np.abs(grad) * (np.abs(x if name == "x" else W) + h * np.abs(v))).sum()) * U / h
        print(f"  {name}: {slope:.6f} and {(ends[0] - ends[1]) / (2 * h):.6f}, bound {tol:.1e}", flush=True)
        assert abs(slope - (ends[0] - ends[1]) / (2 * h)) <= tol
        assert tol < 0.2 * abs(slope) or tol < 0.05


def test_refused_under_capture():
    """The call takes scratch: a captured one would replay on memory of others."""
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import ctypes
        import numpy as np
        import gptc
        rt = gptc.Runtime(gptc.load())
        rt.init()
        x, W, t, out = (rt.from_numpy(np.zeros(s, np.float32)) for s in ((4, 8), (16, 8), (4,), (1,)))
        rt.sync()
        hip = ctypes.CDLL("libamdhip64.so")
        assert hip.hipStreamBeginCapture(ctypes.c_void_p(rt.stream()), 2) == 0
        rt.lib.gptc_linear_cross_entropy_cuda(x, W, t, None, out, None, None, None, 0)
        print("returned")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1 and "not under graph capture" in r.stderr and "returned" not in r.stdout, r.stderr
