"""gptc_embedding_forward_scaled_cuda and gptc_embedding_backward_sorted_cuda on the GPU against their definitions in 64
bits.

Tolerances, u = 2^-24: a looked-up value is one rounding, of scale w or of scale w + p; a sum of m rows is off by at most
(m + 1) u of the sum of their magnitudes in any order, by one u more for the scale and one for the value it is added to.
Subnormal results are off by half their step, 2^-150.
"""
import ctypes
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
TINY = 2.0 ** -150


def close(name, got, want, tol):
    assert np.array_equal(np.isnan(got), np.isnan(want)), name
    err = np.where(np.isnan(want), 0.0, np.abs(got.astype(np.float64) - want))
    bound = np.where(np.isnan(want), 0.0, tol) + TINY
    print(f"  {name}: error at most {(err / bound).max() if err.size else 0:.3f} of its bound", flush=True)
    assert (err <= bound).all(), name


def valid(ids, V):
    with np.errstate(invalid="ignore"):
        ok = (ids > -1.0) & (np.trunc(ids) < V)
        return np.where(ok, np.trunc(np.where(ok, ids, 0)).astype(np.int64), -1)


def lookup(rt, W, P, ids, scale):
    t = [rt.from_numpy(W), None if P is None else rt.from_numpy(P), rt.from_numpy(ids), rt.empty(ids.shape + W.shape[1:])]
    rt.lib.gptc_embedding_forward_scaled_cuda(t[0], t[1], t[2], scale, t[3])
    got = rt.to_numpy(t[3])
    for x in t:
        if x is not None:
            rt.free(x)
    return got


def gather(rt, g, ids, scale, dW, dP=None, accumulate=0):
    """dW, dP: what the tensors hold before."""
    t = [rt.from_numpy(g), rt.from_numpy(ids), rt.from_numpy(dW), None if dP is None else rt.from_numpy(dP)]
    rt.lib.gptc_embedding_backward_sorted_cuda(t[0], t[1], scale, t[2], t[3], accumulate)
    got = rt.to_numpy(t[2]), None if dP is None else rt.to_numpy(t[3])
    for x in t:
        if x is not None:
            rt.free(x)
    return got


def gathered(g, ids, scale, V, positions):
    """(dW, its bound, dP, its bound) in 64 bits."""
    C, T = g.shape[-1], ids.shape[-1]
    rows, at = g.reshape(-1, C).astype(np.float64), valid(ids.ravel(), V)
    dW, mag, count = np.zeros((V, C)), np.zeros((V, C)), np.zeros((V, 1))
    ok = at >= 0
    np.add.at(dW, at[ok], rows[ok])
    np.add.at(mag, at[ok], np.abs(rows[ok]))
    np.add.at(count, at[ok], 1)
    dP, dPm = np.zeros((positions, C)), np.zeros((positions, C))
    dP[:T], dPm[:T] = rows.reshape(-1, T, C).sum(0), np.abs(rows).reshape(-1, T, C).sum(0)
    return scale * dW, (count + 3) * U * mag * abs(scale), dP, (len(rows) // max(T, 1) + 3) * U * dPm


def ids_of(kind, shape, V, seed=0):
    rng = np.random.default_rng([seed, V, *shape])
    n = int(np.prod(shape))
    if kind == "uniform":
        x = rng.integers(0, V, n)
    elif kind == "text":  # the k-th most frequent about 1/k as often as the first
        x = rng.permutation(V)[np.minimum(V - 1, (np.exp(rng.random(n) * np.log(V + 1)) - 1).astype(np.int64))]
    elif kind == "one":
        x = np.full(n, V - 1)
    elif kind == "two":
        x = np.where(rng.random(n) < 0.9, 0, V - 1)
    else:  # a third of them outside the table
        x = rng.integers(0, V, n).astype(np.float64)
        bad = rng.random(n) < 0.34
        x[bad] = rng.choice([-1, -5e8, V, V + 3.5, 1e9, 3e38, np.nan, np.inf, -np.inf], bad.sum())
        x[~bad] += rng.choice([0, 0, 0.25, 0.75], (~bad).sum()) * (V < 1 << 20)
        x[rng.integers(0, n)] = -0.75  # truncates to 0
    return x.astype(np.float32).reshape(shape)


@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("shape,V,C,scale,kind", [
    ((1, 1), 1, 1, 1.0, "one"), ((8, 1), 50257, 768, 1.0, "uniform"), ((3, 5), 10, 3, -2.5, "outside"),
    ((2, 7, 9), 100, 64, 27.7, "outside"), ((4, 129), 1000, 260, 0.3, "text"), ((2, 33), 70, 1601, 40.0, "uniform"),
    ((5,), 9, 8, 1.0, "two"), ((1, 2000), 300, 4, 1e-30, "text")])
def test_lookup(rt, shape, V, C, scale, kind, positions):
    rng = np.random.default_rng(1)
    W = rng.standard_normal((V, C)).astype(np.float32)
    P = rng.standard_normal((shape[-1] + 2, C)).astype(np.float32) if positions else None
    ids = ids_of(kind, shape, V)
    at = valid(ids, V)
    want = np.where((at >= 0)[..., None], np.float64(np.float32(scale)) * W[at].astype(np.float64), np.nan)
    if positions:
        want = want + P[:shape[-1]].astype(np.float64)
    close("rows", lookup(rt, W, P, ids, scale), want, U * np.abs(want))


GATHERS = [
    ((1, 1), 1, 1, "one"), ((1, 1), 5, 4, "one"), ((2, 3), 4, 3, "uniform"), ((3, 333), 5003, 100, "text"),
    ((1, 8), 50, 768, "two"), ((7, 9), 30, 260, "outside"), ((2, 500), 3, 64, "uniform"), ((3, 700), 200, 33, "one"),
    ((12, 1024), 50257, 20, "text"), ((12288, 1), 77, 8, "text"), ((1, 12289), 77, 8, "text"), ((4, 4096), 256, 5, "uniform"),
    ((5, 4096), 255, 12, "two"), ((3, 7001), 70000, 6, "text"), ((2, 9001), 300000, 4, "outside"), ((9, 2048), 1, 16, "one"),
    ((8, 1024), 1000, 768, "outside"), ((100, 1), 20, 1601, "text"), ((3, 6, 70), 40, 16, "text")]


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("shape,V,C,kind", GATHERS)
def test_gradient(rt, shape, V, C, kind, accumulate):
    rng = np.random.default_rng(2)
    g = rng.standard_normal((*shape, C)).astype(np.float32)
    ids = ids_of(kind, shape, V)
    scale = 1.75
    P = shape[-1] + (3 if accumulate else 0)
    fill = (lambda *s: rng.standard_normal(s).astype(np.float32)) if accumulate else (lambda *s: np.full(s, np.nan, np.float32))
    dW0, dP0 = fill(V, C), fill(P, C)
    want_W, tol_W, want_P, tol_P = gathered(g, ids, scale, V, P)
    if accumulate:
        want_W, want_P = want_W + dW0, want_P + dP0
        tol_W, tol_P = tol_W + U * np.abs(want_W), tol_P + U * np.abs(want_P)
    dW, dP = gather(rt, g, ids, scale, dW0, dP0, accumulate)
    close("dW", dW, want_W, tol_W)
    close("dP", dP, want_P, tol_P)
    alone, _ = gather(rt, g, ids, scale, dW0, None, accumulate)
    assert np.array_equal(alone, dW)
    if accumulate:  # what no id names is left alone, to the bit
        named = np.isin(np.arange(V), valid(ids.ravel(), V))
        assert np.array_equal(dW[~named], dW0[~named]) and np.array_equal(dP[shape[-1]:], dP0[shape[-1]:])


@pytest.mark.parametrize("n,V", [(5000, 400), (40000, 400)])
def test_rows_are_added_in_their_order(rt, n, V):
    """Up to eight rows an id that lie in one part: bit for bit the chain of float sums in the order of the rows."""
    rng = np.random.default_rng(3)
    ids = np.full((1, n), np.nan, np.float32)
    places = rng.permutation(n)[:300]
    ids[0, places] = rng.integers(0, V, 300)
    g = rng.standard_normal((1, n, 32)).astype(np.float32)
    dW, _ = gather(rt, g, ids, 1.0, np.zeros((V, 32), np.float32))
    order = np.sort(places)
    order = order[np.argsort(ids[0, order], kind="stable")]
    want, seen = np.zeros((V, 32), np.float32), {}
    for at, i in enumerate(order):
        seen.setdefault(int(ids[0, i]), []).append((at, i))
    whole = 0
    for v, rows in seen.items():
        if rows[0][0] // 8 == rows[-1][0] // 8:  # within one part, whatever its length
            for _, i in rows:
                want[v] = want[v] + g[0, i]
            assert np.array_equal(dW[v], want[v])
            whole += 1
    assert whole > 50


@pytest.mark.parametrize("shape,V,C,kind", [((4, 700), 90, 64, "text"), ((5, 4096), 300, 40, "text")])
def test_the_same_every_time(rt, shape, V, C, kind):
    g = np.random.default_rng(4).standard_normal((*shape, C)).astype(np.float32)
    ids, zero = ids_of(kind, shape, V), np.zeros((V, C), np.float32)
    one, _ = gather(rt, g, ids, 3.0, zero)
    gather(rt, g[:, ::-1], ids_of("uniform", shape, V), 2.0, zero)  # other values in the scratch
    two, _ = gather(rt, g, ids, 3.0, zero)
    assert np.array_equal(one, two)


def test_no_ids(rt):
    """Nothing to add: zeros when overwritten, nothing else."""
    dW, dP = gather(rt, np.zeros((0, 8), np.float32), np.zeros(0, np.float32), 1.0, np.full((5, 8), 3.0), np.full((2, 8), 3.0))
    assert not dW.any() and not dP.any()
    dW, dP = gather(rt, np.zeros((0, 8), np.float32), np.zeros(0, np.float32), 1.0, np.full((5, 8), 3.0),
                    np.full((2, 8), 3.0), 1)
    assert (dW == 3).all() and (dP == 3).all()


@pytest.mark.parametrize("C", [8, 7])
def test_tensors_off_16_bytes(rt, C):
    """Every tensor one float into its block; what lies around the results stays."""
    rng = np.random.default_rng(6)
    V, B, T = 40, 3, 50
    n = {"W": rng.standard_normal((V, C)), "P": rng.standard_normal((T, C)), "ids": ids_of("text", (B, T), V),
         "out": np.zeros((B, T, C)), "g": rng.standard_normal((B, T, C)), "dW": np.zeros((V, C)), "dP": np.zeros((T, C))}
    n = {k: v.astype(np.float32) for k, v in n.items()}
    blocks = {k: torch.full((v.size + 9,), 77.0, device="cuda") for k, v in n.items()}
    for k, v in n.items():
        blocks[k][1:1 + v.size] = torch.tensor(v.ravel(), device="cuda")
    torch.cuda.synchronize()

    def wrap(k):
        t = gptc.Tensor()
        t.t = ctypes.cast(blocks[k].data_ptr() + 4, ctypes.POINTER(ctypes.c_float))
        t.ndims, t.length, t.device = n[k].ndim, n[k].size, gptc.CUDA
        for i, s in enumerate(n[k].shape):
            t.shape[i] = s
        return ctypes.pointer(t)
    rt.lib.gptc_embedding_forward_scaled_cuda(wrap("W"), wrap("P"), wrap("ids"), 2.5, wrap("out"))
    rt.lib.gptc_embedding_backward_sorted_cuda(wrap("g"), wrap("ids"), 2.5, wrap("dW"), wrap("dP"), 0)
    rt.sync()
    got = {k: b.cpu().numpy() for k, b in blocks.items()}
    for k, v in n.items():
        assert got[k][0] == 77 and (got[k][1 + v.size:] == 77).all(), k
    res = {k: got[k][1:1 + n[k].size].reshape(n[k].shape) for k in n}
    want = 2.5 * n["W"].astype(np.float64)[n["ids"].astype(int)] + n["P"].astype(np.float64)
    close("rows", res["out"], want, U * np.abs(want))
    dW, tol_W, dP, tol_P = gathered(n["g"], n["ids"], 2.5, V, T)
    close("dW", res["dW"], dW, tol_W)
    close("dP", res["dP"], dP, tol_P)


def test_gradient_against_differences(rt):
    """The lookup is linear: <out(W + D) - out(W), g> = <D, dW>, to the roundings of the two lookups."""
    rng = np.random.default_rng(7)
    V, C, ids = 50, 12, ids_of("text", (4, 60), 50)
    W, D = (np.round(rng.standard_normal((V, C)) * 64).astype(np.float32) / 64 for _ in range(2))  # W + D is exact
    g = rng.standard_normal((4, 60, C)).astype(np.float32)
    one, two = (lookup(rt, x, None, ids, 1.5).astype(np.float64) for x in (W, W + D))
    dW, _ = gather(rt, g, ids, 1.5, np.zeros_like(W))
    mag = (np.abs(g) * (np.abs(one) + np.abs(two))).sum()
    left, right = ((two - one) * g).sum(), (D.astype(np.float64) * dW).sum()
    _, tol, _, _ = gathered(g, ids, 1.5, V, 60)
    assert abs(left - right) <= U * mag + (np.abs(D) * tol).sum()


def test_refused_under_capture_and_lookup_captured():
    """The gradient takes scratch and is refused; the lookup takes none and replays on new ids."""
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import ctypes
        import numpy as np
        import gptc
        rt = gptc.Runtime(gptc.load())
        rt.init()
        table = np.arange(160, dtype=np.float32).reshape(20, 8)
        W, ids, out = rt.from_numpy(table), rt.from_numpy(np.zeros((1, 6))), rt.empty((1, 6, 8))
        hip, stream, graph, run = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p(rt.stream()), ctypes.c_void_p(), ctypes.c_void_p()
        rt.sync()
        assert hip.hipStreamBeginCapture(stream, 1) == 0
        rt.lib.gptc_embedding_forward_scaled_cuda(W, None, ids, 3.0, out)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
        for k in range(4):
            now = (np.arange(6, dtype=np.float32)[None] * 7 + k) % 20
            new = rt.from_numpy(now)
            rt.lib.tensor_copy(ids, new)
            assert hip.hipGraphLaunch(run, stream) == 0
            assert np.array_equal(rt.to_numpy(out)[0], 3 * table[now[0].astype(int)])
        print("replayed", flush=True)
        assert hip.hipStreamBeginCapture(stream, 1) == 0
        rt.lib.gptc_embedding_backward_sorted_cuda(out, ids, 1.0, W, None, 0)
        print("returned")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1 and "replayed" in r.stdout and "not under graph capture" in r.stderr, r.stderr
    assert "returned" not in r.stdout
