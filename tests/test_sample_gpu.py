"""Drawing tokens on the GPU (gptc_sample_cuda) against the definition in 64 bits.

Ids have to be equal.  A kept token's share is a ratio of whole-number weights that are off by at most half of
2^-46 of the largest each, then rounded to a float: with V weights it is off by at most (1 + V) 2^-47 / total, total
being at least the largest weight, and half a step, 2^-24 of the share.
"""
import numpy as np
import pytest

import gptc

pytestmark = pytest.mark.gpu

FMAX = np.float32(np.finfo(np.float32).max)


def draw(logits, params, u):
    """ids and shares of the rows, from the definition."""
    ids, probs = [], []
    for x, (temperature, top_k, top_p, min_p), coin in zip(logits, params, u):
        x = x.astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        order = np.argsort(-x, kind="stable")
        best = x[order[0]]
        if best == -np.inf:
            ids.append(-1)
            probs.append(0.0)
            continue
        if not temperature > 0:
            ids.append(order[0])
            probs.append(1.0)
            continue
        if 1 <= top_k < len(x):
            order = order[:int(top_k)]
        with np.errstate(invalid="ignore"):
            w = np.where(x[order] == best, 1.0, np.exp((x[order] - best) / min(temperature, 1e30)))
        if top_p < 1:
            before = np.concatenate([[0.0], np.cumsum(w)])
            n = max(1, int((before[:-1] < top_p * before[-1]).sum()))
            order, w = order[:n], w[:n]
        if min_p > 0:
            keep = w >= min(min_p, 1.0)
            order, w = order[keep], w[keep]
        byid = np.argsort(order)
        order, w = order[byid], w[byid]
        upto = np.cumsum(w)
        coin = float(coin) if coin > 0 else 0.0
        n = int((upto <= coin * upto[-1]).sum())
        if n >= len(w):
            n = int(np.flatnonzero(w)[-1])
        ids.append(order[n])
        probs.append(w[n] / upto[-1])
    return np.array(ids), np.array(probs)


def sample(rt, logits, params, u, prob=True):
    rows = len(logits)
    t = [rt.from_numpy(x) for x in (logits, params, u)] + [rt.empty((rows,)), rt.empty((rows,)) if prob else None]
    rt.lib.gptc_sample_cuda(*t)
    out = rt.to_numpy(t[3]), rt.to_numpy(t[4]) if prob else None
    for x in t:
        if x is not None:
            rt.free(x)
    return out


def check(rt, logits, params, u):
    logits, u = np.asarray(logits, np.float32), np.asarray(u, np.float32)
    params = np.asarray(params, np.float32)
    each = np.broadcast_to(params.reshape(-1, 4), (len(logits), 4))
    want, share = draw(logits, each.astype(np.float64), u.astype(np.float64))
    ids, prob = sample(rt, logits, params, u)
    assert np.array_equal(ids, want), np.flatnonzero(ids != want)
    tol = 2.0 ** -24 * share + (1 + logits.shape[1]) * 2.0 ** -47
    assert (np.abs(prob - share) <= tol).all(), np.abs(prob - share).max()
    return ids, prob


def language(rng, rows, V):
    rank = rng.random((rows, V)).argsort(1)
    return (-1.2 * np.log1p(rank) + 0.5 * rng.standard_normal((rows, V)) + 3 * rng.standard_normal((rows, 1))).astype(np.float32)


SETTINGS = {
    "plain": (1.0, 0, 1.0, 0.0),
    "warm": (1.7, 0, 1.0, 0.0),
    "top_k": (0.8, 40, 1.0, 0.0),
    "top_k 1": (0.8, 1, 1.0, 0.0),
    "top_k most": (0.8, 3000, 1.0, 0.0),
    "top_p": (0.9, 0, 0.9, 0.0),
    "top_p most": (1.2, 0, 0.9999, 0.0),
    "top_p none": (0.9, 0, 0.0, 0.0),
    "min_p": (1.0, 0, 1.0, 0.05),
    "min_p all": (1.0, 0, 1.0, 2.0),
    "all": (0.7, 50, 0.95, 0.02),
    "top_k and top_p": (1.1, 5000, 0.8, 0.0),
    "top_p of many": (1.3, 0, 0.97, 0.0),
    "top_p, then less by min_p": (0.9, 0, 0.95, 0.2),
    "top_p, nothing by min_p": (1.2, 0, 0.9, 1e-5),
    "top_p and min_p near": (1.0, 0, 0.8, 0.0015),
    "all, many": (1.4, 4000, 0.9, 1e-4),
    "greedy": (0.0, 40, 0.9, 0.1),
}


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1024, 1025, 4099, 50257, 131072, 200001])
@pytest.mark.parametrize("name", sorted(SETTINGS))
def test_settings(rt, name, V):
    rng = np.random.default_rng(V)
    rows = 6
    check(rt, language(rng, rows, V), SETTINGS[name], rng.random(rows))


def test_settings_of_each_row(rt):
    rng = np.random.default_rng(3)
    params = np.array([SETTINGS[n] for n in sorted(SETTINGS)] * 8)
    check(rt, language(rng, len(params), 50257), params, rng.random(len(params)))


@pytest.mark.parametrize("V", [7, 1000, 3000, 50257])
@pytest.mark.parametrize("name", ["plain", "top_k", "top_k most", "top_p", "top_p most", "min_p", "all"])
def test_equal_logits(rt, name, V):
    """Ties go by index: every logit equal, and logits of a few values."""
    rng = np.random.default_rng(V)
    same = np.full((2, V), 1.25)
    few = rng.integers(-3, 4, (2, V)).astype(np.float64)
    zeros = np.where(rng.random((2, V)) < 0.5, 0.0, -0.0)
    lowest = np.full((1, V), -FMAX)
    check(rt, np.concatenate([same, few, zeros, lowest]), SETTINGS[name], rng.random(7))


@pytest.mark.parametrize("name", sorted(SETTINGS))
def test_masked_and_special_logits(rt, name):
    rng = np.random.default_rng(8)
    x = language(rng, 10, 5000)
    x[0, rng.random(5000) < 0.9] = -np.inf
    x[1, :] = -np.inf
    x[2, :] = -np.inf
    x[2, 4321] = -3.0
    x[3, rng.random(5000) < 0.5] = np.nan
    x[4, :] = np.nan
    x[5, rng.random(5000) < 0.9] = -FMAX
    x[6, [17, 99, 2048]] = np.inf
    x[7, :] = -FMAX
    x[7, 4999] = FMAX
    x[8, :] = np.nan
    x[8, [5, 6]] = -np.inf, 2.0
    x[9] *= 1e-30
    ids, _ = check(rt, x, SETTINGS[name], rng.random(10))
    assert ids[1] == -1 and ids[4] == -1 and ids[2] == 4321 and ids[8] == 6 and ids[6] in (17, 99, 2048)


@pytest.mark.parametrize("temperature", [1e-40, 1e-6, 0.01, 100.0, 1e6, 1e38, np.inf, np.nan, -1.0])
def test_temperatures(rt, temperature):
    rng = np.random.default_rng(11)
    x = language(rng, 5, 4097)
    params = [(temperature, *f) for f in ((0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.3), (2000, 0.5, 0.1))]
    check(rt, x, params, rng.random(5))


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, 2.0 ** -149, np.nan])
def test_ends_of_the_random_number(rt, u):
    rng = np.random.default_rng(12)
    x = language(rng, 3, 3001)
    x[:, [0, 3000]] = -np.inf  # the first and the last token cannot be drawn
    ids, _ = check(rt, x, [SETTINGS[n] for n in ("plain", "top_p", "top_k")], np.full(3, u))
    assert (ids > 0).all() and (ids < 3000).all()


def test_draws_follow_the_distribution_of_evenly_spread_numbers(rt):
    """n evenly spread numbers draw each token as often as its share says, to within one."""
    rng = np.random.default_rng(13)
    n = 4096
    x = np.repeat(2 * rng.standard_normal((1, 50)).astype(np.float32), n, 0)
    ids, prob = check(rt, x, (1.0, 20, 1.0, 0.0), (np.arange(n) + 0.5) / n)
    for i in np.unique(ids):
        assert abs((ids == i).sum() - n * prob[ids == i][0]) <= 1.001
    assert len(np.unique(ids)) <= 20


def test_without_shares_and_repeatable(rt):
    rng = np.random.default_rng(14)
    x, u = language(rng, 40, 50257), rng.random(40).astype(np.float32)
    p = np.array(SETTINGS["top_p"], np.float32)
    first, prob = sample(rt, x, p, u)
    for _ in range(3):
        again, share = sample(rt, x, p, u)
        assert np.array_equal(first, again) and np.array_equal(prob, share)
    assert np.array_equal(first, sample(rt, x, p, u, prob=False)[0])


def test_greedy_is_the_argmax(rt):
    rng = np.random.default_rng(15)
    x = language(rng, 9, 50257)
    ids, _ = sample(rt, x, np.zeros(4, np.float32), np.zeros(9, np.float32))
    tx, best = rt.from_numpy(x), rt.empty((9,))
    rt.lib.gptc_argmax_cuda(tx, best)
    assert np.array_equal(ids, rt.to_numpy(best))
    rt.free(tx)
    rt.free(best)


def test_rows_of_three_dimensions_and_none(rt):
    rng = np.random.default_rng(16)
    x, u = language(rng, 4, 100), rng.random(4).astype(np.float32)
    p = np.array(SETTINGS["all"], np.float32)
    flat, _ = sample(rt, x, p, u)
    t = [rt.from_numpy(a) for a in (x.reshape(4, 1, 100), p, u)] + [rt.empty((4, 1)), None]
    rt.lib.gptc_sample_cuda(*t)
    assert np.array_equal(rt.to_numpy(t[3])[:, 0], flat)


def test_the_largest_vocabulary(rt):
    """2^24 tokens: sums of 2^24 weights, stretches longer than a list, indices that are floats just so."""
    rng = np.random.default_rng(17)
    x = rng.standard_normal((3, 1 << 24)).astype(np.float32)
    x[:, -1] = x.max() + 1
    check(rt, x, [SETTINGS["top_k"], SETTINGS["top_p"], SETTINGS["plain"]], [0.3, 0.97, 1 - 2.0 ** -24])


def test_sampled_generation_over_a_contiguous_cache(rt):
    """gptc_gpt2_decode's logits go to the draw as they are, and the drawn ids to the next step, without a copy between."""
    from test_generate_gpu import c3_params, make_model
    V, block, L, H, C, B, steps = 523, 64, 2, 4, 64, 3, 24
    model = make_model(rt, c3_params(V, block, L, C, 5, std=0.2, jitter=0.05), V, block, L, H, C)
    cache, rng = gptc.KVCache(rt, model, B, block), np.random.default_rng(5)
    settings = np.array([SETTINGS[n] for n in ("top_k", "top_p", "all")], np.float32)
    coins = rng.random((steps, B)).astype(np.float32)
    params, u = rt.from_numpy(settings), [rt.from_numpy(c) for c in coins]
    ids = rt.from_numpy(rng.integers(0, V, (B, 1)).astype(np.float32))
    kept = []
    for pos in range(steps):
        logits, drawn = cache.decode(ids, pos), rt.empty((B, 1))
        rt.lib.gptc_sample_cuda(logits, params, u[pos], ids, None)
        rt.lib.tensor_copy(drawn, ids)
        kept.append((logits, drawn))
    for (logits, drawn), coin in zip(kept, coins):
        want, _ = draw(rt.to_numpy(logits)[:, 0], settings.astype(np.float64), coin.astype(np.float64))
        assert np.array_equal(rt.to_numpy(drawn)[:, 0], want)
    assert len({tuple(rt.to_numpy(d)[:, 0]) for _, d in kept}) > steps // 2
    for t in [params, ids, *u, *(t for pair in kept for t in pair)]:
        rt.free(t)
    cache.free()
    model.free()
