"""Appending to and attending over paged caches (include/paged.h) on the GPU, against the definitions in 64 bits.

Tolerances.  A rounding is off by at most half a step: u = 2^-24 for fp32, 2^-8 for bf16 pages.
  append: a rotated value x c - y s is two products and a sum: off by at most 3 u (|x c| + |y s|) <= 6 u max|x|,
    (in bf16 pages half a step of the value on top); without rotation fp32 pages hold the values themselves and bf16
    pages the nearest.
  attention: y = sum p v / sum p.  A score of D products is off by at most (D + 2) u sum|q k| scale (any order, and
    the scaling), which multiplies p by e^that; exp2 and the running sums of n weights add (log2 n + 8) u for sums in
    trees and runs of a few dozen keys, taken here as 64 u.  The products of bf16 pages with three-part values are
    exact to u.  So |dy| <= max|v| (2 max_j |dt_j| + 128 u), with |dt| <= (D + 2) u max_j sum_d |q k| / sqrt(D).
"""
import ctypes

import numpy as np
import pytest
import torch

import gptc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Pool:
    """A cache whose pages are torch tensors, NaN wherever no token lies, and a plan over it."""

    def __init__(self, rt, past, fresh, H, KV, D, page, dtype, seed=0, spare=3, layers=1, room=0, max_len=None):
        self.rt, self.past, self.fresh = rt, list(past), list(fresh)
        self.H, self.KV, self.D, self.page, self.layers = H, KV, D, page, layers
        self.rng = np.random.default_rng(seed)
        total = [p + f for p, f in zip(past, fresh)]
        need = [-(-t // page) for t in total]
        n_pages = sum(need) + spare
        order = self.rng.permutation(n_pages)
        self.table = np.zeros((len(total), max(need + [1])), np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.tdtype = torch.bfloat16 if dtype == gptc.BF16 else torch.float32
        self.k, self.v = ([torch.full((n_pages, KV, page, D), float("nan"), dtype=self.tdtype, device="cuda")
                           for _ in range(layers)] for _ in range(2))
        torch.cuda.synchronize()
        self.cache = gptc.PagedCache(rt, layers, n_pages, page, KV, D, dtype, [x.data_ptr() for x in self.k],
                                     [x.data_ptr() for x in self.v])
        self.plan = gptc.PagedPlan(rt, self.cache, H, len(total) + room, max(1, sum(fresh)) + room,
                                   max_len or max(total + [1]))

    def set(self):
        self.plan.set(self.past, self.fresh, self.table)

    def normal(self, *shape):
        return self.rng.standard_normal(shape).astype(np.float32)

    def rows(self, s, lo, hi):
        """Where tokens lo .. hi of sequence s lie: (pages, slots)."""
        t = np.arange(lo, hi)
        return torch.tensor(self.table[s, t // self.page], device="cuda").long(), torch.tensor(t % self.page, device="cuda")

    def fill(self, upto, std=1.0, layer=0):
        """Random tokens 0 .. upto[s] of each sequence, rounded to the pages' type; returned in 64 bits."""
        kept = []
        for s, n in enumerate(upto):
            k, v = (torch.tensor(std * self.normal(n, self.KV, self.D)).to(self.tdtype) for _ in range(2))
            at = self.rows(s, 0, n)
            self.k[layer][at[0], :, at[1]] = k.cuda()
            self.v[layer][at[0], :, at[1]] = v.cuda()
            kept.append((k.double().numpy(), v.double().numpy()))
        torch.cuda.synchronize()
        return kept

    def held(self, s, lo, hi, layer=0):
        at = self.rows(s, lo, hi)
        torch.cuda.synchronize()
        return tuple(x[layer][at[0], :, at[1]].double().cpu().numpy() for x in (self.k, self.v))

    def free(self):
        self.rt.sync()
        self.plan.free()
        self.cache.free()


def attention(q, kv, past, H, KV, D):
    """One sequence in 64 bits: q (n, H, D), kv its keys and values (past + n, KV, D); y, and the bound on its error."""
    k, v = kv
    n = q.shape[0]
    y, bound = np.zeros((n, H, D)), np.zeros((n, H, 1))
    for i in range(n):
        for h in range(H):
            kk, vv = k[:past + i + 1, h * KV // H], v[:past + i + 1, h * KV // H]
            t = kk @ q[i, h] / np.sqrt(D)
            p = np.exp(t - t.max())
            y[i, h] = p @ vv / p.sum()
            dt = (D + 2) * U * (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(D)
            bound[i, h] = np.abs(vv).max() * (2 * dt + 128 * U)
    return y, bound


def check_attention(pool, kept, q, got, width=None):
    row = 0
    for s, (p, f) in enumerate(zip(pool.past, pool.fresh)):
        want, bound = attention(q[row:row + f].astype(np.float64), kept[s], p, pool.H, pool.KV, pool.D)
        y = got[row:row + f].reshape(f, pool.H, pool.D)
        err = np.abs(y - want)
        assert (err <= bound).all(), (s, float((err / bound).max()))
        row += f


SHAPES = [
    # past, fresh, H, KV, D, page
    ([0], [1], 1, 1, 64, 16),                          # the very first token
    ([299], [1], 12, 12, 64, 16),
    ([0], [17], 2, 2, 64, 16),                         # one row past a tile
    ([15, 16, 17, 31, 0], [1, 1, 1, 1, 1], 2, 1, 64, 16),  # around the page's end
    ([63, 64, 65, 127, 128, 129], [1] * 6, 4, 2, 128, 64),
    ([1000, 3, 0, 517], [1, 0, 33, 5], 6, 2, 64, 32),  # a sequence that waits, a prompt, chunks
    ([5, 100], [70, 1], 25, 5, 80, 32),                # odd heads
    ([40, 2], [3, 9], 3, 1, 33, 16),                   # rows that are no whole vectors
    ([20], [4], 2, 2, 1, 16),
    ([20], [4], 2, 2, 127, 16),
    ([77, 0], [2, 18], 8, 1, 24, 128),
    ([3000], [1], 2, 2, 128, 256),                     # keys cut into parts
    ([2049, 700], [9, 20], 16, 1, 64, 64),             # cut, several tiles
    # From here on: many rows of a sequence, which share tiles of keys.
    ([0], [64], 1, 1, 64, 16),
    ([0], [130], 2, 2, 128, 16),
    ([17, 300, 5], [127, 129, 2], 2, 2, 64, 16),
    ([3001], [70], 2, 1, 128, 32),                     # cut
    ([2000, 63], [66, 1], 3, 3, 64, 64),               # cut, with rows past the last tile's
    ([7], [65], 3, 1, 33, 16),
    ([90], [70], 2, 2, 127, 16),
    ([20], [80], 1, 1, 1, 16),
    ([33], [41], 10, 2, 72, 32),
    ([0], [100], 4, 2, 24, 128),
    ([70, 2100], [150, 66], 2, 2, 96, 32),             # and heads of 65 .. 96, cut
    ([11], [97], 6, 2, 65, 16),
    ([260], [70], 5, 5, 95, 64),
    ([0, 500], [64, 90], 4, 1, 88, 16),
    ([500], [64], 2, 2, 97, 16),
]


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention(rt, case, dtype):
    past, fresh, H, KV, D, page = SHAPES[case]
    pool = Pool(rt, past, fresh, H, KV, D, page, dtype, seed=case)
    kept = pool.fill([p + f for p, f in zip(past, fresh)])
    pool.set()
    N = sum(fresh)
    q = pool.normal(N, H, D)
    tq, out = rt.from_numpy(q.reshape(N, -1)), rt.empty((N, H * D))
    pool.plan.attention(0, tq, out)
    got = rt.to_numpy(out)
    pool.free()
    check_attention(pool, kept, q, got)
    rt.free(tq)
    rt.free(out)


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("past, fresh", [([40, 3], [90, 9]), ([2000, 0], [70, 30])])
def test_prompts_under_a_plan_of_single_tokens(rt, dtype, past, fresh):
    pool = Pool(rt, past, fresh, 3, 3, 64, 32, dtype, seed=9)
    kept = pool.fill([p + f for p, f in zip(past, fresh)])
    plan = gptc.PagedPlan(rt, pool.cache, 3, 100, 100, 2100)
    plan.set(past, fresh, pool.table)
    q = pool.normal(sum(fresh), 3, 64)
    tq, out = rt.from_numpy(q.reshape(sum(fresh), -1)), rt.empty((sum(fresh), 192))
    plan.attention(0, tq, out)
    check_attention(pool, kept, q, rt.to_numpy(out))
    plan.free()
    pool.free()


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
def test_attention_is_the_same_every_time_and_in_the_qkv_layout(rt, dtype):
    pool = Pool(rt, [2500, 31], [3, 40], 6, 2, 64, 16, dtype, seed=5)
    kept = pool.fill([2503, 71])
    pool.set()
    q = pool.normal(43, 6, 64)
    wide = np.concatenate([q.reshape(43, -1), np.full((43, 2 * 2 * 64), np.nan, np.float32)], 1)
    tq, tw, out = rt.from_numpy(q.reshape(43, -1)), rt.from_numpy(wide), rt.empty((43, 384))
    got = []
    for t in (tq, tw, tq):
        pool.plan.attention(0, t, out)
        got.append(rt.to_numpy(out))
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    check_attention(pool, kept, q, got[0])
    pool.free()
    for t in (tq, tw, out):
        rt.free(t)


def rotate(x, table, rot, interleaved):
    """x (n, heads, D) in 64 bits by rows of the table."""
    x = x.copy()
    cos, sin = table[:, None, :rot // 2], table[:, None, rot // 2:]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    one, two = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        x[..., 0:rot:2], x[..., 1:rot:2] = one, two
    else:
        x[..., :rot // 2], x[..., rot // 2:rot] = one, two
    return x


APPENDS = [
    # past, fresh, H, KV, D, page, rot, interleaved
    ([0], [1], 1, 1, 64, 16, 0, False),
    ([0, 15, 16, 500], [1, 1, 1, 1], 12, 12, 64, 16, 0, False),
    ([7, 0, 40], [30, 0, 2], 4, 2, 128, 32, 128, False),
    ([7, 0, 40], [30, 0, 2], 4, 2, 128, 32, 128, True),
    ([3, 90], [50, 1], 5, 1, 80, 16, 32, True),
    ([3, 90], [50, 1], 5, 1, 80, 16, 40, False),
    ([1, 2], [3, 4], 2, 1, 66, 16, 4, False),   # rot 4: pairs of two halves of two
    ([1, 2], [3, 4], 3, 3, 33, 16, 32, True),   # rows that are no whole vectors
    ([1, 2], [3, 4], 3, 3, 33, 16, 30, False),
    ([10], [5], 1, 1, 2, 16, 2, False),
    ([10], [5], 2, 1, 1, 64, 0, False),
]


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(rt, case, dtype):
    past, fresh, H, KV, D, page, rot, interleaved = APPENDS[case]
    pool = Pool(rt, past, fresh, H, KV, D, page, dtype, seed=case, max_len=600)
    pool.set()
    N, rows = sum(fresh), sum(fresh) + 2
    x = pool.normal(rows, H + 2 * KV, D)
    tx, rotary, q_out = rt.from_numpy(x.reshape(rows, -1)), None, None
    if rot:
        rotary = rt.lib.gptc_rotary_table(600, rot, 10000.0)
        q_out = rt.from_numpy(np.full((rows, H * D), 7.5, np.float32))
        table = rt.to_numpy(rotary).astype(np.float64)
        angle = np.arange(600)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
        # The nearest floats to the 64-bit values.
        assert np.abs(table - np.concatenate([np.cos(angle), np.sin(angle)], 1)).max() <= U * (1 + 1e-6)
    before = [pool.k[0].clone(), pool.v[0].clone()]
    pool.plan.append(0, tx, rotary, interleaved, q_out)
    rt.sync()
    q = rt.to_numpy(q_out) if rot else None
    row, written = 0, torch.zeros(pool.k[0].shape[0], page, dtype=torch.bool, device="cuda")
    for s, (p, f) in enumerate(zip(past, fresh)):
        if f == 0:
            continue
        mine = x[row:row + f].astype(np.float64)
        k, v = pool.held(s, p, p + f)
        want_k, want_v = mine[:, H:H + KV], mine[:, H + KV:]
        tol_k = np.zeros(())
        if rot:
            want_q = rotate(mine[:, :H], table[p:p + f], rot, interleaved)
            want_k = rotate(want_k, table[p:p + f], rot, interleaved)
            tol = tol_k = 6 * U * np.abs(mine).max()
            assert np.abs(q[row:row + f].reshape(f, H, D) - want_q).max() <= tol
        if dtype == gptc.BF16:
            tol_k = tol_k + 2.0 ** -8 * np.abs(want_k)
            want_v = torch.tensor(x[row:row + f, H + KV:]).bfloat16().double().numpy()
        assert (np.abs(k - want_k) <= tol_k).all()
        assert np.array_equal(v, want_v)
        at = pool.rows(s, p, p + f)
        written[at[0], at[1]] = True
        row += f
    # Nothing else was touched: other slots hold what they held (NaN), and so do q_out's rows past the last token.
    for now, was in zip((pool.k[0], pool.v[0]), before):
        keep = ~written[:, None, :, None].expand_as(now)
        assert torch.isnan(now[keep]).all() and torch.isnan(was).all()
    if rot:
        assert (q[N:] == 7.5).all()
        rt.free(rotary)
        rt.free(q_out)
    rt.free(tx)
    pool.free()


def test_rows_past_the_last_token_are_left_as_they_were(rt):
    pool = Pool(rt, [40, 9], [2, 1], 2, 2, 64, 16, gptc.F32)
    kept = pool.fill([42, 10])
    pool.set()
    q = pool.normal(8, 2, 64)
    tq, out = rt.from_numpy(q.reshape(8, -1)), rt.from_numpy(np.full((8, 128), 7.5, np.float32))
    pool.plan.attention(0, tq, out)
    got = rt.to_numpy(out)
    assert (got[3:] == 7.5).all()
    check_attention(pool, kept, q, got)
    pool.free()


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
def test_tensors_off_16_bytes(rt, dtype):
    """The step's tensors start anywhere a float can."""
    H, KV, D, past, fresh = 4, 2, 64, 40, 90
    pool = Pool(rt, [past], [fresh], H, KV, D, 16, dtype, seed=12, max_len=200)
    kept = pool.fill([past])
    pool.set()
    x = pool.normal(fresh, H + 2 * KV, D)
    table = rt.lib.gptc_rotary_table(200, 32, 10000.0)
    turned = rotate(x[:, :H + KV].astype(np.float64), rt.to_numpy(table)[past:past + fresh].astype(np.float64), 32, False)

    def off(a):
        t = torch.zeros(a.size + 3, device="cuda")
        t[3:] = torch.tensor(a.reshape(-1))
        view = gptc.Tensor()
        view.t = ctypes.cast(t.data_ptr() + 12, ctypes.POINTER(ctypes.c_float))
        view.ndims, view.length, view.device = 2, a.size, gptc.CUDA
        view.shape[0], view.shape[1] = len(a), a.size // len(a)
        return t, ctypes.pointer(view)

    (_, tx), (q, tq), (out, tout) = off(x), off(np.zeros((fresh, H * D), np.float32)), off(np.zeros((fresh, H * D), np.float32))
    torch.cuda.synchronize()
    pool.plan.append(0, tx, table, False, tq)
    pool.plan.attention(0, tq, tout)
    rt.sync()
    got_q = q[3:].cpu().numpy().reshape(fresh, H, D)
    assert np.abs(got_q - turned[:, :H]).max() <= 6 * U * np.abs(x).max()
    held = pool.held(0, past, past + fresh)
    kv = [(np.concatenate([kept[0][0], held[0]]), np.concatenate([kept[0][1], held[1]]))]
    check_attention(pool, kv, got_q.reshape(fresh, H, D), out[3:].cpu().numpy().reshape(fresh, H * D))
    assert np.abs(held[0] - turned[:, H:]).max() <= 6 * U * np.abs(x).max() + (2.0 ** -8 * np.abs(turned).max() if dtype else 0)
    pool.free()
    rt.free(table)


def test_a_step_without_tokens_does_nothing(rt):
    pool = Pool(rt, [40, 0], [0, 0], 2, 2, 64, 16, gptc.F32)
    pool.set()
    x, q, out = rt.from_numpy(pool.normal(1, 6 * 64)), rt.from_numpy(pool.normal(1, 128)), rt.from_numpy(np.full((1, 128), 7.5, np.float32))
    pool.plan.append(0, x)
    pool.plan.attention(0, q, out)
    assert (rt.to_numpy(out) == 7.5).all()
    assert torch.isnan(pool.k[0]).all()
    pool.plan.set([], [], np.zeros((0, 1), np.int32))
    pool.plan.attention(0, q, out)
    assert (rt.to_numpy(out) == 7.5).all()
    pool.free()


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
def test_large_scores_and_far_positions(rt, dtype):
    """Scores of some hundreds: all weight on one key, others underflow to nothing; no infinities on the way."""
    pool = Pool(rt, [700], [3], 2, 2, 64, 16, dtype, seed=9)
    kept = pool.fill([703], std=6.0)
    pool.set()
    q = 6 * pool.normal(3, 2, 64)
    tq, out = rt.from_numpy(q.reshape(3, -1)), rt.empty((3, 128))
    pool.plan.attention(0, tq, out)
    got = rt.to_numpy(out)
    assert np.isfinite(got).all()
    check_attention(pool, kept, q, got)
    pool.free()


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("H, KV, D", [(1, 1, 64), (4, 2, 128), (3, 1, 40), (2, 2, 33)])
@pytest.mark.parametrize("fresh", [20, 150])
def test_a_later_tokens_values_stay_hidden(rt, dtype, fresh, H, KV, D):
    """NaN and infinities in the keys and values of some new tokens: rows before them are what they are without, and
    rows that see a value that is not finite are not finite in its place alone."""
    pool = Pool(rt, [45], [fresh], H, KV, D, 16, dtype, seed=fresh)
    kept = pool.fill([45 + fresh])
    pool.set()
    q = pool.normal(fresh, H, D)
    tq, out = rt.from_numpy(q.reshape(fresh, -1)), rt.empty((fresh, H * D))
    bad = [(fresh // 3, D - 1, float("nan")), (fresh // 2, 3, float("inf")), (fresh - 2, 0, float("-inf"))]
    for i, d, x in bad:
        page, slot = pool.rows(0, 45 + i, 46 + i)
        pool.v[0][page[0], :, slot[0], d] = x
    # A key that is no number: for its own row and the rows after it everything is lost.
    page, slot = pool.rows(0, 45 + fresh - 1, 45 + fresh)
    pool.k[0][page[0], :, slot[0], 0] = float("nan")
    torch.cuda.synchronize()
    pool.plan.attention(0, tq, out)
    got = rt.to_numpy(out).reshape(fresh, H, D)
    want, bound = attention(q.astype(np.float64), kept[0], 45, H, KV, D)
    for i in range(fresh):
        if i == fresh - 1:
            assert np.isnan(got[i]).all()
            continue
        seen = {d for j, d, _ in bad if j <= i}
        fine = [d for d in range(D) if d not in seen]
        assert (np.abs(got[i][:, fine] - want[i][:, fine]) <= bound[i]).all(), i
        for d in seen:
            assert not np.isfinite(got[i][:, d]).any(), (i, d)
    pool.free()
    rt.free(tq)
    rt.free(out)


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16])
@pytest.mark.parametrize("past, fresh, bad", [(300, 1, (64, 96)), (6000, 1, (1024, 2048)), (400, 70, (32, 64)),
                                              (200, 130, (200, 210)), (40000, 3, (20000, 20600))])
def test_keys_that_are_nan_are_not_lost(rt, dtype, past, fresh, bad):
    """Whole rounds, waves and parts whose keys' scores are NaN: every row that attends to them is NaN."""
    pool = Pool(rt, [past], [fresh], 2, 2, 32, 32, dtype, seed=4)
    pool.fill([past + fresh])
    page, slot = pool.rows(0, *bad)
    pool.k[0][page, :, slot] = float("nan")
    torch.cuda.synchronize()
    pool.set()
    out = rt.empty((fresh, 64))
    pool.plan.attention(0, rt.from_numpy(pool.normal(fresh, 64)), out)
    got = rt.to_numpy(out)
    sees = past + np.arange(fresh) >= bad[0]
    assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()
    pool.free()


def test_two_layers_and_shared_prefix(rt):
    """Two sequences read the same first pages; each layer has its own."""
    pool = Pool(rt, [64, 64], [1, 2], 4, 4, 64, 32, gptc.F32, layers=2, seed=4)
    kept = [pool.fill([65, 66], layer=i) for i in range(2)]
    pool.table[1, :2] = pool.table[0, :2]
    pool.set()
    q = pool.normal(3, 4, 64)
    tq, out = rt.from_numpy(q.reshape(3, -1)), rt.empty((3, 256))
    for i in range(2):
        k, v = kept[i][1]
        k0, v0 = kept[i][0]
        kept[i][1] = np.concatenate([k0[:64], k[64:]]), np.concatenate([v0[:64], v[64:]])
        pool.plan.attention(i, tq, out)
        check_attention(pool, kept[i], q, rt.to_numpy(out))
    pool.free()


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
def test_matches_the_frameworks_causal_forward(rt, dtype):
    """A prompt in chunks and then single tokens: every row is that of the causal forward over the whole sequence."""
    T, H, D = 130, 4, 64
    C = H * D
    pool = Pool(rt, [0], [T], H, H, D, 16, dtype, max_len=T)
    x = pool.normal(T, 3 * C)
    ref = x.copy()
    if dtype == gptc.BF16:
        ref[:, C:] = torch.tensor(x[:, C:]).bfloat16().float().numpy()
    layer = gptc.AttentionLayer(rt, C, H, T)
    layer.to(gptc.CUDA)
    yt = layer.forward(rt.from_numpy(ref.reshape(1, T, 3 * C)))
    want = rt.to_numpy(yt)[0]
    rt.free(yt)
    layer.free()
    at, got = 0, []
    for n in (1, 50, 16, 61, 1, 1):
        pool.plan.set([at], [n], pool.table)
        tx, out = rt.from_numpy(x[at:at + n]), rt.empty((n, C))
        pool.plan.append(0, tx)
        pool.plan.attention(0, tx, out)
        got.append(rt.to_numpy(out))
        rt.free(tx)
        rt.free(out)
        at += n
    assert at == T
    # Two fp32 evaluations of the same rows: 2 (2 dt + 128 u) max|v| with |t| terms of this size.
    kv = ref[:, C:].reshape(T, 2, H, D).astype(np.float64)
    _, bound = attention(x[:, :C].reshape(T, H, D).astype(np.float64), (kv[:, 0], kv[:, 1]), 0, H, H, D)
    err = np.abs(np.concatenate(got) - want).reshape(T, H, D)
    assert (err <= 2 * bound).all(), float((err / bound).max())
    pool.free()


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("H, KV, D", [(1, 1, 64), (4, 2, 128), (3, 1, 40), (2, 2, 33), (2, 2, 80)])
@pytest.mark.parametrize("fresh", [20, 150])
def test_a_later_tokens_largest_values_stay_hidden(rt, dtype, fresh, H, KV, D):
    """Values at the end of the pages' range (of fp32 also the least that is rounded to infinity as bf16, and the one
    before it), and keys of that size: rows before them are what they are without."""
    pool = Pool(rt, [45], [fresh], H, KV, D, 16, dtype, seed=fresh + D)
    kept = pool.fill([45 + fresh])
    pool.set()
    q = pool.normal(fresh, H, D)
    tq, out = rt.from_numpy(q.reshape(fresh, -1)), rt.empty((fresh, H * D))
    most = float(torch.finfo(pool.tdtype).max)
    over, under = (float(np.array([b], np.uint32).view(np.float32)[0]) for b in (0x7f7f8000, 0x7f7f7fff))
    bad = [(fresh // 3, D - 1, most), (fresh // 2, 3, -most), (fresh // 2 + 1, 4, -over), (fresh - 2, 5, over),
           (fresh - 1, 0, under)]
    for i, d, x in bad:
        page, slot = pool.rows(0, 45 + i, 46 + i)
        pool.v[0][page[0], :, slot[0], d] = x if dtype == gptc.F32 else np.copysign(most, x)
    page, slot = pool.rows(0, 45 + fresh - 1, 45 + fresh)
    pool.k[0][page[0], :, slot[0], 1] = most
    torch.cuda.synchronize()
    pool.plan.attention(0, tq, out)
    got = rt.to_numpy(out).reshape(fresh, H, D)
    want, bound = attention(q.astype(np.float64), kept[0], 45, H, KV, D)
    for i in range(fresh - 1):
        fine = [d for d in range(D) if d not in {d for j, d, _ in bad if j <= i}]
        assert (np.abs(got[i][:, fine] - want[i][:, fine]) <= bound[i]).all(), i
    pool.free()
    rt.free(tq)
    rt.free(out)
