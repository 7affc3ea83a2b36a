"""Paged steps as a server runs them (include/paged.h): a GPT-2 over pages with sequences that come, grow in chunks and
generate side by side; steps in captured graphs; several plans over one pool; a pool past 32 bits of offsets.
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
from generation import kv_generate
from test_capture_gpu import Graph
from test_generate_gpu import c3_params, check, make_model
from test_paged_gpu import Pool, attention, check_attention
from test_sample_gpu import SETTINGS, draw, language

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Server:
    """A GPT-2 whose steps run over pages: any number of new tokens of each sequence, logits of each one's last."""

    def __init__(self, rt, params, V, L, H, C, page, dtype=gptc.F32, seqs=4, room=64, max_len=64):
        self.rt, self.H, self.C, self.V = rt, H, C, V
        self.wte, self.wpe = params[0], params[1]
        self.t = [rt.from_numpy(p) for p in params]
        self.layers = [self.t[2 + 12 * i:14 + 12 * i] for i in range(L)]
        self.pages = seqs * (max_len // page + 1)
        self.cache = gptc.PagedCache(rt, L, self.pages, page, H, C // H, dtype)
        self.plan = gptc.PagedPlan(rt, self.cache, H, seqs, room, max_len)
        self.page, self.free_pages, self.tables = page, list(np.random.default_rng(1).permutation(self.pages)), {}

    def norm(self, W, b, x):
        n = x.contents.shape[0]
        y, mean, rstd = self.rt.empty((n, self.C)), self.rt.empty((n,)), self.rt.empty((n,))
        self.rt.lib.layer_norm_forward_cuda_kernel(W, b, x, 1e-5, (gptc.TensorP * 3)(mean, rstd, x), y)
        self.rt.free(mean)
        self.rt.free(rstd)
        return y

    def linear(self, W, b, x, width):
        y = self.rt.empty((x.contents.shape[0], width))
        self.rt.lib.linear_forward_cuda_kernel(W, b, x, y)
        return y

    def step(self, work):
        """work: {sequence: (tokens before, new ids)}; the logits tensor (sequences, 1, V) of their last tokens."""
        rt, lib, C = self.rt, self.rt.lib, self.C
        seqs = list(work)
        past, fresh = [work[s][0] for s in seqs], [len(work[s][1]) for s in seqs]
        for s, p, f in zip(seqs, past, fresh):
            mine = self.tables.setdefault(s, [])
            while len(mine) * self.page < p + f:
                mine.append(self.free_pages.pop())
        table = np.zeros((len(seqs), max(len(self.tables[s]) for s in seqs)), np.int32)
        for i, s in enumerate(seqs):
            table[i, :len(self.tables[s])] = self.tables[s]
        self.plan.set(past, fresh, table)
        x = rt.from_numpy(np.concatenate([self.wte[work[s][1]] + self.wpe[p:p + f] for s, p, f in zip(seqs, past, fresh)]))
        for i, (w1, b1, wqkv, bqkv, wo, bo, w2, b2, wfc, bfc, wp, bp) in enumerate(self.layers):
            h = self.norm(w1, b1, x)
            qkv, a, x2, f, x3 = self.linear(wqkv, bqkv, h, 3 * C), *(rt.empty(s) for s in [(sum(fresh), C)] * 2 + [(sum(fresh), 4 * C), (sum(fresh), C)])
            self.plan.append(i, qkv)
            self.plan.attention(i, qkv, a)
            lib.gptc_linear_forward_add_cuda(wo, bo, a, x, x2)
            h2 = self.norm(w2, b2, x2)
            g = self.linear(wfc, bfc, h2, 4 * C)
            lib.gelu_forward_cuda_kernel(g, f)
            lib.gptc_linear_forward_add_cuda(wp, bp, f, x2, x3)
            for t in (x, h, qkv, a, x2, h2, g, f):
                rt.free(t)
            x = x3
        last = rt.from_numpy(rt.to_numpy(x)[np.cumsum(fresh) - 1])
        h = self.norm(self.t[-2], self.t[-1], last)
        logits = rt.empty((len(seqs), 1, self.V))
        lib.linear_forward_cuda_kernel(self.t[0], None, h, logits)
        for t in (x, last, h):
            rt.free(t)
        return logits

    def free(self):
        self.rt.sync()
        self.plan.free()
        self.cache.free()
        for t in self.t:
            self.rt.free(t)


@pytest.mark.parametrize("C, H, page", [(64, 4, 16), (128, 2, 32)])
def test_generation_over_pages_is_the_caches(rt, C, H, page):
    """Three users: one prompt whole, one in chunks, one that starts later; greedy tokens and every step's logits are
    those of the one-token steps over contiguous caches."""
    V, L, T = 211, 2, 48
    params = c3_params(V, 64, L, C, 5, std=0.1, jitter=0.05)
    model = make_model(rt, params, V, 64, L, H, C)
    rng = np.random.default_rng(C)
    prompts = [rng.integers(0, V, n) for n in (5, 30, 9)]
    want = [kv_generate(rt, model, p, T, 64, keep_logits=True) for p in prompts]
    server = Server(rt, params, V, L, H, C, page)
    tokens, done, steps = [list(map(int, p)) for p in prompts], [0, 0, 0], 0
    params_t, u = rt.from_numpy(np.zeros(4, np.float32)), rt.from_numpy(np.zeros(3, np.float32))
    while min(len(t) for t in tokens) < T:
        work = {}
        for s in range(3):
            if (s == 2 and steps < 4) or len(tokens[s]) >= T:
                continue
            left = len(tokens[s]) - done[s]
            work[s] = (done[s], np.array(tokens[s][done[s]:done[s] + (min(left, 11) if s == 1 else left)]))
        logits = server.step(work)
        ids, coin = rt.empty((len(work),)), rt.from_numpy(np.zeros(len(work), np.float32))
        rt.lib.gptc_sample_cuda(logits, params_t, coin, ids, None)
        got, rows = rt.to_numpy(ids), rt.to_numpy(logits)[:, 0]
        for i, s in enumerate(work):
            done[s] += len(work[s][1])
            if done[s] == len(tokens[s]):
                check(f"logits of sequence {s} at {done[s]}", rows[i], want[s][1][done[s] - len(prompts[s])])
                tokens[s].append(int(got[i]))
        for t in (logits, ids, coin):
            rt.free(t)
        steps += 1
    for s in range(3):
        assert tokens[s] == list(want[s][0]), s
    rt.free(params_t)
    rt.free(u)
    server.free()
    model.free()


def test_sampled_generation_draws_what_the_logits_say(rt):
    V, L, H, C = 503, 2, 2, 64
    params = c3_params(V, 64, L, C, 6, std=0.2, jitter=0.05)
    server = Server(rt, params, V, L, H, C, 16, dtype=gptc.BF16)
    rng = np.random.default_rng(3)
    settings = np.array([SETTINGS["top_k"], SETTINGS["top_p"], SETTINGS["all"]], np.float32)
    tokens, done = [list(rng.integers(0, V, n)) for n in (3, 20, 1)], [0, 0, 0]
    ps = rt.from_numpy(settings)
    for _ in range(20):
        work = {s: (done[s], np.array(tokens[s][done[s]:])) for s in range(3)}
        logits = server.step(work)
        coin = rng.random(3).astype(np.float32)
        u, ids = rt.from_numpy(coin), rt.empty((3,))
        rt.lib.gptc_sample_cuda(logits, ps, u, ids, None)
        got = rt.to_numpy(ids)
        want, _ = draw(rt.to_numpy(logits)[:, 0], settings.astype(np.float64), coin.astype(np.float64))
        assert np.array_equal(got, want)
        for s in range(3):
            done[s] = len(tokens[s])
            tokens[s].append(int(got[s]))
        for t in (logits, u, ids):
            rt.free(t)
    rt.free(ps)
    server.free()


def as_tensor(rt, x):
    t = gptc.Tensor()
    t.t, t.ndims, t.length, t.device = ctypes.cast(x.data_ptr(), ctypes.POINTER(ctypes.c_float)), x.dim(), x.numel(), gptc.CUDA
    for i, n in enumerate(x.shape):
        t.shape[i] = n
    return ctypes.pointer(t)


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
def test_a_captured_step_follows_the_plan(rt, dtype):
    """One graph of append and attention, replayed for steps of other lengths than the captured one: single tokens,
    keys cut into parts, a prompt, more tokens than its tensors have rows for, nothing at all; with eager steps of
    another plan over the same pool in between.  Each replay is the eager call's result bit for bit."""
    H, KV, D, page, rows = 4, 2, 64, 16, 300
    pool = Pool(rt, [3000, 700, 40], [100, 200, 200], H, KV, D, page, dtype, seed=2, max_len=3200)
    pool.fill([3100, 900, 240])
    other = gptc.PagedPlan(rt, pool.cache, H, 3, 500, 3200)
    x = torch.tensor(pool.normal(rows, (H + 2 * KV) * D)).cuda()
    table = rt.lib.gptc_rotary_table(3200, D, 10000.0)
    q, out = (torch.zeros(rows, H * D, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    tx, tq, tout = (as_tensor(rt, v) for v in (x, q, out))
    plan = pool.plan

    def step(p):
        p.append(0, tx, table, False, tq)
        p.attention(0, tq, tout)

    plan.set([2999, 5, 0], [1, 1, 1], pool.table)
    step(plan)  # once eagerly: the kernels are loaded, and the plan has its memory
    graph = Graph(rt, lambda: step(plan))
    steps = [([2999, 699, 39], [1, 1, 1]), ([10, 20, 0], [100, 1, 199]), ([0, 0, 0], [0, 0, 0]), ([3000, 700, 40], [100, 200, 0]),
             ([5, 16, 31], [1, 0, 1]), ([3000, 0, 0], [60, 0, 0])]
    for past, fresh in steps * 2:
        n = min(sum(fresh), rows)
        start = [pool.k[0].clone(), pool.v[0].clone()]
        q.fill_(7.5)
        out.fill_(7.5)
        torch.cuda.synchronize()
        plan.set(past, fresh, pool.table)
        graph.replay()
        rt.sync()
        got = [v.clone() for v in (q, out, pool.k[0], pool.v[0])]
        for now, was in zip((pool.k[0], pool.v[0]), start):
            now.copy_(was)
        q.fill_(7.5)
        out.fill_(7.5)
        torch.cuda.synchronize()
        if sum(fresh) <= rows:
            other.set(past, fresh, pool.table)
            step(other)
            rt.sync()
            for a, b in zip(got, (q, out, pool.k[0], pool.v[0])):
                assert torch.equal(a.view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32),
                                   b.view(torch.int16 if b.dtype == torch.bfloat16 else torch.int32))
        assert (got[0][n:] == 7.5).all() and (got[1][n:] == 7.5).all()
        assert n == 0 or not (got[1][:n] == 7.5).any()
    graph.free()
    other.free()
    pool.free()
    rt.free(table)


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 30, 130])
def test_a_captured_step_with_more_tokens_than_rows(rt, dtype, rows):
    """A graph whose tensors have fewer rows than a later step has tokens serves the first of them, reads no others (they
    would be NaN) and writes nothing behind its own rows."""
    H, KV, D, page = 2, 2, 64, 16
    past, fresh = [500, 20, 3], [100, 2, 150]
    pool = Pool(rt, past, fresh, H, KV, D, page, dtype, seed=3)
    pool.fill([p + f for p, f in zip(past, fresh)])
    n = sum(fresh)
    q = torch.full((n, H * D), float("nan"), device="cuda")
    q[:rows] = torch.tensor(pool.normal(rows, H * D))
    out = torch.full((n, H * D), 7.5, device="cuda")
    whole, want = torch.nan_to_num(q), torch.empty(n, H * D, device="cuda")
    torch.cuda.synchronize()
    tq, tout = as_tensor(rt, q[:rows]), as_tensor(rt, out[:rows])
    pool.plan.set(past, [1, 0, 0], pool.table)
    pool.plan.attention(0, tq, tout)
    graph = Graph(rt, lambda: pool.plan.attention(0, tq, tout))
    out.fill_(7.5)
    torch.cuda.synchronize()
    for _ in range(2):
        pool.plan.set(past, fresh, pool.table)
        graph.replay()
        rt.sync()
        pool.plan.attention(0, as_tensor(rt, whole), as_tensor(rt, want))
        rt.sync()
        assert torch.equal(out[:rows], want[:rows]) and (out[rows:] == 7.5).all()
    graph.free()
    pool.free()


def test_captured_sampling(rt):
    rng = np.random.default_rng(4)
    rows, V = 6, 5003
    params = np.array([SETTINGS[n] for n in ("plain", "top_k", "top_p", "all", "greedy", "top_k most")], np.float32)
    x, p, u = rt.from_numpy(language(rng, rows, V)), rt.from_numpy(params), rt.from_numpy(rng.random(rows).astype(np.float32))
    ids, prob = rt.empty((rows,)), rt.empty((rows,))
    call = lambda: rt.lib.gptc_sample_cuda(x, p, u, ids, prob)  # noqa: E731
    call()
    graph = Graph(rt, call)
    for _ in range(4):
        logits, coins = language(rng, rows, V), rng.random(rows).astype(np.float32)
        for t, a in ((x, logits), (u, coins)):
            fresh = rt.from_numpy(a)
            rt.lib.tensor_copy(t, fresh)
            rt.free(fresh)
        graph.replay()
        rt.sync()
        want, share = draw(logits, params.astype(np.float64), coins.astype(np.float64))
        assert np.array_equal(rt.to_numpy(ids), want)
        assert np.abs(rt.to_numpy(prob) - share).max() <= 2.0 ** -23
        call()
        assert np.array_equal(rt.to_numpy(ids), want)
    graph.free()
    for t in (x, p, u, ids, prob):
        rt.free(t)


def test_two_plans_take_turns(rt):
    """Plans set one after the other, their calls interleaved: each keeps its own step and workspace."""
    a = Pool(rt, [5000], [3], 4, 2, 64, 32, gptc.BF16, seed=6)
    kept_a = a.fill([5003])
    b = Pool(rt, [900, 33], [80, 1], 4, 4, 64, 16, gptc.F32, seed=7)
    kept_b = b.fill([980, 34])
    a.set()
    b.set()
    qa, qb = a.normal(3, 4, 64), b.normal(81, 4, 64)
    ta, tb = rt.from_numpy(qa.reshape(3, -1)), rt.from_numpy(qb.reshape(81, -1))
    oa, ob = rt.empty((3, 256)), rt.empty((81, 256))
    for _ in range(3):
        a.plan.attention(0, ta, oa)
        b.plan.attention(0, tb, ob)
    check_attention(a, kept_a, qa, rt.to_numpy(oa))
    check_attention(b, kept_b, qb, rt.to_numpy(ob))
    a.free()
    b.free()


def test_a_plan_is_set_again_while_its_steps_are_queued(rt):
    """Five steps without waiting: each uses the plan as it was set before it."""
    pool = Pool(rt, [600, 600], [4, 4], 2, 2, 64, 16, gptc.F32, seed=8, room=8)
    kept = pool.fill([604, 604])
    q = pool.normal(8, 2, 64)
    tq = rt.from_numpy(q.reshape(8, -1))
    steps = [([600, 599], [1, 1]), ([10, 500], [4, 0]), ([0, 17], [1, 4]), ([600, 600], [4, 4]), ([3, 4], [0, 2])]
    outs = [rt.empty((8, 128)) for _ in steps]
    for (past, fresh), out in zip(steps, outs):
        pool.plan.set(past, fresh, pool.table)
        pool.plan.attention(0, tq, out)
    for (past, fresh), out in zip(steps, outs):
        got, row = rt.to_numpy(out), 0
        for s, (p, f) in enumerate(zip(past, fresh)):
            want, bound = attention(q[row:row + f].astype(np.float64), kept[s], p, 2, 2, 64)
            assert (np.abs(got[row:row + f].reshape(f, 2, 64) - want) <= bound).all()
            row += f
        rt.free(out)
    pool.free()


@pytest.mark.parametrize("dtype, page", [(gptc.F32, 64), (gptc.BF16, 16)], ids=["f32", "bf16"])
def test_pool_past_32_bits(rt, dtype, page):
    """A sequence in the last pages of a pool of 2.3e9 values a block."""
    KV, D, H, past, fresh = 8, 128, 8, 150, 3
    pages = 2_250_000 // page
    tdtype = torch.float32 if dtype == gptc.F32 else torch.bfloat16
    k, v = (torch.empty(pages, KV, page, D, dtype=tdtype, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    used = -(-(past + fresh) // page)
    table = np.arange(pages - 1, pages - 1 - used, -1, dtype=np.int32)[None]
    rng = np.random.default_rng(9)
    x = rng.standard_normal((past + fresh, H + 2 * KV, D)).astype(np.float32)
    torch.cuda.synchronize()
    cache = gptc.PagedCache(rt, 1, pages, page, KV, D, dtype, [k.data_ptr()], [v.data_ptr()])
    plan = gptc.PagedPlan(rt, cache, H, 1, past + fresh, past + fresh)
    out = rt.empty((fresh, H * D))
    for lo, hi in ((0, past), (past, past + fresh)):
        plan.set([lo], [hi - lo], table)
        tx = rt.from_numpy(x[lo:hi].reshape(hi - lo, -1))
        plan.append(0, tx)
        if lo:
            plan.attention(0, tx, out)
        rt.sync()
        rt.free(tx)
    held = torch.tensor(x).to(tdtype).double().numpy()
    want, bound = attention(x[past:, :H].astype(np.float64), (held[:, H:H + KV], held[:, H + KV:]), past, H, KV, D)
    assert (np.abs(rt.to_numpy(out).reshape(fresh, H, D) - want) <= bound).all()
    rt.free(out)
    plan.free()
    cache.free()


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("past, fresh, seqs, tokens", [([40, 3], [90, 9], 100, 100), ([2000, 0], [70, 30], 128, 100),
                                                       ([0], [64], 64, 64), ([700, 5, 90], [1, 1, 1], 3, 3)])
def test_every_plan_gives_a_step_the_same_results(rt, dtype, past, fresh, seqs, tokens):
    """A prompt is cut the same way under a plan of no more tokens than sequences as under one with room for more."""
    H, KV, D = 6, 3, 64
    pool = Pool(rt, past, fresh, H, KV, D, 32, dtype, seed=9, max_len=2100)
    pool.fill([p + f for p, f in zip(past, fresh)])
    N = sum(fresh)
    tq, got = rt.from_numpy(pool.normal(N, H * D)), []
    plans = [gptc.PagedPlan(rt, pool.cache, H, seqs, n, 2100) for n in (tokens, 4096)]
    if max(fresh) == 1:
        plans.append(gptc.PagedPlan.single(rt, pool.cache, H, seqs, 2100))
    for plan in plans:
        out = rt.empty((N, H * D))
        plan.set(past, fresh, pool.table)
        plan.attention(0, tq, out)
        got.append(rt.to_numpy(out))
        rt.free(out)
        plan.free()
    for y in got[1:]:
        assert np.array_equal(y, got[0])
    pool.free()
    rt.free(tq)


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("H, KV", [(4, 2), (64, 1)], ids=["group2", "group64"])
def test_captured_single_tokens_follow_their_plan(rt, dtype, H, KV):
    """A graph under a plan of single tokens: sequences that come, go, wait and grow, cut and uncut; 64 heads on one kv
    head are rows of a wide item each.  Each replay is the eager call of a general plan bit for bit."""
    D, page, n = 64, 16, 4
    pool = Pool(rt, [3000, 700, 40, 17], [1] * n, H, KV, D, page, dtype, seed=5, max_len=3200)
    pool.fill([3001, 701, 41, 18])
    plan = gptc.PagedPlan.single(rt, pool.cache, H, n, 3200)
    x = torch.tensor(pool.normal(n, (H + 2 * KV) * D)).cuda()
    table = rt.lib.gptc_rotary_table(3200, D, 10000.0)
    q, out = (torch.zeros(n, H * D, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    tx, tq, tout = (as_tensor(rt, v) for v in (x, q, out))

    def step(p):
        p.append(0, tx, table, False, tq)
        p.attention(0, tq, tout)

    plan.set([5, 0, 0, 0], [1, 0, 0, 0], pool.table)
    step(plan)
    graph = Graph(rt, lambda: step(plan))
    steps = [([3000, 700, 40, 17], [1, 1, 1, 1]), ([0, 0, 0, 0], [1, 1, 0, 1]), ([2999, 16, 15, 0], [0, 1, 1, 1]),
             ([0, 0, 0, 0], [0, 0, 0, 0]), ([3000, 1, 1, 1], [1, 0, 0, 0])]
    for past, fresh in steps * 2:
        rows = sum(fresh)
        got = []
        for p, run in ((plan, graph.replay), (pool.plan, lambda: step(pool.plan))):
            q.fill_(7.5)
            out.fill_(7.5)
            torch.cuda.synchronize()
            p.set(past, fresh, pool.table)
            run()
            rt.sync()
            got.append((q.clone(), out.clone()))
        for a, b in zip(*got):
            assert torch.equal(a, b) and (a[rows:] == 7.5).all() and (rows == 0 or not (a[:rows] == 7.5).any())
    graph.free()
    plan.free()
    pool.free()
    rt.free(table)


def test_plans_dropped_during_a_capture(rt):
    """Their memory goes back to the library once the capture is over; the graph and other plans are as they were."""
    pool = Pool(rt, [500], [3], 8, 8, 128, 64, gptc.F32, seed=1)
    kept = pool.fill([503])
    q = pool.normal(3, 8, 128)
    tq, out = rt.from_numpy(q.reshape(3, -1)), rt.empty((3, 1024))
    pool.set()
    pool.plan.attention(0, tq, out)
    free = None
    for i in range(20):
        held = [gptc.PagedPlan(rt, pool.cache, 8, 64, 4096, 1024) for _ in range(2)]  # 85 MB each
        for plan in held:
            plan.set(pool.past, pool.fresh, pool.table)
            plan.attention(0, tq, out)

        def call():
            held.pop().free()
            held.clear()  # the finalizer
            pool.plan.attention(0, tq, out)

        graph = Graph(rt, call)
        for _ in range(2):
            rt.lib.fill_tensor_data_cuda(out, ctypes.c_float(7.0))
            graph.replay()
            check_attention(pool, kept, q, rt.to_numpy(out))
            pool.set()
        graph.free()
        rt.sync()
        if i == 1:
            free = torch.cuda.mem_get_info()[0]
    assert free - torch.cuda.mem_get_info()[0] < 2 ** 28
    pool.free()
    rt.free(tq)
    rt.free(out)


def test_plans_and_caches_that_outlive_the_runtime(rt):
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import gptc
        rt = gptc.Runtime(gptc.load())
        rt.init()
        left = [gptc.PagedCache(rt, 1, 8, 16, 2, 64) for _ in range(2)]
        left += [gptc.PagedPlan(rt, c, 2, 1, 40, 64) for c in left]
        for plan in left[2:]:
            plan.set([0], [1], [[3]])
        rt.lib.runtime_destroy(gptc.CUDA)
        left[0] = left[2] = None
        print("survived")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "survived" in r.stdout and "ERROR" not in r.stderr, r.stderr


@pytest.mark.parametrize("dtype", [gptc.F32, gptc.BF16], ids=["f32", "bf16"])
def test_a_graph_on_another_stream(rt, dtype):
    """Events order it behind its plan_set, and the next plan_set behind it: several steps without waiting on the host."""
    H, KV, D = 4, 2, 64
    pool = Pool(rt, [900, 500, 30], [1, 70, 1], H, KV, D, 32, dtype, seed=6, max_len=1000, room=40)
    kept = pool.fill([901, 570, 31])
    q = pool.normal(72, H, D)
    tq = rt.from_numpy(q.reshape(72, -1))
    steps = [([900, 500, 30], [1, 70, 1]), ([3, 0, 2], [1, 0, 1]), ([880, 520, 0], [20, 50, 2]), ([0, 0, 7], [0, 0, 1])]
    outs, graphs = [torch.full((72, H * D), 7.5, device="cuda") for _ in steps], []
    torch.cuda.synchronize()
    pool.set()
    for out in outs:
        call = lambda: pool.plan.attention(0, tq, as_tensor(rt, out))  # noqa: E731
        call()
        graphs.append(Graph(rt, call))
        rt.sync()
    mine, other = torch.cuda.ExternalStream(rt.stream()), torch.cuda.Stream()
    for out in outs:
        out.fill_(7.5)
    torch.cuda.synchronize()
    for (past, fresh), graph in zip(steps, graphs):
        pool.plan.set(past, fresh, pool.table)
        other.wait_event(mine.record_event())
        assert graph.hip.hipGraphLaunch(graph.exec, ctypes.c_void_p(other.cuda_stream)) == 0
        mine.wait_event(other.record_event())
    torch.cuda.synchronize()
    for (past, fresh), out, graph in zip(steps, outs, graphs):
        got, row = out.cpu().numpy(), 0
        for s, (p, f) in enumerate(zip(past, fresh)):
            kv = tuple(x[:p + f] for x in kept[s])
            want, bound = attention(q[row:row + f].astype(np.float64), kv, p, H, KV, D)
            assert (np.abs(got[row:row + f].reshape(f, H, D) - want) <= bound).all()
            row += f
        assert (got[row:] == 7.5).all()
        graph.free()
    pool.free()
    rt.free(tq)


def test_a_plan_freed_while_another_stream_is_captured(rt):
    """In the mode in which a capture forbids waits and frees of the process: it ends as if nothing had been."""
    pool = Pool(rt, [500], [3], 4, 2, 64, 64, gptc.F32, seed=2)
    kept = pool.fill([503])
    q = pool.normal(3, 4, 64)
    tq, out = rt.from_numpy(q.reshape(3, -1)), rt.empty((3, 256))
    plan = gptc.PagedPlan(rt, pool.cache, 4, 2, 100, 600)
    plan.set(pool.past, pool.fresh, pool.table)
    plan.attention(0, tq, out)
    x = torch.arange(1000.0, device="cuda")
    y = torch.zeros_like(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="global"):
        y.add_(x)
        plan.free()
        y.mul_(2.0)
    for _ in range(3):
        y.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, 2 * (x + 1))
    pool.set()
    pool.plan.attention(0, tq, out)
    check_attention(pool, kept, q, rt.to_numpy(out))
    pool.free()
    rt.free(tq)
    rt.free(out)
