"""Paged caches (include/paged.h) without a GPU: the refusals, which all come before any device work, and the
attention's work list, which has to name every key of every query row exactly once.
"""
import ctypes
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest
from hypothesis import given, settings
from hypothesis import strategies as st

import gptc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_c(body):
    """Library calls in a child process (errors are fatal exits): a cache over addresses that no call reaches."""
    code = textwrap.dedent(f"""
        import ctypes, sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import gptc
        import numpy as np
        rt = gptc.Runtime(gptc.load())

        def cache(layers=1, pages=8, page=16, heads=2, dim=4, dtype=gptc.F32, k=None, v=None):
            k = [4096 + 16 * i for i in range(layers)] if k is None else k
            return gptc.PagedCache(rt, layers, pages, page, heads, dim, dtype, k, k if v is None else v)

        def plan(heads=4, seqs=3, tokens=40, length=64, **kw):
            return gptc.PagedPlan(rt, cache(**kw), heads, seqs, tokens, length)

        def sched(past, fresh, dim=64, cap=4):
            a, b, items = (np.array(x, np.int32).ctypes.data_as(ctypes.POINTER(ctypes.c_int)) for x in (past, fresh, [0] * 32))
            rt.lib.gptc_paged_schedule(len(past), a, b, 4, 2, dim, gptc.F32, items, cap)

        def host(*shape):
            return rt.from_numpy(np.zeros(shape, np.float32), gptc.CPU)
    """) + textwrap.dedent(body) + "\nprint('survived')\n"
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)


REFUSALS = {
    "page not a power of two": ("cache(page=24)", "power of two"),
    "page too small": ("cache(page=8)", "power of two"),
    "page too large": ("cache(page=8192)", "power of two"),
    "no layers": ("cache(layers=0)", "at least one layer"),
    "no pages": ("cache(pages=0)", "pages of 16 tokens"),
    "slots past 31 bits": ("cache(pages=1 << 27)", "pages of 16 tokens"),
    "head size 0": ("cache(dim=0)", "Head size 0"),
    "head size 129": ("cache(dim=129)", "Head size 129"),
    "kv heads": ("cache(heads=0)", "kv heads"),
    "type": ("cache(dtype=2)", "page type 2"),
    "null pages": ("cache(k=[None], v=[4096])", "are NULL"),
    "unaligned pages": ("cache(k=[4100])", "16-byte aligned"),
    "pages without a runtime": ("gptc.PagedCache(rt, 1, 8, 16, 2, 4)", "runtime_init"),
    "heads no multiple": ("plan(heads=3)", "multiple of the cache's 2 kv heads"),
    "too many tokens for the grid": ("plan(tokens=(1 << 22) + 1)", "is too large"),
    "too many rows for the grid": ("plan(tokens=1 << 20, heads=128)", "is too large"),
    "too many items for the grid": ("gptc.PagedPlan(rt, cache(heads=64), 64, 1 << 20, 1 << 20, 64)", "is too large"),
    "schedule past": ("sched([-1], [1])", "-1 tokens"),
    "schedule rows": ("sched([0], [1 << 25])", "new ones"),
    "schedule head size": ("sched([0], [1], dim=129)", "Head size 129"),
    "schedule room": ("sched([0], [1], cap=(1 << 24) + 1)", "2^24 items"),
    "too many pages": ("plan(seqs=1 << 20, length=1 << 20)", "too many pages"),
    "no room": ("plan(seqs=0)", "Expected room"),
    "too many sequences": ("plan().set([0] * 4, [1] * 4, [[0], [1], [2], [3]])", "room for 3 sequences"),
    "negative past": ("plan().set([-1], [1], [[0]])", "-1 tokens"),
    "negative new": ("plan().set([1], [-1], [[0]])", "-1 new"),
    "too long": ("plan().set([60], [5], [[0, 1, 2, 3, 4]])", "grows to 65 tokens"),
    "sum past 31 bits": ("plan().set([2**31 - 1], [2**31 - 1], [[0]])", "grows to 4294967294 tokens"),
    "too many tokens": ("plan().set([0, 0], [20, 21], [[0, 1], [2, 3]])", "room for 40 new tokens"),
    "table too narrow": ("plan().set([16], [1], [[0]])", "needs 2 pages"),
    "page below the pool": ("plan().set([0], [1], [[-1]])", "is -1"),
    "page past the pool": ("plan().set([16], [1], [[0, 8]])", "is 8"),
    "read page past the pool": ("plan().set([16], [0], [[9]])", "is 9"),
    "two write a page": ("plan().set([3, 2], [1, 1], [[5], [5]])", "receive tokens of sequences 0 and 1"),
    "one writes a page twice": ("plan().set([0], [20], [[5, 5]])", "receive tokens of sequences 0 and 0"),
    "written and read by another": ("plan().set([3, 20], [1, 1], [[5, 0], [5, 1]])", "which sequence 1 reads"),
    "written and read by one that waits": ("plan().set([3, 10], [1, 0], [[5], [5]])", "which sequence 1 reads"),
    "written and read by itself": ("plan().set([20], [1], [[5, 5]])", "which sequence 0 reads"),
    "set without a runtime": ("plan().set([0], [1], [[0]])", "runtime_init"),
    "layer": ("plan().append(1, host(1, 32))", "0 <= layer < 1"),
    "host tensor": ("plan().append(0, host(1, 32))", "qkv to be a tensor on the GPU"),
    "host q": ("plan().attention(0, host(1, 16), host(1, 16))", "q to be a tensor on the GPU"),
    "rotary rows": ("rt.lib.gptc_rotary_table(0, 4, 1e4)", "rows >= 1"),
    "odd rotary": ("rt.lib.gptc_rotary_table(4, 3, 1e4)", "even rot"),
    "theta": ("rt.lib.gptc_rotary_table(4, 4, 0.0)", "theta > 0"),
}


@pytest.mark.parametrize("name", sorted(REFUSALS))
def test_refused(name):
    call, message = REFUSALS[name]
    r = run_c(call)
    assert r.returncode == 1 and "survived" not in r.stdout, r.stderr
    assert message in r.stderr, r.stderr


def test_shared_pages_that_are_only_read_pass_the_checks():
    """A common prefix: the refusal that ends this call is the missing device, past all the checks of pages."""
    r = run_c("plan().set([20, 17, 16], [1, 1, 0], [[5, 0], [5, 1], [5, 7]])")
    assert r.returncode == 1 and "runtime_init" in r.stderr, r.stderr


def schedule(lib, past, fresh, heads, kv, dtype, cap, dim=64):
    past, fresh = (np.ascontiguousarray(x, np.int32) for x in (past, fresh))
    items = np.zeros((cap, 8), np.int32)
    ip = ctypes.POINTER(ctypes.c_int)
    n = lib.gptc_paged_schedule(len(past), past.ctypes.data_as(ip), fresh.ctypes.data_as(ip), heads, kv, dim, dtype,
                                items.ctypes.data_as(ip), cap)
    return n, items[:max(n, 0)]


@settings(max_examples=100, deadline=None)
@given(st.lists(st.tuples(st.integers(0, 3000), st.integers(0, 300)), min_size=1, max_size=7),
       st.sampled_from([(1, 1), (12, 12), (32, 8), (25, 5), (8, 1)]), st.sampled_from([gptc.F32, gptc.BF16]),
       st.sampled_from([64, 80]))
def test_work_list_covers_every_key_once(seqs, heads, dtype, dim):
    lib = gptc.load()
    past, fresh = zip(*seqs)
    H, KV = heads
    group = H // KV
    n, items = schedule(lib, past, fresh, H, KV, dtype, 1 << 16, dim)
    assert n >= 0
    # Every cut item has its place in the workspace: one for each 16 of its rows.
    parts = [part + i for part, kind in items[:, 6:].tolist() if part >= 0 for i in range((8 if dtype == gptc.F32 else 4) if kind else 1)]
    assert sorted(parts) == list(range(len(parts)))
    seen, token = {}, 0
    for s, (p, f) in enumerate(seqs):
        for row in range(f * group):
            seen[(token, row)] = []
        token += f
    ends = {}
    token = 0
    for p, f in seqs:
        ends[token] = (p, f) if f else ends.get(token, (p, f))
        token += f
    for tok0, p, rows, row0, key0, key1, part, kind in items.tolist():
        assert ends[tok0] == (p, rows // group) and kind in (0, 1) and key0 < key1
        for row in range(row0, min(row0 + ((128 if dtype == gptc.F32 else 64) if kind else 16), rows)):
            seen[(tok0, row)].append((key0, key1))
    for (tok0, row), spans in seen.items():
        need = ends[tok0][0] + row // group + 1
        at = 0
        for a, b in sorted(spans):
            assert a == at
            at = b
        assert at >= need and sorted(spans)[-1][0] < at


def test_work_list_that_does_not_fit_says_so(lib):
    n, _ = schedule(lib, [100, 5], [200, 3], 12, 12, gptc.F32, 3)
    assert n == -1


def test_long_contexts_are_cut_and_short_ones_are_not(lib):
    n, items = schedule(lib, [100], [1], 12, 12, gptc.F32, 4096)
    assert n == 1 and items[0][6] == -1
    n, items = schedule(lib, [100000], [1], 12, 12, gptc.F32, 4096)
    assert n > 30 and (items[:, 6] >= 0).all()
    sizes = items[:, 5] - items[:, 4]
    assert sizes.max() - sizes.min() <= 64


SAMPLE_REFUSALS = {
    "host logits": ("sample(host(2, 8), host(4), host(2), host(2))", "logits to be a tensor on the GPU"),
    "null params": ("sample(gpu(2, 8), None, gpu(2), gpu(2))", "`params` (NULL)"),
    "params of some rows": ("sample(gpu(3, 8), gpu(2, 4), gpu(3), gpu(3))", "4 for each of 3 rows"),
    "random numbers": ("sample(gpu(3, 8), gpu(4), gpu(2), gpu(3))", "Expected 3 random numbers"),
    "ids": ("sample(gpu(3, 8), gpu(4), gpu(3), gpu(4))", "Expected 3 ids"),
    "shares": ("sample(gpu(3, 8), gpu(4), gpu(3), gpu(3), gpu(2))", "Expected 3 probabilities"),
    "rows": ("sample(gpu((1 << 22) + 1, 1), gpu(4), gpu(1), gpu(1))", "Fewer than 2^22 rows"),
    "rows of 2^32 threads": ("sample(gpu(1 << 22, 1), gpu(4), gpu(1), gpu(1))", "Fewer than 2^22 rows"),
    "vocabulary": ("sample(gpu(1, (1 << 24) + 1), gpu(4), gpu(1), gpu(1))", "up to 2^24 tokens"),
    "ids over the random numbers": ("sample(gpu(3, 8), gpu(4), gpu(3, at=8192), gpu(3, at=8200))", "may not overlap"),
    "ids over the logits": ("sample(gpu(3, 8, at=8192), gpu(4), gpu(3), gpu(3, at=8284))", "may not overlap"),
    "shares over the parameters": ("sample(gpu(3, 8), gpu(4, at=8192), gpu(3), gpu(3), gpu(3, at=8192))", "may not overlap"),
    "ids over the shares": ("sample(gpu(3, 8), gpu(4), gpu(3), gpu(3, at=8192), gpu(3, at=8192))", "ids and prob may not overlap"),
    "without a runtime": ("sample(gpu(3, 8), gpu(4), gpu(3), gpu(3))", "runtime_init"),
}


@pytest.mark.parametrize("name", sorted(SAMPLE_REFUSALS))
def test_sampling_refused(name):
    call, message = SAMPLE_REFUSALS[name]
    r = run_c("""
        free = [4096]

        def gpu(*shape, at=None):
            t = gptc.Tensor()
            at = free[0] if at is None else at
            free[0] = max(free[0], at + 4 * int(np.prod(shape)))
            t.t, t.ndims, t.length, t.device = ctypes.cast(at, ctypes.POINTER(ctypes.c_float)), len(shape), int(np.prod(shape)), gptc.CUDA
            for i, n in enumerate(shape):
                t.shape[i] = n
            return ctypes.pointer(t)

        def sample(logits, params, u, ids, prob=None):
            rt.lib.gptc_sample_cuda(logits, params, u, ids, prob)
    """ + "\n        " + call)
    assert r.returncode == 1 and "survived" not in r.stdout, r.stderr
    assert message in r.stderr, r.stderr


SINGLE_REFUSALS = {
    "two tokens of one": ("single().set([0, 4], [1, 2], [[0], [1]])", "Sequence 1 has 2 new tokens: the plan was made for 1"),
    "heads no multiple": ("single(heads=3)", "multiple of the cache's 2 kv heads"),
    "too many sequences": ("single().set([0] * 4, [1] * 4, [[0], [1], [2], [3]])", "room for 3 sequences"),
    "too long": ("single().set([64], [1], [[0, 1, 2, 3, 4]])", "grows to 65 tokens"),
    "single tokens pass, set without a runtime": ("single().set([0, 63, 5], [1, 1, 0], [[0, 0, 0, 0], [1, 2, 3, 4], [5, 0, 0, 0]])",
                                                  "runtime_init"),
    "a general plan of as many tokens as sequences takes prompts": (
        "plan(seqs=40, tokens=40).set([0, 4], [33, 2], [[0, 1, 2], [3, 0, 0]])", "runtime_init"),
}


@pytest.mark.parametrize("name", sorted(SINGLE_REFUSALS))
def test_plans_of_single_tokens_refuse_others(name):
    call, message = SINGLE_REFUSALS[name]
    r = run_c("""
        def single(heads=4, seqs=3, length=64):
            return gptc.PagedPlan.single(rt, cache(), heads, seqs, length)
    """ + "\n        " + call)
    assert r.returncode == 1 and "survived" not in r.stdout, r.stderr
    assert message in r.stderr, r.stderr


def test_a_cache_that_could_not_be_made_ends_quietly():
    r = run_c("""
        try:
            gptc.PagedCache(rt, 1, 8, 16, 2, 4, gptc.F32, [4096, 8192], [4096, 8192])
        except IndexError:
            pass
        try:
            gptc.PagedPlan(rt, None, 2, 1, 1, 16)
        except AttributeError:
            pass
        plan(), cache()
    """)
    assert r.returncode == 0 and "survived" in r.stdout and r.stderr == "", r.stderr


@pytest.mark.parametrize("call", [
    "set(np.array([2**32 + 5]), [1], [[0]])", "set([5], np.array([1 - 2**32]), [[0]])", "set([0], [1], np.array([[2**32]]))",
    "set([0], [1], np.array([[2**63]], np.uint64))", "set([0.5], [1], [[0]])", "set([0], [1], [[float('nan')]])",
    "set([[0]], [1], [[0]])", "set([0], [1], [[0], [1]])"])
def test_plans_take_32_bit_whole_numbers(call):
    """Nothing is cut to 32 bits on its way to the checks of the library."""
    r = run_c(f"""
        try:
            plan().{call}
        except ValueError as e:
            print("refused", e)
    """)
    assert r.returncode == 0 and "refused" in r.stdout, r.stderr


def test_plans_take_whole_numbers_of_other_types():
    r = run_c("plan().set(np.array([5, 0], np.int64), np.array([1.0, 2.0]), np.array([[5, 0], [6, 0]], np.uint8))")
    assert r.returncode == 1 and "runtime_init" in r.stderr, r.stderr
    r = run_c("plan().set([], [], np.zeros((0, 1)))")
    assert r.returncode == 1 and "runtime_init" in r.stderr, r.stderr


@pytest.mark.parametrize("main_stays", [False, True])
def test_plans_left_to_the_interpreter_end_quietly(main_stays):
    """Also where the names of the gptc module go before them, as where an extension holds on to the main module."""
    r = run_c(f"""
        kept = plan(), cache()
        if {main_stays}:
            ctypes.pythonapi.Py_IncRef(ctypes.py_object(sys.modules["__main__"]))
    """)
    assert r.returncode == 0 and "survived" in r.stdout and r.stderr == "", r.stderr
