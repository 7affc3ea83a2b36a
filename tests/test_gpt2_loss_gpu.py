"""GPT2 steps without the logits (gptc_gpt2_loss, gptc_gpt2_loss_backward): lookup, blocks, loss over the vocabulary and
both gradients of the tied table together, against the CPU oracle's step and against the library's own loop with logits.

Tolerances as for that loop's parity with the oracle: 1e-4 x max(1, max|ref|) per tensor.
"""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

import gptc
from gpt2_oracle import GPT2Oracle, param_shapes

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONFIGS = [
    # V, block, layers, heads, C, B, T
    (97, 32, 2, 2, 64, 2, 32),
    (50257, 1024, 1, 12, 768, 2, 200),  # GPT-2 small's widths, one layer
    (211, 64, 3, 4, 96, 3, 40),         # T below the window, head size 24
    (1000, 16, 1, 1, 20, 1, 1),         # one token
]


def init(V, block, L, C, seed):
    rng = np.random.default_rng(seed)
    return [(rng.standard_normal(s) * (0.05 if len(s) > 1 else 0.1) + (n.endswith(("ln1.W", "ln2.W")) or n == "ln_f.W"))
            .astype(np.float32) for n, s in param_shapes(V, block, L, C)]


def model_of(rt, params, V, block, L, H, C):
    m = gptc.GPT2Model(rt, block, V, L, H, C)
    m.fast_load(params)
    m.to(gptc.CUDA)
    return m


def check(name, got, ref, rel=1e-4):
    tol = rel * max(1.0, float(np.abs(ref).max()))
    err = float(np.abs(np.asarray(got, np.float64) - ref).max())
    print(f"  {name}: max abs err {err:.3e} (tol {tol:.1e})")
    assert np.isfinite(got).all() and err <= tol, f"{name}: {err:.3e} > {tol:.1e}"


def taken(rt, t):
    a = rt.to_numpy(t)
    rt.free(t)
    return a


@pytest.mark.parametrize("V,block,L,H,C,B,T", CONFIGS)
def test_step_matches_the_oracle(rt, oracle, V, block, L, H, C, B, T):
    rng = np.random.default_rng(V)
    params = init(V, block, L, C, V)
    ids, tg = rng.integers(0, V, (B, T)), rng.integers(0, V, (B, T))
    ids[0, : T // 2] = ids[0, 0]  # a frequent token
    ref = GPT2Oracle(oracle, params, L, H)
    loss = ref.loss(ref.forward(ids), tg)
    grads = [g.copy() for g in ref.backward()]
    m = model_of(rt, params, V, block, L, H, C)
    x, t = rt.from_numpy(ids), rt.from_numpy(tg)
    check("loss alone", taken(rt, m.loss(x, t)), np.array([loss]))
    check("loss", taken(rt, m.loss_backward(x, t)), np.array([loss]))
    once = [rt.to_numpy(g) for g in m.gradients()]
    for (n, _), g, r in zip(param_shapes(V, block, L, C), once, grads):
        check(f"grad {n}", g, r)
    # Ids and targets are still the caller's; gradients add up.
    assert np.array_equal(rt.to_numpy(x), ids) and np.array_equal(rt.to_numpy(t), tg)
    rt.free(m.loss_backward(x, t))
    for (n, _), g, r in zip(param_shapes(V, block, L, C), m.gradients(), grads):
        check(f"twice {n}", rt.to_numpy(g), 2 * r)
    for y in (x, t):
        rt.free(y)
    m.free()


def test_weights_match_the_loop_with_logits(rt):
    """Weights are the upstream gradient of gpt.c's loss; a position of weight 0 may have any target."""
    V, block, L, H, C, B, T = 300, 48, 2, 4, 64, 3, 41
    rng = np.random.default_rng(8)
    params = init(V, block, L, C, 8)
    ids, tg = rng.integers(0, V, (B, T)), rng.integers(0, V, (B, T)).astype(np.float32)
    w = np.where(rng.random((B, T)) < 0.3, 0, rng.uniform(0.2, 3, (B, T))).astype(np.float32)
    m = model_of(rt, params, V, block, L, H, C)
    loss_fn = gptc.CrossEntropy(rt)
    logits = m.forward(rt.from_numpy(ids))
    z = rt.to_numpy(logits).astype(np.float64)
    rt.free(loss_fn.forward(logits, rt.from_numpy(tg)))
    rt.free(logits)
    m.backward(loss_fn.backward(rt.from_numpy(w)))
    want = [rt.to_numpy(g) for g in m.gradients()]
    losses = np.log(np.exp(z - z.max(-1, keepdims=True)).sum(-1)) + z.max(-1) - np.take_along_axis(z, tg.astype(int)[..., None], -1)[..., 0]
    loss_fn.free()
    m.free()
    m = model_of(rt, params, V, block, L, H, C)
    x, t, wt = rt.from_numpy(ids), rt.from_numpy(np.where(w == 0, -100, tg)), rt.from_numpy(w)
    check("loss", taken(rt, m.loss(x, t, wt)), np.array([(w * losses).sum() / (B * T)]))
    check("loss", taken(rt, m.loss_backward(x, t, wt)), np.array([(w * losses).sum() / (B * T)]))
    for (n, _), g, r in zip(param_shapes(V, block, L, C), m.gradients(), want):
        check(f"grad {n}", rt.to_numpy(g), r, 1e-5)
    for y in (x, t, wt):
        rt.free(y)
    m.free()


def test_training_lowers_no_precision(rt):
    """Two AdamW steps by this step and by the loop with logits: the same parameters, and the same bits every time."""
    V, block, L, H, C, B, T = 500, 64, 2, 2, 64, 4, 64
    params = init(V, block, L, C, 3)
    batches = [np.random.default_rng(k).integers(0, V, (2, B, T)) for k in range(2)]

    def train(without_logits):
        m = model_of(rt, params, V, block, L, H, C)
        opt = gptc.AdamWOptimizer(rt, m, lr=1e-3, eps=1e-4, weight_decay=0.1)
        loss_fn = gptc.CrossEntropy(rt)
        for ids, tg in batches:
            opt.zero_grad()
            x, t = rt.from_numpy(ids), rt.from_numpy(tg)
            if without_logits:
                rt.free(m.loss_backward(x, t))
                rt.free(x)
                rt.free(t)
            else:
                logits = m.forward(x)
                rt.free(loss_fn.forward(logits, t))
                rt.free(logits)
                m.backward(loss_fn.backward(rt.from_numpy(np.ones((B, T)))))
            opt.step()
        out = [rt.to_numpy(p) for p in m.parameters()]
        opt.free()
        loss_fn.free()
        m.free()
        return out
    one, two, ref = train(True), train(True), train(False)
    for (n, _), a, b, r in zip(param_shapes(V, block, L, C), one, two, ref):
        assert np.array_equal(a, b), n
        check(n, a, r, 1e-5)


@pytest.mark.parametrize("call,message", [
    ("m.loss(host, t)", "runs on the GPU"),
    ("m.loss(x, host)", "runs on the GPU"),
    ("m.loss_backward(x, t, host)", "runs on the GPU"),
    ("m.loss(x, rt.from_numpy(np.zeros(7)))", "as many targets"),
    ("m.loss_backward(x, t, rt.from_numpy(np.zeros(7)))", "as many weights"),
    ("m.loss(rt.from_numpy(np.zeros((1, 9))), rt.from_numpy(np.zeros(9)))", "block size is 8"),
    ("m.loss(rt.from_numpy(np.zeros(8)), t)", "shape (B, T)"),
    ("m.loss(None, t)", "NULL"),
])
def test_refusals(call, message):
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import numpy as np
        import gptc
        rt = gptc.Runtime(gptc.load())
        rt.init()
        m = gptc.GPT2Model(rt, 8, 20, 1, 1, 8)
        m.to(gptc.CUDA)
        x, t, host = rt.from_numpy(np.zeros((1, 8))), rt.from_numpy(np.zeros((1, 8))), rt.from_numpy(np.zeros((1, 8)), gptc.CPU)
        {call}
        print("returned")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1 and message in r.stderr and "returned" not in r.stdout, r.stderr
