"""gptc_linear_cross_entropy_cuda and the scaled embedding without a GPU: their refusals, which all come before any
device work."""
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_c(body):
    """Library calls in a child process (errors are fatal exits), on tensors over addresses that no call reaches."""
    code = textwrap.dedent(f"""
        import ctypes, sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import gptc
        lib = gptc.load()
        place = [1 << 40]

        def t(*shape, device=gptc.CUDA, at=None):
            x, n = gptc.Tensor(), 1
            for i, s in enumerate(shape):
                x.shape[i] = s
                n *= s
            x.ndims, x.length, x.device = len(shape), n, device
            x.t = ctypes.cast(place[0] if at is None else at, ctypes.POINTER(ctypes.c_float))
            place[0] += 4 * n + 64
            return ctypes.pointer(x)

        def head(x=t(2, 3, 8), W=t(10, 8), targets=t(2, 3), weights=None, out=t(1), losses=None, dx=None, dW=None):
            lib.gptc_linear_cross_entropy_cuda(x, W, targets, weights, out, losses, dx, dW, 0)

        def look(W=t(10, 8), pos=None, ids=t(2, 3), out=t(2, 3, 8)):
            lib.gptc_embedding_forward_scaled_cuda(W, pos, ids, 1.0, out)

        def back(g=t(2, 3, 8), ids=t(2, 3), dW=t(10, 8), dpos=None):
            lib.gptc_embedding_backward_sorted_cuda(g, ids, 1.0, dW, dpos, 0)
    """) + textwrap.dedent(body) + "\nprint('survived')\n"
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)


REFUSALS = {
    "no x": ("head(x=None)", "`x`"),
    "no W": ("head(W=None)", "`W`"),
    "no targets": ("head(targets=None)", "`targets`"),
    "no output": ("head(out=None)", "`output`"),
    "x on the host": ("head(x=t(6, 8, device=gptc.CPU))", "x to be a tensor on the GPU"),
    "dW on the host": ("head(dW=t(10, 8, device=gptc.CPU))", "dW to be a tensor on the GPU"),
    "weights on the host": ("head(weights=t(6, device=gptc.CPU))", "weights to be a tensor on the GPU"),
    "W of three dimensions": ("head(W=t(2, 5, 8))", "(vocabulary, features)"),
    "other features": ("head(W=t(10, 9))", "last dimension to be 9"),
    "vocabulary too large": ("head(x=t(1, 1), targets=t(1), W=t(1 << 22, 1))", "up to 4194303"),
    "no vocabulary": ("head(W=t(0, 8))", "but got 0 x 8"),
    "no rows": ("head(x=t(0, 8), targets=t(0))", "at least one row"),
    "targets of another length": ("head(targets=t(7))", "Expected 6 targets"),
    "weights of another length": ("head(weights=t(5))", "Expected 6 weights"),
    "row losses of another length": ("head(losses=t(5))", "row_losses to hold 6"),
    "empty output": ("head(out=t(0))", "hold the loss"),
    "dx of another length": ("head(dx=t(6, 9))", "dx to match"),
    "dW of another length": ("head(dW=t(9, 8))", "dW to match"),
    "dx over x": ("x = t(6, 8)\nhead(x=x, targets=t(6), dx=x)", "overlap"),
    "dW over W": ("W = t(10, 8)\nhead(W=W, dW=W)", "overlap"),
    "dW over dx": ("head(dx=t(6, 8, at=1 << 41), dW=t(10, 8, at=(1 << 41) + 188))", "overlap"),
    "losses over weights": ("w = t(6)\nhead(weights=w, losses=w)", "overlap"),
    "output over targets": ("head(targets=t(6, at=1 << 41), out=t(1, at=(1 << 41) + 20))", "overlap"),
    "head without a runtime": ("head(weights=t(6), losses=t(6), dx=t(6, 8), dW=t(10, 8))", "runtime_init"),
    "no table": ("look(W=None)", "`W`"),
    "no ids": ("look(ids=None)", "`ids`"),
    "no rows to write": ("look(out=None)", "`output`"),
    "table of one dimension": ("look(W=t(80))", "(num_embeddings, embedding_dim)"),
    "table without rows": ("look(W=t(0, 8))", "0 x 8"),
    "output of another size": ("look(out=t(2, 3, 7))", "output to hold 6 x 8"),
    "ids on the host": ("look(ids=t(2, 3, device=gptc.CPU))", "ids to be a tensor on the GPU"),
    "positions of another width": ("look(pos=t(3, 7))", "(positions, 8)"),
    "too few positions": ("look(pos=t(2, 8))", "at least 3 rows of pos"),
    "output over the table": ("W = t(10, 8)\nlook(W=W, ids=t(10), out=W)", "overlap"),
    "output over positions": ("p = t(3, 8)\nlook(pos=p, ids=t(1, 3), out=p)", "overlap"),
    "lookup without a runtime": ("look(pos=t(3, 8))", "runtime_init"),
    "no gradient": ("back(g=None)", "`global_grad`"),
    "gradient of another size": ("back(g=t(2, 3, 9))", "global_grad to hold 6 x 8"),
    "no dW": ("back(dW=None)", "`dW`"),
    "dpos on the host": ("back(dpos=t(3, 8, device=gptc.CPU))", "dpos to be a tensor on the GPU"),
    "dpos too short": ("back(dpos=t(2, 8))", "at least 3 rows of dpos"),
    "dW over the gradient": ("g = t(6, 8)\nback(g=g, dW=g)", "overlap"),
    "dpos over dW": ("back(dW=t(10, 8, at=1 << 41), dpos=t(3, 8, at=(1 << 41) + 300))", "overlap"),
    "gradient without a runtime": ("back(dpos=t(3, 8))", "runtime_init"),
}


@pytest.mark.parametrize("what", REFUSALS)
def test_refusals(what):
    body, message = REFUSALS[what]
    r = run_c(body)
    assert r.returncode == 1 and "survived" not in r.stdout and message in r.stderr, r.stderr
