"""gptc_gpt2_loss and gptc_gpt2_loss_backward between a forward and its backward: the forward is dropped, and the backward
refused."""
import os
import subprocess
import sys
import textwrap

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("call", ["loss", "loss_backward"])
def test_between_a_forward_and_its_backward(call):
    code = textwrap.dedent(f"""
        import sys
        sys.path.insert(0, {os.path.join(ROOT, 'gpt.c_amd')!r})
        import numpy as np
        import gptc
        rt = gptc.Runtime(gptc.load())
        rt.init()
        m = gptc.GPT2Model(rt, 8, 20, 1, 1, 8)
        m.to(gptc.CUDA)
        x, t = rt.from_numpy(np.zeros((1, 8))), rt.from_numpy(np.zeros((1, 8)))
        logits = m.forward(rt.from_numpy(np.zeros((1, 8))))
        rt.free(m.{call}(x, t))
        rt.sync()
        print("lost", flush=True)
        m.backward(logits)
        print("returned")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 1 and "lost" in r.stdout and "without a forward" in r.stderr, r.stderr
    assert "returned" not in r.stdout
