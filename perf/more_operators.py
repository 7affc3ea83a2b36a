"""The two ends of a GPT in training, as measurable cases.

A program that trains a GPT with tied embeddings looks tokens up in one table at the start of a step and projects onto
the same table at its end.  The vocabulary is so much wider than the model that logits, their log-softmax and their
gradient are the largest tensors of a step by far; these operators keep none of them:

  head_loss  the cross entropy of softmax(x W^T) against the targets, of every row and their mean (validation)
  head_step  the mean with the gradients of x and W (training); a row may have a weight, 0 for padding
  lookup     rows of the table, scaled, with the rows of the positions added
  gather     the gradient of the lookup: what every token's rows add up to, and every position's

All values are 32-bit floats, ids and targets included, as everywhere in this library.
"""
import ctypes
import math
import os
import sys

import torch

own = False

V_GPT2 = 50257


def listed():
    return [
        # A handful of tokens of a prompt scored by GPT-2 small: the smallest call, all of it reading the table.
        {"name": "head_loss_r16_c768", "kind": "head_loss", "rows": 16, "C": 768, "V": V_GPT2, "weights": False},
        # A validation batch of GPT-2 small, 8 windows of 1024.
        {"name": "head_loss_r8192_c768", "kind": "head_loss", "rows": 8192, "C": 768, "V": V_GPT2, "weights": False},
        # A small model on a small vocabulary; no size is a multiple of any tile, and some rows are padding.
        {"name": "head_step_r333_c100_v5003", "kind": "head_step", "rows": 333, "C": 100, "V": 5003, "weights": True},
        # Fine-tuning on one short conversation.
        {"name": "head_step_r100_c768", "kind": "head_step", "rows": 100, "C": 768, "V": V_GPT2, "weights": True},
        # GPT-2 small on one window.
        {"name": "head_step_r1024_c768", "kind": "head_step", "rows": 1024, "C": 768, "V": V_GPT2, "weights": False},
        # GPT-2 XL's width, ragged rows with padding.
        {"name": "head_step_r2000_c1600", "kind": "head_step", "rows": 2000, "C": 1600, "V": V_GPT2, "weights": True},
        # GPT-2 small in training, 8 windows of 1024.
        {"name": "head_step_r8192_c768", "kind": "head_step", "rows": 8192, "C": 768, "V": V_GPT2, "weights": False},
        # The tokens of one generation step for eight users.
        {"name": "lookup_b8_t1_c768", "kind": "lookup", "B": 8, "T": 1, "C": 768, "V": V_GPT2, "positions": True,
         "scale": 1.0},
        # A training batch of a model that scales its embeddings by the root of their width.
        {"name": "lookup_b8_t1024_c768", "kind": "lookup", "B": 8, "T": 1024, "C": 768, "V": V_GPT2, "positions": True,
         "scale": math.sqrt(768.0)},
        # A small model's batch; odd width, no positions.
        {"name": "gather_b3_t333_c100", "kind": "gather", "B": 3, "T": 333, "C": 100, "V": 5003, "positions": False,
         "scale": 10.0},
        # GPT-2 small in training: the words of natural text, a few of them very frequent.
        {"name": "gather_b8_t1024_c768", "kind": "gather", "B": 8, "T": 1024, "C": 768, "V": V_GPT2,
         "positions": True, "scale": 1.0},
        # A large batch at GPT-2 XL's width.
        {"name": "gather_b64_t1024_c1600", "kind": "gather", "B": 64, "T": 1024, "C": 1600, "V": V_GPT2,
         "positions": True, "scale": 40.0},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["head_loss", "head_step", "head_step", "lookup", "gather", "gather"])
    while True:
        C = rng.choice([768, 1600, _spread(rng, 16, 2000), _spread(rng, 4, 500) * 4])
        V = rng.choice([V_GPT2, V_GPT2, _spread(rng, 100, 130000)])
        if kind.startswith("head"):
            rows = _spread(rng, 1, 16384)
            if rows * C * V <= 8192 * 768 * V_GPT2 and V * C <= 1600 * V_GPT2:
                return {"kind": kind, "rows": rows, "C": C, "V": V, "weights": rng.random() < 0.5}
        else:
            B, T = _spread(rng, 1, 64), _spread(rng, 1, 2048)
            if B * T * C <= 64 * 1024 * 1600 and V * C <= 1600 * V_GPT2:
                return {"kind": kind, "B": B, "T": T, "C": C, "V": V, "positions": rng.random() < 0.5,
                        "scale": rng.choice([1.0, math.sqrt(C), round(rng.uniform(0.1, 50.0), 3)])}


# ---- inputs ----

class _Draws:
    """Torch tensors on the GPU from one seed, in the order they are asked for."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=self.gen)

    def uniform(self, *shape):
        return torch.rand(shape, device="cuda", generator=self.gen)

    def words(self, V, *shape):
        """Ids of natural text: the n-th most frequent word about 1/n as often as the first, in scattered places."""
        order = torch.rand(V, device="cuda", generator=self.gen).argsort()
        rank = torch.exp(self.uniform(*shape).double() * math.log(V + 1.0)).long().clamp(1, V) - 1
        return order[rank].float()


def _head_inputs(case, seed):
    """The last LayerNorm's output (a few channels much larger than the rest), and a table whose logits it predicts
    some of the targets with."""
    d = _Draws(seed)
    R, C, V = case["rows"], case["C"], case["V"]
    W = d.normal(V, C, std=2.8 / math.sqrt(C))
    targets = d.words(V, R)
    mine = W[targets.long()]
    # The target's logit is between 0 and most of the others' log sum, give or take the others' spread.
    x = d.normal(R, C) + 0.7 * (math.log(V) + 2.0) * d.uniform(R, 1) * mine / mine.square().sum(1, keepdim=True)
    loud = torch.where(d.uniform(C) < 0.01, 10.0, 1.0)
    weights = torch.where(d.uniform(R) < 0.2, 0.0, 1.0) if case["weights"] else None
    return {"case": case, "x": x * loud, "W": W / loud.sqrt(), "targets": targets, "weights": weights}


def _table_inputs(case, seed):
    d = _Draws(seed)
    B, T, C, V = case["B"], case["T"], case["C"], case["V"]
    s = {"case": case, "ids": d.words(V, B, T)}
    if case["kind"] == "gather":
        s["g"] = d.normal(B, T, C, std=0.01)
    else:
        s["W"] = d.normal(V, C, std=0.02)
        s["P"] = d.normal(T, C, std=0.01) if case["positions"] else None
    return s


# ---- the plain forms ----

def _head(s):
    x, W, w, R = s["x"], s["W"], s["weights"], s["case"]["rows"]
    t = s["targets"].long()[:, None]
    if w is not None:
        x = torch.where(w[:, None] != 0, x, 0.0)
    logits = x @ W.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    losses = (total.log() + top - logits.gather(1, t))[:, 0]
    if w is not None:
        losses = torch.where(w != 0, losses, 0.0)
    loss = (losses if w is None else losses * w).double().sum().float() / R
    if s["case"]["kind"] == "head_loss":
        return loss, losses
    scale = 1.0 / R if w is None else (w / R)[:, None]
    e /= total
    e.scatter_add_(1, t, torch.full_like(top, -1.0))
    e *= scale
    return loss, e @ W, e.t() @ x


def _lookup(s):
    out = s["W"][s["ids"].long()] * s["case"]["scale"]
    return out if s["P"] is None else out + s["P"]


def _gather(s):
    case = s["case"]
    g = s["g"]
    dW = torch.zeros(case["V"], case["C"], device="cuda")
    dW.index_add_(0, s["ids"].long().flatten(), (g * case["scale"]).view(-1, case["C"]))
    return (dW, g.sum(0)) if case["positions"] else dW


# ---- the library's calls ----

_runtime = None


def _rt():
    global _runtime
    if _runtime is None:
        path = os.path.join(os.getcwd(), "gpt.c_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import gptc
        torch.cuda.init()
        _runtime = gptc.Runtime()
        _runtime.init()
    return _runtime


def _wrap(x):
    """A tensor_t over a torch tensor's memory (the torch tensor stays the owner)."""
    import gptc
    if x is None:
        return None
    t = gptc.Tensor()
    t.t = ctypes.cast(x.data_ptr(), ctypes.POINTER(ctypes.c_float))
    t.ndims, t.length, t.device = x.dim(), x.numel(), gptc.CUDA
    for i, n in enumerate(x.shape):
        t.shape[i] = n
    return ctypes.pointer(t)


def _calls(s):
    case, lib = s["case"], _rt().lib
    kind, C, V = case["kind"], case["C"], case["V"]
    if kind.startswith("head"):
        loss, losses, dx, dW = torch.empty((), device="cuda"), None, None, None
        if kind == "head_loss":
            losses = torch.empty(case["rows"], device="cuda")
            s["out"] = loss, losses
        else:
            dx, dW = torch.empty(case["rows"], C, device="cuda"), torch.empty(V, C, device="cuda")
            s["out"] = loss, dx, dW
        args = [_wrap(t) for t in (s["x"], s["W"], s["targets"], s["weights"], loss.view(1), losses, dx, dW)]
        s["call"] = lib.gptc_linear_cross_entropy_cuda, (*args, 0)
    elif kind == "lookup":
        s["out"] = torch.empty(case["B"], case["T"], C, device="cuda")
        s["call"] = lib.gptc_embedding_forward_scaled_cuda, (_wrap(s["W"]), _wrap(s["P"]), _wrap(s["ids"]), case["scale"],
                                                           _wrap(s["out"]))
    else:
        dW = torch.empty(V, C, device="cuda")
        dP = torch.empty(case["T"], C, device="cuda") if case["positions"] else None
        s["out"] = dW if dP is None else (dW, dP)
        s["call"] = lib.gptc_embedding_backward_sorted_cuda, (_wrap(s["g"]), _wrap(s["ids"]), case["scale"], _wrap(dW),
                                                              _wrap(dP), 0)


def prepare(case, seed):
    s = _head_inputs(case, seed) if case["kind"].startswith("head") else _table_inputs(case, seed)
    if own:
        torch.cuda.synchronize()
        _calls(s)
    return s


def run(s):
    if own:
        call, args = s["call"]
        call(*args)
        return s["out"]
    return {"head_loss": _head, "head_step": _head, "lookup": _lookup, "gather": _gather}[s["case"]["kind"]](s)


def work(case):
    C, V = case["C"], case["V"]
    if case["kind"].startswith("head"):
        R = case["rows"]
        inputs = R * C + V * C + R * (2 if case["weights"] else 1)
        if case["kind"] == "head_loss":
            return {"bytes": 4 * (inputs + 1 + R), "flops": 2 * R * V * C}
        return {"bytes": 4 * (inputs + 1 + R * C + V * C), "flops": 6 * R * V * C}
    n, T = case["B"] * case["T"], case["T"]
    if case["kind"] == "lookup":
        rows = int(round(V * (1 - (1 - 1 / V) ** n)))  # of the table, at most about so many
        return {"bytes": 4 * (n * C + min(n, rows) * C + n + (T * C if case["positions"] else 0)),
                "flops": n * C * (2 if case["positions"] else 1)}
    return {"bytes": 4 * (n * C + V * C + n + (T * C if case["positions"] else 0)),
            "flops": n * C * (3 if case["positions"] else 2)}


# ---- the results in 64 bits, from the definitions ----

def _exact_head(s):
    x, W, t, w = s["x"].double(), s["W"].double(), s["targets"].long(), s["weights"]
    R, V, C = s["case"]["rows"], s["case"]["V"], s["case"]["C"]
    step = s["case"]["kind"] == "head_step"
    losses = torch.zeros(R, dtype=torch.float64, device="cuda")
    loss, dx, dW = 0.0, torch.zeros(R, C, dtype=torch.float64, device="cuda"), torch.zeros(V, C, dtype=torch.float64,
                                                                                         device="cuda")
    piece = max(1, 40000000 // V)
    Wt = W.t().contiguous()
    for lo in range(0, R, piece):
        rows = torch.arange(lo, min(lo + piece, R), device="cuda")
        if w is not None:
            rows = rows[w[rows] != 0]
        if len(rows) == 0:
            continue
        factor = (torch.ones(len(rows), dtype=torch.float64, device="cuda") if w is None else w[rows].double()) / R
        logp = torch.log_softmax(torch.mm(x[rows], Wt), 1)
        at = torch.arange(len(rows), device="cuda")
        losses[rows] = -logp[at, t[rows]]
        loss = loss + (losses[rows] * factor).sum()
        if step:
            logp.exp_()
            logp[at, t[rows]] -= 1
            logp *= factor[:, None]
            dx[rows] = torch.mm(logp, W)
            dW += torch.mm(logp.t().contiguous(), x[rows])
    loss = torch.as_tensor(loss, dtype=torch.float64, device="cuda")
    return (loss, dx, dW) if step else (loss, losses)


def _exact_lookup(s):
    case = s["case"]
    out = torch.stack([s["W"].double().index_select(0, row) for row in s["ids"].long()]) * case["scale"]
    if s["P"] is not None:
        for b in range(case["B"]):
            out[b] += s["P"].double()
    return out


def _exact_gather(s):
    case = s["case"]
    C, V = case["C"], case["V"]
    ids, order = s["ids"].flatten().long().sort(stable=True)
    rows = s["g"].view(-1, C)[order].double()
    dW = torch.zeros(V, C, dtype=torch.float64, device="cuda")
    # The sum of a run is the difference of the running sums at its ends.
    end = torch.cat([ids[1:] != ids[:-1], torch.ones(1, dtype=torch.bool, device="cuda")]).nonzero()[:, 0]
    upto = rows.cumsum(0)[end]
    dW[ids[end]] = case["scale"] * torch.cat([upto[:1], upto[1:] - upto[:-1]])
    if not case["positions"]:
        return dW
    dP = torch.zeros(case["T"], C, dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        dP += s["g"][b].double()
    return dW, dP


def exact(case, seed):
    if case["kind"].startswith("head"):
        return _exact_head(_head_inputs(case, seed))
    return {"lookup": _exact_lookup, "gather": _exact_gather}[case["kind"]](_table_inputs(case, seed))
