"""The operators of a paged serving step, as measurable cases.

A program that serves a GPT to many users at once keeps every sequence's keys and values in pages of one pool, gives
the model each step's new tokens of all sequences as one ragged batch, and draws the next tokens on the GPU:

  append     the step's new keys and values go into their sequences' pages, rotated by their positions where the model
             has rotary positions (the queries are rotated in the same pass)
  attention  the new tokens of every sequence attend to the keys in its pages, up to their own positions
  sample     a token of every row of logits from a given random number, after temperature, top-k, top-p and min-p

Keys and values lie in (pages, kv heads, page, head size) buffers of 32-bit floats or bf16; all else is 32-bit floats,
token ids included, as everywhere in this library.
"""
import ctypes
import math
import os
import random
import sys

import numpy as np
import torch

own = False


def listed():
    return [
        # One generation step of GPT-2 small for eight users: the smallest append (no rotation, learned positions).
        {"name": "append_decode_b8_h12_d64", "kind": "append", "B": 8, "mode": "decode", "past": 500, "fresh": 1,
         "H": 12, "KV": 12, "D": 64, "page": 16, "dtype": "f32", "rot": 0, "interleaved": False},
        # Four prompts of a model with shared kv heads and full rotary positions, into bf16 pages.
        {"name": "append_prompts_h32_kv8_d128", "kind": "append", "B": 4, "mode": "chunk", "past": 0, "fresh": 2048,
         "H": 32, "KV": 8, "D": 128, "page": 64, "dtype": "bf16", "rot": 128, "interleaved": False},
        # Chunks in the middle of ragged sequences; odd heads, a part of each rotated, in adjacent pairs.
        {"name": "append_chunk_h25_kv5_d80", "kind": "append", "B": 5, "mode": "chunk", "past": 700, "fresh": 300,
         "H": 25, "KV": 5, "D": 80, "page": 32, "dtype": "f32", "rot": 32, "interleaved": True},
        # GPT-2 small generating for one user.
        {"name": "attention_decode_b1_h12_d64", "kind": "attention", "B": 1, "mode": "decode", "past": 300, "fresh": 1,
         "H": 12, "KV": 12, "D": 64, "page": 16, "dtype": "f32"},
        # The same heads for 64 users with contexts of very different lengths.
        {"name": "attention_decode_b64_h12_d64", "kind": "attention", "B": 64, "mode": "decode", "past": 4000,
         "fresh": 1, "H": 12, "KV": 12, "D": 64, "page": 64, "dtype": "f32"},
        # Long contexts over shared kv heads in bf16 pages.
        {"name": "attention_decode_b16_h32_kv8_d128", "kind": "attention", "B": 16, "mode": "decode", "past": 30000,
         "fresh": 1, "H": 32, "KV": 8, "D": 128, "page": 128, "dtype": "bf16"},
        # GPT-2 small's full window as one prompt.
        {"name": "attention_prompt_t1024_h12_d64", "kind": "attention", "B": 1, "mode": "chunk", "past": 0,
         "fresh": 1024, "H": 12, "KV": 12, "D": 64, "page": 64, "dtype": "f32"},
        # A chunk of a long prompt, the earlier chunks in the pages.
        {"name": "attention_chunk_t2048_h32_kv8_d128", "kind": "attention", "B": 1, "mode": "chunk", "past": 8192,
         "fresh": 2048, "H": 32, "KV": 8, "D": 128, "page": 128, "dtype": "bf16"},
        # A chunk of one prompt beside eight generating users; odd heads and lengths.
        {"name": "attention_mixed_b9_h25_kv5_d80", "kind": "attention", "B": 9, "mode": "mixed", "past": 3001,
         "fresh": 200, "H": 25, "KV": 5, "D": 80, "page": 32, "dtype": "f32"},
        # GPT-2's vocabulary: one user, then 64 with settings of their own.
        {"name": "sample_b1_v50257", "kind": "sample", "rows": 1, "V": 50257, "mix": "top_k"},
        {"name": "sample_b64_v50257", "kind": "sample", "rows": 64, "V": 50257, "mix": "all"},
        # A large batch over a large vocabulary, top-p only.
        {"name": "sample_b256_v131072", "kind": "sample", "rows": 256, "V": 131072, "mix": "top_p"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "sample"])
    if kind == "sample":
        while True:
            rows, V = _spread(rng, 1, 512), rng.choice([50257, _spread(rng, 64, 200000)])
            if rows * V <= 256 * 131072:
                return {"kind": kind, "rows": rows, "V": V,
                        "mix": rng.choice(["plain", "top_k", "top_p", "min_p", "all", "all"])}
    while True:
        KV = rng.choice([1, 2, 4, 5, 8, 12, 16])
        H = KV * rng.choice([1, 1, 2, 3, 4, 8])
        D = rng.choice([64, 64, 128, 128, 16, 24, 32, 40, 72, 80, 96, 112])
        mode = rng.choice(["decode", "decode", "chunk", "mixed"])
        B = _spread(rng, 1, 64)
        fresh = 1 if mode == "decode" else _spread(rng, 2, 2048)
        past = rng.choice([0, _spread(rng, 1, 32000), _spread(rng, 1, 4096)])
        case = {"kind": kind, "B": B, "mode": mode, "past": past, "fresh": fresh, "H": H, "KV": KV, "D": D,
                "page": rng.choice([16, 16, 32, 64, 128, 256]), "dtype": rng.choice(["f32", "bf16"])}
        longest = past + fresh
        if B * longest * KV * D > 16 * 30000 * 8 * 128 or B * fresh * longest * H > 2048 * 10240 * 32:
            continue
        if kind == "append":
            if B * fresh * (H + 2 * KV) * D > 4 * 2048 * 48 * 128:
                continue
            rot = rng.choice([0, D, D, D // 2 // 2 * 2])
            case.update(rot=rot, interleaved=rot > 0 and rng.random() < 0.4)
        elif B * fresh * longest * H * D > 2048 * 10240 * 32 * 128:
            continue
        return case


def _lengths(case):
    """(tokens in the pages before the step, new tokens) of every sequence: ragged, and the same for every seed."""
    B, past, fresh = case["B"], case["past"], case["fresh"]
    r = random.Random(1000003 * B + 1009 * past + fresh)
    if B == 1:
        return [past], [fresh]
    before = [past] + [r.randint(past // 16, past) for _ in range(B - 1)]
    if case["mode"] == "chunk":
        new = [fresh] + [r.randint(1, fresh) for _ in range(B - 1)]
    else:
        new = [fresh] + [1] * (B - 1)
    return before, new


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_THETA = 10000.0


# ---- inputs ----

class _Draws:
    """Torch tensors on the GPU from one seed, in the order they are asked for."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=self.gen)

    def uniform(self, *shape):
        return torch.rand(shape, device="cuda", generator=self.gen)

    def whole(self, lo, hi, *shape):
        """Whole numbers of [lo, hi], held in floats."""
        return torch.randint(lo, hi + 1, shape, device="cuda", generator=self.gen).float()

    def order(self, n):
        return torch.rand(n, device="cuda", generator=self.gen).argsort()


def _rotary(rows, rot):
    """The rotary table of a model, made once: cos | sin of position * theta^(-2i/rot), formed in 64 bits."""
    at = torch.arange(rows, dtype=torch.float64)[:, None] * _THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.cat([at.cos(), at.sin()], 1).float().cuda()


def _paged_inputs(case, seed):
    """A pool of pages in the middle of its use, with the sequences' pages scattered over it."""
    d = _Draws(seed)
    before, new = _lengths(case)
    B, KV, D, page = case["B"], case["KV"], case["D"], case["page"]
    total = [p + n for p, n in zip(before, new)]
    count = [-(-t // page) for t in total]
    most, pages = max(count), sum(count) + 7
    k, v = (torch.empty(pages, KV, page, D, device="cuda", dtype=_TYPES[case["dtype"]]).normal_(generator=d.gen)
            for _ in range(2))
    ids = d.order(pages)
    first = torch.tensor(np.cumsum([0] + count[:-1]), device="cuda")
    at = torch.arange(most, device="cuda")
    table = torch.where(at < torch.tensor(count, device="cuda")[:, None], ids[(first[:, None] + at).clamp(max=pages - 1)], 0)
    width = case["H"] + 2 * KV if case["kind"] == "append" else case["H"]
    return {"case": case, "before": before, "new": new, "longest": max(total), "k": k, "v": v, "table": table,
            "past": torch.tensor(before, device="cuda"), "x": d.normal(sum(new), width * D),
            # which sequence each token is of, and its place among that sequence's new tokens
            "seq": torch.tensor(np.repeat(np.arange(B), new), device="cuda"),
            "place": torch.tensor(np.concatenate([np.arange(n) for n in new]), device="cuda")}


def _sample_inputs(case, seed):
    """Logits of a language model: probabilities fall with the rank about as its power -1.2, some tokens are banned."""
    d = _Draws(seed)
    rows, V, mix = case["rows"], case["V"], case["mix"]
    rank = d.uniform(rows, V).argsort(1).float()
    logits = -1.2 * torch.log(1.0 + rank) + d.normal(rows, V, std=0.5) + d.normal(rows, 1, std=3.0)
    logits[:, d.order(V)[:3]] = -math.inf
    temperature = 0.6 + 0.6 * d.uniform(rows)
    top_k = d.whole(1, min(100, V), rows) if mix in ("top_k", "all") else torch.zeros(rows, device="cuda")
    top_p = 0.7 + 0.29 * d.uniform(rows) if mix in ("top_p", "all") else torch.ones(rows, device="cuda")
    min_p = 0.1 * d.uniform(rows) if mix in ("min_p", "all") else torch.zeros(rows, device="cuda")
    if mix == "all":  # users who leave one or the other out, and some who want the best token
        top_k, top_p, min_p = (torch.where(d.uniform(rows) < 0.4, off, x) for x, off in ((top_k, 0.0), (top_p, 1.0), (min_p, 0.0)))
        temperature = torch.where(d.uniform(rows) < 0.1, 0.0, temperature)
    return {"case": case, "logits": logits, "params": torch.stack([temperature, top_k, top_p, min_p], 1).contiguous(),
            "u": d.uniform(rows)}


# ---- the plain forms ----

def _append(s):
    case = s["case"]
    H, KV, D, rot, page = case["H"], case["KV"], case["D"], case["rot"], case["page"]
    at = s["past"][s["seq"]] + s["place"]
    q, k, v = s["x"].view(-1, H + 2 * KV, D).split([H, KV, KV], 1)
    if rot:
        cos, sin = s["rotary"][at][:, None, :].split(rot // 2, 2)

        def turn(x):
            head, rest = x[..., :rot], x[..., rot:]
            pairs = head.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
            a, b = pairs[..., 0], pairs[..., 1]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1)
            turned = turned if case["interleaved"] else turned.transpose(-1, -2)
            return torch.cat([turned.flatten(-2), rest], -1)
        q, k = turn(q), turn(k)
    pages, slots = s["table"][s["seq"], at // page], at % page
    s["k"][pages, :, slots] = k.to(s["k"].dtype)
    s["v"][pages, :, slots] = v.to(s["v"].dtype)
    return (q.reshape(-1, H * D), s["k"], s["v"]) if rot else (s["k"], s["v"])


def _attention(s):
    case = s["case"]
    B, H, KV, D, fresh, longest = case["B"], case["H"], case["KV"], case["D"], max(s["new"]), s["longest"]
    k, v = (c[s["table"]].permute(0, 2, 1, 3, 4).reshape(B, KV, -1, D)[:, :, :longest].float() for c in (s["k"], s["v"]))
    q = torch.zeros(B, fresh, H, D, device="cuda")
    q[s["seq"], s["place"]] = s["x"].view(-1, H, D)
    q = q.view(B, fresh, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(B, KV, -1, D)
    score = (q @ k.transpose(2, 3).contiguous()).view(B, KV, fresh, H // KV, longest) / math.sqrt(D)
    last = s["past"][:, None] + torch.arange(fresh, device="cuda")
    score.masked_fill_((torch.arange(longest, device="cuda") > last[:, :, None])[:, None, :, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    y = (p.view(B, KV, -1, longest) @ v) / p.sum(-1).view(B, KV, -1, 1)
    y = y.view(B, KV, fresh, H // KV, D).permute(0, 2, 1, 3, 4)
    return y[s["seq"], s["place"]].reshape(-1, H * D)


def _sample(s):
    x, u = s["logits"], s["u"].double()[:, None]
    temperature, top_k, top_p, min_p = s["params"].double().unsqueeze(2).unbind(1)
    V = x.shape[1]
    ranked, order = x.sort(dim=1, descending=True, stable=True)
    ranked, rank = ranked.double(), torch.arange(V, device="cuda")
    greedy = temperature <= 0
    w = torch.exp((ranked - ranked[:, :1]) / torch.where(greedy, 1.0, temperature))
    keep = rank < torch.where(top_k > 0, top_k, V)
    among = torch.where(keep, w, 0.0)
    total = among.cumsum(1)
    keep &= (top_p >= 1) | (total - among < top_p * total[:, -1:]) | (rank == 0)
    keep &= w >= min_p
    keep = torch.where(greedy, rank == 0, keep)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    below = w.cumsum(1)
    ids = (below <= u * below[:, -1:]).sum(1, keepdim=True).clamp(max=V - 1)
    return ids[:, 0].float(), (w.gather(1, ids) / below[:, -1:])[:, 0].float()


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
    t = gptc.Tensor()
    t.t = ctypes.cast(x.data_ptr(), ctypes.POINTER(ctypes.c_float))
    t.ndims, t.length, t.device = x.dim(), x.numel(), gptc.CUDA
    for i, n in enumerate(x.shape):
        t.shape[i] = n
    return ctypes.pointer(t)


def _paged_calls(s):
    case, rt = s["case"], _rt()
    import gptc
    cache = gptc.PagedCache(rt, 1, s["k"].shape[0], case["page"], case["KV"], case["D"],
                            gptc.F32 if case["dtype"] == "f32" else gptc.BF16,
                            k=[s["k"].data_ptr()], v=[s["v"].data_ptr()])
    plan = gptc.PagedPlan(rt, cache, case["H"], case["B"], sum(s["new"]), s["longest"])
    plan.set(s["before"], s["new"], s["table"].cpu().numpy())
    s["plan"], x = plan, _wrap(s["x"])
    if case["kind"] == "attention":
        s["out"] = torch.empty(sum(s["new"]), case["H"] * case["D"], device="cuda")
        s["call"] = rt.lib.gptc_paged_attention_cuda, (plan.raw, 0, x, _wrap(s["out"]))
        return
    q = rotary = None
    s["out"] = s["k"], s["v"]
    if case["rot"]:
        s["q"] = torch.empty(sum(s["new"]), case["H"] * case["D"], device="cuda")
        q, rotary = _wrap(s["q"]), _wrap(s["rotary"])
        s["out"] = s["q"], s["k"], s["v"]
    s["call"] = rt.lib.gptc_paged_append_cuda, (plan.raw, 0, x, rotary, int(case["interleaved"]), q)


def _sample_calls(s):
    lib = _rt().lib
    s["out"] = torch.empty(s["case"]["rows"], device="cuda"), torch.empty(s["case"]["rows"], device="cuda")
    args = [_wrap(x) for x in (s["logits"], s["params"], s["u"], *s["out"])]
    s["call"] = lib.gptc_sample_cuda, args


def prepare(case, seed):
    if case["kind"] == "sample":
        s = _sample_inputs(case, seed)
    else:
        s = _paged_inputs(case, seed)
        if case.get("rot"):
            s["rotary"] = _rotary(s["longest"], case["rot"])
    if own:
        torch.cuda.synchronize()
        (_sample_calls if case["kind"] == "sample" else _paged_calls)(s)
    return s


def run(s):
    if own:
        call, args = s["call"]
        call(*args)
        return s["out"]
    return {"append": _append, "attention": _attention, "sample": _sample}[s["case"]["kind"]](s)


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["V"]
        # Each logit is read, scaled by its temperature, exponentiated and summed.
        return {"bytes": 4 * n + 4 * 7 * case["rows"], "flops": 4 * n}
    before, new = _lengths(case)
    N, H, KV, D, size = sum(new), case["H"], case["KV"], case["D"], 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "append":
        rot = case["rot"]
        moved = N * 2 * KV * D * (4 + size) + (N * H * D * 8 + N * rot * 4 if rot else 0)
        return {"bytes": moved, "flops": N * (H + KV) * rot * 3}
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(before, new))
    return {"bytes": 2 * sum(before + new) * KV * D * size + 8 * N * H * D, "flops": 4 * pairs * H * D}


# ---- the results in 64 bits, from the definitions ----

def _exact_append(s):
    case = s["case"]
    H, KV, D, rot, page = case["H"], case["KV"], case["D"], case["rot"], case["page"]
    k_out, v_out = s["k"].double(), s["v"].double()
    x = s["x"].double()
    q_out = x[:, :H * D].clone()
    row = 0
    for b, (p, n) in enumerate(zip(s["before"], s["new"])):
        rows = x[row:row + n].view(n, H + 2 * KV, D).clone()
        if rot:
            table = s["rotary"][p:p + n].double()
            for i in range(rot // 2):
                one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
                z = torch.complex(rows[:, :H + KV, one], rows[:, :H + KV, two])
                z = z * torch.complex(table[:, i], table[:, rot // 2 + i])[:, None]
                rows[:, :H + KV, one], rows[:, :H + KV, two] = z.real, z.imag
            q_out[row:row + n] = rows[:, :H].reshape(n, -1)
        for g in range(p // page, (p + n - 1) // page + 1):
            lo, hi = max(p, g * page), min(p + n, (g + 1) * page)
            place = s["table"][b, g]
            k_out[place, :, lo - g * page:hi - g * page] = rows[lo - p:hi - p, H:H + KV].transpose(0, 1)
            v_out[place, :, lo - g * page:hi - g * page] = rows[lo - p:hi - p, H + KV:].transpose(0, 1)
        row += n
    return (q_out, k_out, v_out) if rot else (k_out, v_out)


def _exact_attention(s):
    case = s["case"]
    H, KV, D, page = case["H"], case["KV"], case["D"], case["page"]
    out = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (p, n) in enumerate(zip(s["before"], s["new"])):
        t = p + n
        mine = s["table"][b, :-(-t // page)]
        hidden = torch.ones(n, t, dtype=torch.bool, device="cuda").triu_(p + 1)
        for h in range(H):
            g = h * KV // H
            k, v = (c[mine, g].reshape(-1, D)[:t].double() for c in (s["k"], s["v"]))
            q = s["x"][row:row + n, h * D:(h + 1) * D].double()
            a = torch.matmul(q, k.t().contiguous()).div_(math.sqrt(D)).masked_fill_(hidden, -math.inf)
            out[row:row + n, h * D:(h + 1) * D] = torch.softmax(a, 1) @ v
        row += n
    return out


def _exact_sample(s):
    logits, params, u = (s[n].cpu().numpy().astype(np.float64) for n in ("logits", "params", "u"))
    ids, probs = np.zeros(len(u)), np.ones(len(u))
    for r, (temperature, top_k, top_p, min_p) in enumerate(params):
        order = np.argsort(-logits[r], kind="stable")
        if temperature <= 0:
            ids[r] = order[0]
            continue
        if top_k > 0:
            order = order[:int(top_k)]
        w = np.exp((logits[r][order] - logits[r][order[0]]) / temperature)
        if top_p < 1:
            upto = np.cumsum(w)
            n = int(np.searchsorted(upto, top_p * upto[-1])) + 1
            order, w = order[:n], w[:n]
        order, w = order[w >= min_p], w[w >= min_p]
        byid = np.argsort(order)
        order, w = order[byid], w[byid]
        upto = np.cumsum(w)
        n = min(int(np.searchsorted(upto, u[r] * upto[-1], side="right")), len(w) - 1)
        ids[r], probs[r] = order[n], w[n] / upto[-1]
    return ids, probs


def exact(case, seed):
    s = _sample_inputs(case, seed) if case["kind"] == "sample" else _paged_inputs(case, seed)
    if case.get("rot"):
        s["rotary"] = _rotary(s["longest"], case["rot"])
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](s)
