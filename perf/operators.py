"""Workloads of the token and attention operators, with their plain forms.

Three operators that stand beside the segment reductions:

* ``embedding(tokens, weight, scale, padding_idx)``: rows of a table by token, scaled, and
  the gradient of the table, a sum of gradient rows per token;
* ``clip_grads(grads, max_norm, out)``: the 2-norm over many gradient tensors and their
  copies scaled down to it;
* ``segment_attention(q, k, v, data, ...)``: softmax attention within the segments of a
  ``ScatterData`` (voxels of a region, documents packed into one batch).

``run`` computes a case in elementary torch operations on 32-bit values, or through the
package where ``own`` is true; ``exact`` states the same results in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_DEV = "cuda"


def listed():
    return [
        # one decoding step of 64 sequences: a lookup of 64 rows, all latency
        dict(name="embed_decode", op="embedding", tokens=64, vocab=32768, dim=1024, dtype="bf16", train=False,
             zipf=True, scale=1.0, pad=0.0),
        # a training micro-batch of text (frequent tokens dominate, a tenth is padding), table rows scaled by sqrt(dim)
        dict(name="embed_train", op="embedding", tokens=16384, vocab=32768, dim=1024, dtype="bf16", train=True,
             zipf=True, scale=32.0, pad=0.1),
        # learned features per voxel id: uniform ids, a width that no vector load divides, 32-bit values
        dict(name="embed_odd", op="embedding", tokens=9973, vocab=50021, dim=515, dtype="fp32", train=True,
             zipf=False, scale=1.0, pad=0.0),
        # a large batch on a large table, wide rows
        dict(name="embed_large", op="embedding", tokens=131072, vocab=131072, dim=4096, dtype="bf16", train=True,
             zipf=True, scale=1.0, pad=0.02),
        # the gradients of a small point encoder (widths 16 to 128 and their biases)
        dict(name="clip_encoder", op="clip", tensors=12, total=60_000, dtype="fp32", out="fp32", factor=0.5),
        # a model of a hundred million parameters in 16 bits, odd sizes among them
        dict(name="clip_model", op="clip", tensors=60, total=100_000_007, dtype="bf16", out="bf16", factor=0.1),
        # a stage of a larger one: 16-bit gradients into 32-bit ones for the optimizer
        dict(name="clip_large", op="clip", tensors=48, total=400_000_000, dtype="bf16", out="fp32", factor=0.5),
        # a handful of regions at inference: latency
        dict(name="attn_few", op="attention", rows=96, longest=16, heads=8, kv_heads=8, dim=16, dtype="bf16",
             train=False, causal=False, cap=0.0, slopes=False, shuffled=True),
        # voxels of one frame grouped by region, rows in the order of the scan, a training step
        dict(name="attn_regions", op="attention", rows=20_000, longest=128, heads=8, kv_heads=8, dim=16, dtype="bf16",
             train=True, causal=False, cap=0.0, slopes=False, shuffled=True),
        # documents packed into one batch, shared key/value heads, a training step
        dict(name="attn_documents", op="attention", rows=8192, longest=2048, heads=16, kv_heads=4, dim=128,
             dtype="bf16", train=True, causal=True, cap=0.0, slopes=False, shuffled=False),
        # capped scores and a bias by distance, an odd head width and odd lengths, a training step
        dict(name="attn_capped", op="attention", rows=6007, longest=700, heads=6, kv_heads=3, dim=40, dtype="fp16",
             train=True, causal=False, cap=30.0, slopes=True, shuffled=False),
        # long prompts at once, forward only
        dict(name="attn_prompts", op="attention", rows=32_768, longest=4096, heads=8, kv_heads=2, dim=128,
             dtype="bf16", train=False, causal=True, cap=0.0, slopes=False, shuffled=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["embedding", "clip", "attention"])
    if op == "embedding":
        most = 131072 * 4096  # values of the table, and of the looked-up rows, of the largest listed case
        dim = _log_int(rng, 1, 8192)
        return dict(op=op, tokens=_log_int(rng, 1, min(262144, most // dim)),
                    vocab=_log_int(rng, 2, min(262144, most // dim)), dim=dim,
                    dtype=rng.choice(["fp32", "bf16", "bf16", "fp16"]) if dim <= 2048 else rng.choice(["bf16", "fp16"]),
                    train=rng.random() < 0.7, zipf=rng.random() < 0.7, scale=rng.choice([1.0, math.sqrt(dim)]),
                    pad=rng.choice([0.0, 0.05, 0.5]))
    if op == "clip":
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        total = _log_int(rng, 1, 200_000_000)
        return dict(op=op, tensors=min(total, _log_int(rng, 1, 60)), total=total, dtype=dtype,
                    out=rng.choice([dtype, "fp32"]), factor=rng.choice([0.01, 0.3, 1.5]))
    longest = _log_int(rng, 1, 4096)
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    # padded to the longest segment the plain form holds about 2 * rows * longest * heads scores
    most = 2 ** 30 // (longest * heads)
    return dict(op=op, rows=_log_int(rng, 1, max(1, min(32_768, most))), longest=longest, heads=heads,
                kv_heads=kv_heads, dim=rng.choice([8, 16, 24, 32, 40, 64, 64, 80, 96, 128, 128]),
                dtype=rng.choice(["bf16", "bf16", "fp16"]), train=rng.random() < 0.6, causal=rng.random() < 0.5,
                cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, shuffled=rng.random() < 0.4)


# ---- inputs -----------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 1009 + 17)
    return g


def _randn(shape, g, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device=_DEV, dtype=dtype).mul_(scale)


def _lengths(case) -> list:
    """Segment lengths by the case alone: uniform in 1 .. longest until the rows are used up."""
    rng = random.Random(case["rows"] * 7919 + case["longest"])
    left, got = case["rows"], []
    while left > 0:
        got.append(min(left, rng.randint(1, case["longest"])))
        left -= got[-1]
    return got


def _sizes(case) -> list:
    """Sizes of the gradient tensors: from vectors to matrices, spread over three decades, summing to the total."""
    rng = random.Random(case["total"] * 31 + case["tensors"])
    weight = [10.0 ** rng.uniform(-3, 0) for _ in range(case["tensors"])]
    rest = case["total"] - case["tensors"]
    sizes = [1 + int(rest * w / sum(weight)) for w in weight]
    sizes[-1] += case["total"] - sum(sizes)
    return sizes


def _embedding_inputs(case, seed):
    g, dt = _gen(seed), _TYPES[case["dtype"]]
    t, v, d = case["tokens"], case["vocab"], case["dim"]
    u = torch.rand(t, generator=g, device=_DEV, dtype=torch.float64)
    rank = (torch.pow(float(v), u) - 1).long() if case["zipf"] else (u * v).long()  # density 1 / rank, or flat
    tokens = torch.randperm(v, generator=g, device=_DEV)[rank.clamp_(0, v - 1)]
    if case["pad"]:
        tokens[torch.rand(t, generator=g, device=_DEV) < case["pad"]] = 1
    weight = _randn((v, d), g, dt, 0.02)
    grad = _randn((t, d), g, dt) if case["train"] else None
    return {"tokens": tokens, "weight": weight, "grad": grad, "scale": case["scale"],
            "padding_idx": 1 if case["pad"] else None}


def _clip_inputs(case, seed):
    g, dt = _gen(seed), _TYPES[case["dtype"]]
    grads = [_randn((n,), g, dt, 1e-3) for n in _sizes(case)]
    outs = [torch.empty(x.shape, device=_DEV, dtype=_TYPES[case["out"]]) for x in grads]
    return {"grads": grads, "outs": outs, "max_norm": case["factor"] * 1e-3 * math.sqrt(case["total"])}


def _attention_inputs(case, seed):
    g, dt = _gen(seed), _TYPES[case["dtype"]]
    lens = torch.tensor(_lengths(case), device=_DEV)
    t, h, hk, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    ids = torch.repeat_interleave(torch.arange(lens.numel(), device=_DEV), lens)
    if case["shuffled"]:
        ids = ids[torch.randperm(t, generator=g, device=_DEV)]
    q, k, v = (_randn((t, n, d), g, dt) for n in (h, hk, hk))
    grad = _randn((t, h, d), g, dt) if case["train"] else None
    slopes = torch.pow(2.0, -8.0 * torch.arange(1, h + 1, device=_DEV, dtype=torch.float32) / h) if case["slopes"] else None
    return {"q": q, "k": k, "v": v, "grad": grad, "ids": ids, "lens": lens, "slopes": slopes, "causal": case["causal"],
            "cap": case["cap"], "scale": 1.0 / math.sqrt(d), "longest": max(_lengths(case))}


_INPUTS = {"embedding": _embedding_inputs, "clip": _clip_inputs, "attention": _attention_inputs}


def prepare(case, seed):
    state = _INPUTS[case["op"]](case, seed)
    state["op"] = case["op"]
    if own and case["op"] == "attention":
        # a program groups its rows once and keeps the plan for every layer; the plain form groups them by the ids
        from torchex_b200 import ScatterData
        state["data"] = ScatterData(state["ids"], state["lens"])
    if state.get("grad") is not None:
        for name in ("weight", "q", "k", "v"):
            if name in state:
                state[name].requires_grad_(True)
    return state


# ---- the calls, and their plain forms ---------------------------------------------------


def run(state):
    return _RUN[state["op"]](state)


def _run_embedding(s):
    if own:
        from torchex_b200 import embedding
        out = embedding(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding_idx"])
        if s["grad"] is None:
            return {"out": out}
        (g_weight,) = torch.autograd.grad(out, s["weight"], s["grad"])
        return {"out": out.detach(), "g_weight": g_weight}
    weight = s["weight"].detach()
    out = (weight[s["tokens"]].float() * s["scale"]).to(weight.dtype)
    if s["grad"] is None:
        return {"out": out}
    g = s["grad"].float()
    if s["padding_idx"] is not None:
        g = g * (s["tokens"] != s["padding_idx"])[:, None]
    total = torch.zeros(weight.shape, device=weight.device, dtype=torch.float32)
    total.index_add_(0, s["tokens"], g)
    return {"out": out, "g_weight": (total * s["scale"]).to(weight.dtype)}


def _run_clip(s):
    if own:
        from torchex_b200 import clip_grads
        clipped, norm = clip_grads(s["grads"], s["max_norm"], out=s["outs"])
        return {"norm": norm, "clipped": clipped}
    norm = torch.stack([x.float().square().sum(dtype=torch.float64) for x in s["grads"]]).sum().sqrt().float()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "clipped": [o.copy_(x.float() * coef) for x, o in zip(s["grads"], s["outs"])]}


def _run_attention(s):
    if own:
        from torchex_b200 import segment_attention
        out = segment_attention(s["q"], s["k"], s["v"], s["data"], scale=s["scale"], causal=s["causal"],
                                softcap=s["cap"], slopes=s["slopes"])
    else:
        out = _plain_attention(s)
    if s["grad"] is None:
        return {"out": out}
    g_q, g_k, g_v = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])
    return {"out": out.detach(), "g_q": g_q, "g_k": g_k, "g_v": g_v}


def _plain_attention(s):
    """Attention over segments padded to the longest one."""
    q, k, v, lens, dev = s["q"], s["k"], s["v"], s["lens"], s["q"].device
    order = torch.argsort(s["ids"], stable=True)
    start = torch.cumsum(lens, 0) - lens
    rank = torch.arange(q.shape[0], device=dev) - start[s["ids"][order]]
    place = torch.empty_like(order)
    place[order] = s["ids"][order] * s["longest"] + rank  # padded place of each row
    at = torch.arange(s["longest"], device=dev)
    rows = order[(start[:, None] + at).clamp(max=q.shape[0] - 1)]  # [segment, place]: the row there
    group = q.shape[1] // k.shape[1]

    def padded(x):  # [segment, head, place, dim]
        return x.float()[rows].transpose(1, 2)

    qp, kp, vp = padded(q), padded(k).repeat_interleave(group, 1), padded(v).repeat_interleave(group, 1)
    x = torch.matmul(qp, kp.transpose(2, 3)) * s["scale"]
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * (at[:, None] - at).abs()
    hidden = (at >= lens[:, None])[:, None, None, :]
    if s["causal"]:
        hidden = hidden | (at > at[:, None])
    x = x.masked_fill(hidden, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True).detach())
    out = torch.matmul(p / p.sum(-1, keepdim=True), vp)
    return out.transpose(1, 2).reshape(-1, q.shape[1], q.shape[2])[place].to(q.dtype)


_RUN = {"embedding": _run_embedding, "clip": _run_clip, "attention": _run_attention}


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "embedding":
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        ranks = range(1, v + 1)
        if case["zipf"]:  # expected number of distinct rows among t draws of density 1 / rank
            distinct = sum(1.0 - (1.0 - math.log1p(1.0 / r) / math.log(v + 1)) ** t for r in ranks)
        else:
            distinct = v * (1.0 - (1.0 - 1.0 / v) ** t)
        moved = 8 * t + size * d * (distinct + t)
        if case["train"]:
            moved += 8 * t + size * d * (t * (1.0 - case["pad"]) + v)
        return {"bytes": moved, "flops": t * d * (3 if case["train"] else 1)}
    if case["op"] == "clip":
        out = {"fp32": 4, "bf16": 2, "fp16": 2}[case["out"]]
        return {"bytes": case["total"] * (size + out), "flops": 3 * case["total"]}
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))
    rows = case["rows"] * case["dim"] * size
    moved = rows * (2 * case["heads"] + 2 * case["kv_heads"])
    flops = 4.0 * case["dim"] * case["heads"] * pairs
    if case["train"]:
        moved += rows * (3 * case["heads"] + 4 * case["kv_heads"])
        flops *= 3.5  # the scores again, and the products for the gradients of p, v, q and k
    return {"bytes": moved, "flops": flops}


# ---- the same results in 64 bits --------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["op"]](_INPUTS[case["op"]](case, seed))


def _exact_embedding(s):
    w, tok = s["weight"].double(), s["tokens"]
    found = {"out": w.index_select(0, tok) * s["scale"]}
    if s["grad"] is not None:
        keep = torch.ones_like(tok, dtype=torch.bool) if s["padding_idx"] is None else tok != s["padding_idx"]
        at, order = torch.sort(tok[keep], stable=True)
        total = torch.zeros_like(w)
        if at.numel():
            rows, n = torch.unique_consecutive(at, return_counts=True)
            g = s["grad"][keep][order].double()
            total[rows] = torch.segment_reduce(g, "sum", lengths=n, axis=0)
        found["g_weight"] = total * s["scale"]
    return found


def _exact_clip(s):
    total = sum(float((x.double() * x.double()).sum()) for x in s["grads"])
    norm = math.sqrt(total)
    coef = min(1.0, s["max_norm"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64), "clipped": [x.double() * coef for x in s["grads"]]}


def _exact_attention(s):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out, gq, gk, gv = (torch.zeros_like(x) for x in (q, q, k, v))
    group = q.shape[1] // k.shape[1]
    order = torch.argsort(s["ids"], stable=True)
    begin = 0
    for n in s["lens"].tolist():
        rows = order[begin:begin + n]
        begin += n
        qs, ks, vs = q[rows].transpose(0, 1), k[rows].transpose(0, 1), v[rows].transpose(0, 1)
        ks, vs = ks.repeat_interleave(group, 0), vs.repeat_interleave(group, 0)
        x = torch.bmm(qs, ks.mT) * s["scale"]
        slope = 1.0  # derivative of the capped score by the score
        if s["cap"]:
            bent = torch.tanh(x / s["cap"])
            x, slope = s["cap"] * bent, 1.0 - bent * bent
        at = torch.arange(n, device=q.device)
        if s["slopes"] is not None:
            x = x - s["slopes"].double()[:, None, None] * (at[:, None] - at[None]).abs()
        if s["causal"]:
            x = torch.where(at[None] <= at[:, None], x, -math.inf)
        p = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
        o = torch.bmm(p, vs)
        out[rows] = o.transpose(0, 1)
        if s["grad"] is None:
            continue
        g = s["grad"][rows].double().transpose(0, 1)
        ds = p * (torch.bmm(g, vs.mT) - (g * o).sum(-1, keepdim=True)) * slope * s["scale"]
        gq[rows] = torch.bmm(ds, ks).transpose(0, 1)
        gk[rows] = torch.bmm(ds.mT, qs).unflatten(0, (-1, group)).sum(1).transpose(0, 1)
        gv[rows] = torch.bmm(p.mT, g).unflatten(0, (-1, group)).sum(1).transpose(0, 1)
    return {"out": out} if s["grad"] is None else {"out": out, "g_q": gq, "g_k": gk, "g_v": gv}


_EXACT = {"embedding": _exact_embedding, "clip": _exact_clip, "attention": _exact_attention}
