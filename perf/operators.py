"""The cache operators (append, attention over a cache, attention with a shared
prefix, eviction by accumulated attention weight) as measurable cases.

Kinds of case (``case["kind"]``) and the use each stands for:

* ``append``  new keys and values written behind each sequence of a cache, its
              weights there cleared: a decode step, or a chunk of a prompt;
* ``attend``  the newest tokens' attention over their cache, with the sigmoid
              output gate of a gated layer and the accumulated weights where a
              program evicts by them;
* ``prefix``  the same where every sequence of the batch continues one prompt,
              whose keys and values are held once;
* ``evict``   each sequence cut to a budget of rows: the first ones, the latest
              ones, and those of greatest accumulated weight between them.

``own`` chooses the framework's kernels; without it the same is computed in
elementary torch operations.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a decode step of a batch: one row per sequence and head (the smallest work: latency)
        {"name": "append_step", "kind": "append", "dtype": "bf16", "B": 64, "Hkv": 2, "D": 256, "S": 1024, "T": 1,
         "lo": 100, "hi": 1000, "ragged": False, "weight": True},
        # a padded batch of prompt chunks, laid behind what the caches hold
        {"name": "append_chunk", "kind": "append", "dtype": "fp16", "B": 4, "Hkv": 8, "D": 64, "S": 16384, "T": 2048,
         "lo": 1999, "hi": 8192, "ragged": True, "weight": True},
        # one short sequence, one token: launches and latency
        {"name": "attend_short_fp32", "kind": "attend", "dtype": "fp32", "B": 1, "Hq": 4, "Hkv": 4, "D": 64, "S": 4096,
         "T": 1, "lo": 1999, "hi": 1999, "ragged": False, "gate": False, "weight": False},
        # a serving batch of a gated GQA layer, lengths as they come, weights kept for eviction
        {"name": "attend_gqa_batch", "kind": "attend", "dtype": "bf16", "B": 32, "Hq": 16, "Hkv": 2, "D": 256, "S": 8192,
         "T": 1, "lo": 1000, "hi": 8192, "ragged": False, "gate": True, "weight": True},
        # one token over the longest cache of the long-context layer
        {"name": "attend_262k", "kind": "attend", "dtype": "bf16", "B": 1, "Hq": 8, "Hkv": 8, "D": 64, "S": 262144,
         "T": 1, "lo": 262144, "hi": 262144, "ragged": False, "gate": False, "weight": False},
        # a prompt's chunk over what came before it, its weights kept
        {"name": "attend_chunk_16k", "kind": "attend", "dtype": "bf16", "B": 1, "Hq": 16, "Hkv": 2, "D": 256, "S": 16384,
         "T": 2048, "lo": 16301, "hi": 16301, "ragged": False, "gate": True, "weight": True},
        # four answers to a short question
        {"name": "prefix_short", "kind": "prefix", "dtype": "fp16", "B": 4, "Hq": 8, "Hkv": 8, "D": 64, "P": 1000, "S": 128,
         "T": 1, "lo": 1, "hi": 128, "ragged": False, "gate": False, "weight": False},
        # a batch that answers about one long document through a gated GQA layer
        {"name": "prefix_gqa_batch", "kind": "prefix", "dtype": "bf16", "B": 64, "Hq": 16, "Hkv": 2, "D": 256, "P": 16301,
         "S": 512, "T": 1, "lo": 1, "hi": 512, "ragged": False, "gate": True, "weight": True},
        # several drafted tokens at a time behind the longest shared document
        {"name": "prefix_drafts_64k", "kind": "prefix", "dtype": "bf16", "B": 32, "Hq": 8, "Hkv": 8, "D": 64, "P": 65536,
         "S": 1024, "T": 5, "lo": 5, "hi": 1024, "ragged": True, "gate": False, "weight": False},
        # one row over the budget: what a step evicts
        {"name": "evict_step", "kind": "evict", "dtype": "fp32", "B": 1, "Hkv": 4, "D": 64, "S": 1152, "lo": 1025, "hi": 1025,
         "budget": 1024, "recent": 128, "sink": 4},
        # a batch of prompts, some short, cut to a cache's budget
        {"name": "evict_prompts", "kind": "evict", "dtype": "bf16", "B": 8, "Hkv": 2, "D": 256, "S": 16384, "lo": 1999,
         "hi": 16301, "budget": 4096, "recent": 512, "sink": 4},
        # the longest prompt of the long-context layer
        {"name": "evict_262k", "kind": "evict", "dtype": "bf16", "B": 1, "Hkv": 8, "D": 64, "S": 262144, "lo": 262144,
         "hi": 262144, "budget": 16384, "recent": 1024, "sink": 64},
    ]


# ------------------------------------------------------------------- drawing
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(("append", "attend", "attend", "prefix", "prefix", "evict"))
    c = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "B": _log(rng, 1, 64),
         "Hkv": rng.choice((2, 4, 8)), "D": rng.choice((32, 64, 64, 128, 256))}
    row = c["B"] * c["Hkv"] * c["D"] * (4 if c["dtype"] == "fp32" else 2)
    most = max(64, min(262144, (1 << 29) // row))       # rows of half a gigabyte of keys
    if kind == "evict":
        c["hi"] = _log(rng, 50, most)
        c["lo"] = rng.randint(1, c["hi"])
        c["S"] = c["hi"] + rng.choice((0, 0, 127))
        c["budget"] = _log(rng, 20, max(21, c["hi"]))
        c["recent"] = rng.randint(0, c["budget"] // 4)
        c["sink"] = min(4, c["budget"] - c["recent"]) if rng.random() < 0.5 else 0
        return c
    c["T"] = 1 if rng.random() < 0.5 else _log(rng, 2, 16 if rng.random() < 0.6 else 2048)
    c["T"] = min(c["T"], most)
    c["ragged"] = rng.random() < 0.4
    c["weight"] = rng.random() < 0.5
    if kind == "append":
        c["S"] = _log(rng, max(64, c["T"]), max(64, c["T"], min(most, 16384)))
        c["lo"], c["hi"] = 0, c["S"] - c["T"]
        return c
    c["Hq"] = c["Hkv"] * rng.choice((1, 2, 4, 8))
    c["gate"] = rng.random() < 0.5
    if kind == "prefix":
        c["P"] = _log(rng, 30, 65536)
        c["hi"] = _log(rng, 1, min(most, 2048))
    else:
        c["hi"] = _log(rng, 16, most)
    c["T"] = min(c["T"], c["hi"])
    c["lo"] = rng.randint(c["T"], c["hi"])
    c["S"] = c["hi"] + rng.choice((0, 0, 1, 100))
    return c


def _cost(c):
    """Seconds at 30 TFLOP/s in 32 bits, 300 in 16 bits, and 2 TB/s."""
    w = work(c)
    return w["flops"] / (3e13 if c["dtype"] == "fp32" else 3e14) + w["bytes"] / 2e12


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        # (the plain form holds every score: at most 4 GB of them)
        scores = c["B"] * c.get("Hq", 0) * c.get("T", 0) * (c["S"] + c.get("P", 0))
        if _cost(c) <= most and scores <= 1 << 30:
            return c


# -------------------------------------------------------------------- inputs
def _lens(c):
    """Rows that each sequence holds, spread over [lo, hi]."""
    return [c["lo"] + int((c["hi"] - c["lo"]) * ((b + 1) * 0.6180339887 % 1.0) + 0.5) for b in range(c["B"])]


def _counts(c):
    """New tokens of each sequence: T, or fewer in a padded batch."""
    return [max(1, c["T"] - (b % 3) * c["T"] // 4) if c["ragged"] else c["T"] for b in range(c["B"])]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def make(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    kind, B, Hkv, S, D = case["kind"], case["B"], case["Hkv"], case["S"], case["D"]
    st = {"case": case, "k": make(B, Hkv, S, D), "v": make(B, Hkv, S, D),
          "lens": torch.tensor(_lens(case), dtype=torch.int32, device=DEV)}
    # weight gathered so far: a few keys hold most of it
    heavy = make(B, Hkv, S, dtype=torch.float32).mul_(2.0).exp_() if kind == "evict" or case["weight"] else None
    st["weight"] = heavy
    if kind == "evict":
        heavy.masked_fill_(torch.rand(B, Hkv, S, generator=g, device=DEV) < 0.05, 0.0)  # never looked at: ties
        n = min(case["budget"], S)
        st["out"] = (torch.zeros(B, Hkv, n, D, dtype=dt, device=DEV), torch.zeros(B, Hkv, n, D, dtype=dt, device=DEV),
                     torch.zeros(B, Hkv, n, device=DEV))
        return st
    T = case["T"]
    st["count"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
    if kind == "append":
        # new rows straight from their projection
        st["k_new"], st["v_new"] = (make(B, T, Hkv, D).transpose(1, 2) for _ in range(2))
        return st
    Hq = case["Hq"]
    st["q"] = make(B, T, Hq, D).transpose(1, 2)
    st["gate"] = make(B, T, Hq, D).transpose(1, 2) if case["gate"] else None
    st["out_weight"] = torch.zeros_like(heavy) if heavy is not None else None
    if kind == "prefix":
        st["k_prefix"], st["v_prefix"] = make(Hkv, case["P"], D), make(Hkv, case["P"], D)
    return st


# ---------------------------------------------------------------------- pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    if "cache" not in _modules:
        sys.path.insert(1, os.path.abspath("fused-block-sparse-attention_amd"))
        from fbsa_amd import cache
        _modules["cache"] = cache
    cache, kind = _modules["cache"], st["case"]["kind"]
    if kind == "append":
        cache.append(st["k"], st["v"], st["k_new"], st["v_new"], st["lens"], count=st["count"], weight=st["weight"])
        return [t for t in (st["k"], st["v"], st["weight"]) if t is not None]
    if kind == "evict":
        c = st["case"]
        index, lens = cache.evict(st["k"], st["v"], st["weight"], st["lens"], c["budget"], recent=c["recent"],
                                  sink=c["sink"], out=st["out"])
        return [index, lens, *st["out"]]
    kw = {"count": st["count"], "out_gate": st["gate"], "weight": st["weight"], "out_weight": st["out_weight"],
          "need_lse": True}
    if kind == "prefix":
        o, lse = cache.shared_prefix_attention(st["q"], st["k_prefix"], st["v_prefix"], st["k"], st["v"], st["lens"], **kw)
    else:
        o, lse = cache.cache_attention(st["q"], st["k"], st["v"], st["lens"], **kw)
    return [o, lse] if st["out_weight"] is None else [o, lse, st["out_weight"]]


_modules = {}


def _run_plain(st):
    case = st["case"]
    kind, S = case["kind"], case["S"]
    k, v, lens = st["k"], st["v"], st["lens"].long()
    B, Hkv, _, D = k.shape
    row = torch.arange(S, device=DEV)
    if kind == "append":
        T = case["T"]
        t = row[:T]
        at = lens.view(B, 1) + t
        ok = at < S
        if st["count"] is not None:
            ok = ok & (t < st["count"].view(B, 1))
        # places that are not written go to the last row, whose old value is put back
        at = torch.where(ok, at, S - 1).view(B, 1, T).expand(B, Hkv, T)
        last = (lens + (T if st["count"] is None else st["count"])) == S
        for x, new in ((k, st["k_new"]), (v, st["v_new"]), (st["weight"], None)):
            if x is None:
                continue
            keep = x[:, :, S - 1].clone()
            if new is None:
                x.scatter_(2, at, 0.0)
                x[:, :, S - 1] = torch.where(last.view(B, 1), x[:, :, S - 1], keep)
            else:
                x.scatter_(2, at.unsqueeze(-1).expand(B, Hkv, T, D), new)
                end = new[torch.arange(B, device=DEV), :, (S - 1 - lens).clamp(0, T - 1)]
                x[:, :, S - 1] = torch.where(last.view(B, 1, 1), end, keep)
        return [x for x in (k, v, st["weight"]) if x is not None]
    if kind == "evict":
        n, budget = lens.view(B, 1, 1), min(case["budget"], S)
        key = st["weight"].masked_fill((row < case["sink"]) | ((row >= n - case["recent"]) & (row < n)), math.inf)
        key = key.masked_fill(row >= n, -1.0)
        order = key.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
        kept = torch.minimum(n, torch.full_like(n, budget))
        place = torch.arange(budget, device=DEV)
        order = order.masked_fill(place >= kept, S).sort(dim=-1).values
        live = place < kept
        index = order.masked_fill(~live, -1).int()
        src = order.clamp(max=S - 1)
        wide = src.unsqueeze(-1).expand(B, Hkv, budget, D)
        for dst, x, at in zip(st["out"], (k, v, st["weight"]), (wide, wide, src)):
            ok = live.expand(B, Hkv, budget)
            ok = ok.unsqueeze(-1) if x.dim() == 4 else ok
            dst.copy_(torch.where(ok, x.gather(2, at), dst))
        return [index, kept.view(B).int(), *st["out"]]
    q = st["q"].float()
    Hq, T = q.shape[1], q.shape[2]
    G = Hq // Hkv
    count = torch.full_like(lens, T) if st["count"] is None else st["count"].long()
    t = row.new_tensor(range(T))
    q = q.reshape(B, Hkv, G * T, D) * D ** -0.5
    seen = (lens.view(B, 1) - count.view(B, 1) + t + 1).clamp(min=0)             # rows that query t sees
    real = t < count.view(B, 1)
    seen = torch.where(real, seen, 0)
    ok = row < seen.view(B, 1, 1, T, 1)
    s = torch.matmul(q, k.float().transpose(-1, -2)).view(B, Hkv, G, T, S).masked_fill(~ok, -math.inf)
    top = s.amax(-1, keepdim=True)
    if kind == "prefix":
        qs = q.view(B, Hkv, G * T, D).transpose(0, 1).reshape(Hkv, B * G * T, D)
        sp = torch.matmul(qs, st["k_prefix"].float().transpose(-1, -2))             # (Hkv, B*G*T, P)
        sp = sp.view(Hkv, B, G, T, -1).transpose(0, 1).masked_fill(~real.view(B, 1, 1, T, 1), -math.inf)
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (s - top).exp()
    total = p.sum(-1, keepdim=True)
    acc = torch.matmul(p.view(B, Hkv, G * T, S), v.float()).view(B, Hkv, G, T, D)
    if kind == "prefix":
        pp = (sp - top).exp()
        total = total + pp.sum(-1, keepdim=True)
        pp = pp.transpose(0, 1).reshape(Hkv, B * G * T, -1)
        acc = acc + torch.matmul(pp, st["v_prefix"].float()).view(Hkv, B, G, T, D).transpose(0, 1)
    one = total.masked_fill(total == 0, 1.0)
    o = (acc / one).reshape(B, Hq, T, D)
    if st["gate"] is not None:
        o = o / (1 + (-st["gate"].float()).exp())
    out = [o.to(st["q"].dtype), (top + total.log()).reshape(B, Hq, T)]
    if st["out_weight"] is not None:
        w = st["weight"] + (p / one).sum((2, 3))
        st["out_weight"].copy_(torch.where(row < lens.view(B, 1, 1), w, st["out_weight"]))
        out.append(st["out_weight"])
    return out


# ---------------------------------------------------------------------- work
def work(case):
    """Inputs read once and outputs written once (of a cache the rows that
    sequences hold); multiply-adds of the visible (query, key) pairs."""
    kind, s, Hkv, D = case["kind"], 4 if case["dtype"] == "fp32" else 2, case["Hkv"], case["D"]
    lens = _lens(case)
    if kind == "append":
        rows = Hkv * sum(_counts(case))
        return {"bytes": 4 * rows * D * s + (4 * rows if case["weight"] else 0), "flops": 0}
    if kind == "evict":
        kept = Hkv * sum(min(n, case["budget"]) for n in lens)
        return {"bytes": 4 * kept * D * s + 4 * Hkv * sum(lens) + 12 * kept, "flops": 0}
    Hq, T, P = case["Hq"], case["T"], case.get("P", 0)
    counts = _counts(case)
    new = Hq * case["B"] * T
    pairs = Hq * sum(sum(max(0, n - c + t + 1) for t in range(c)) + c * P for n, c in zip(lens, counts))
    byt = (3 if case["gate"] else 2) * new * D * s + 4 * new + 2 * Hkv * (sum(lens) + P) * D * s
    return {"bytes": byt + (8 * Hkv * sum(lens) if case["weight"] else 0), "flops": 4 * pairs * D}


# ------------------------------------------------- the same in 64 bits (torch)
def exact(case, seed):
    st = prepare(case, seed)
    kind, Hkv, D = case["kind"], case["Hkv"], case["D"]
    lens = _lens(case)
    if kind == "append":
        k, v = st["k"].double(), st["v"].double()
        w = st["weight"].double() if case["weight"] else None
        for b, (n, c) in enumerate(zip(lens, _counts(case))):
            m = min(c, case["S"] - n)
            k[b, :, n:n + m], v[b, :, n:n + m] = st["k_new"][b, :, :m].double(), st["v_new"][b, :, :m].double()
            if w is not None:
                w[b, :, n:n + m] = 0
        return [x for x in (k, v, w) if x is not None]
    if kind == "evict":
        k, v, w = (x.double() for x in st["out"])
        index = torch.full(w.shape, -1, dtype=torch.int32, device=DEV)
        for b, n in enumerate(lens):
            for h in range(Hkv):
                rows = list(range(n))
                if n > case["budget"]:
                    sink, tail = case["sink"], n - case["recent"]
                    mid = st["weight"][b, h, sink:tail].tolist()
                    best = sorted(range(len(mid)), key=lambda i: (-mid[i], i))
                    best = best[:case["budget"] - sink - case["recent"]]
                    rows = list(range(sink)) + sorted(i + sink for i in best) + list(range(tail, n))
                r, m = torch.tensor(rows, device=DEV), len(rows)
                index[b, h, :m] = r.int()
                k[b, h, :m], v[b, h, :m], w[b, h, :m] = (st[x][b, h, r].double() for x in ("k", "v", "weight"))
        kept = torch.tensor([min(n, case["budget"]) for n in lens], dtype=torch.int32, device=DEV)
        return [index, kept, k, v, w]
    B, Hq, T = case["B"], case["Hq"], case["T"]
    G = Hq // Hkv
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=DEV)
    out_w = st["out_weight"].double() if case["weight"] else None
    for h in range(Hkv):
        if kind == "prefix":
            kp, vp = st["k_prefix"][h].double(), st["v_prefix"][h].double()
        for b, (n, c) in enumerate(zip(lens, _counts(case))):
            kb, vb = st["k"][b, h, :n].double(), st["v"][b, h, :n].double()
            place = n - c + torch.arange(c, device=DEV)
            if kind == "prefix":
                kb, vb = torch.cat([kp, kb]), torch.cat([vp, vb])
                place = place + case["P"]
            hide = torch.arange(kb.shape[0], device=DEV) > place.view(c, 1)
            if out_w is not None:
                out_w[b, h, :n] = st["weight"][b, h, :n].double()
            for g in range(h * G, h * G + G):
                x = (st["q"][b, g, :c].double() @ kb.t()).div_(math.sqrt(D)).masked_fill_(hide, -math.inf)
                lse[b, g, :c] = x.logsumexp(-1)
                pr = x.sub_(lse[b, g, :c].unsqueeze(-1)).exp_()
                o[b, g, :c] = pr @ vb
                if out_w is not None:
                    out_w[b, h, :n] += pr.sum(0)[-n:]
    if case["gate"]:
        o *= st["gate"].double().sigmoid()
    return [o, lse] if out_w is None else [o, lse, out_w]
