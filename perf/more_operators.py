"""The operators of a cache held in 4 bits (rows quantised as they are written,
rows read back, attention over them) as measurable cases.

Kinds of case (``case["kind"]``) and the use each stands for:

* ``write``   new keys and values written behind each sequence, and read back as
              the cache holds them: a step's row, or a prompt's chunk whose own
              attention is to see what later tokens will see;
* ``read``    rows of long caches read back in the operands' type: what comes
              before a second prompt, for attention over whole prompts;
* ``attend``  the newest tokens' attention over their cache, with the sigmoid
              output gate of a gated layer;
* ``step``    a decode step: one row of each sequence written, then attended.

A value is held as step * code: code a 4-bit float (1 sign, 2 exponent and 1
mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), one step for 64 elements of a row (32
in the last group where the head dim is an odd multiple of 32), the group's
largest magnitude over 6 rounded to 6 significant bits.

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
        {"name": "write_step", "kind": "write", "dtype": "bf16", "B": 64, "Hkv": 2, "D": 256, "S": 1024, "T": 1,
         "lo": 100, "hi": 1000, "ragged": False},
        # a padded batch of prompt chunks behind what the caches hold
        {"name": "write_chunk", "kind": "write", "dtype": "fp16", "B": 4, "Hkv": 8, "D": 64, "S": 16384, "T": 2048,
         "lo": 1999, "hi": 8192, "ragged": True},
        # a long prompt taken in whole, in 32 bits, its head dim no power of two
        {"name": "write_prompt_fp32", "kind": "write", "dtype": "fp32", "B": 1, "Hkv": 8, "D": 96, "S": 65536, "T": 65531,
         "lo": 0, "hi": 0, "ragged": False},
        # a few short sequences read back
        {"name": "read_short_fp32", "kind": "read", "dtype": "fp32", "B": 3, "Hkv": 4, "D": 64, "S": 1024, "T": 999,
         "lo": 999, "hi": 1024, "ragged": True},
        # the longest cache of the long-context layer read back before a second prompt
        {"name": "read_262k", "kind": "read", "dtype": "bf16", "B": 1, "Hkv": 8, "D": 64, "S": 262144, "T": 262144,
         "lo": 262144, "hi": 262144, "ragged": False},
        # one short sequence, one token: launches and latency
        {"name": "attend_short_fp32", "kind": "attend", "dtype": "fp32", "B": 1, "Hq": 4, "Hkv": 4, "D": 64, "S": 4096,
         "T": 1, "lo": 1999, "hi": 1999, "ragged": False, "gate": False},
        # a serving batch of a gated GQA layer, lengths as they come
        {"name": "attend_gqa_batch", "kind": "attend", "dtype": "bf16", "B": 32, "Hq": 16, "Hkv": 2, "D": 256, "S": 8192,
         "T": 1, "lo": 1000, "hi": 8192, "ragged": False, "gate": True},
        # one token over the longest cache of the long-context layer
        {"name": "attend_262k", "kind": "attend", "dtype": "bf16", "B": 1, "Hq": 8, "Hkv": 8, "D": 64, "S": 262144,
         "T": 1, "lo": 262144, "hi": 262144, "ragged": False, "gate": False},
        # several drafted tokens at a time, padded, in fp16
        {"name": "attend_drafts_fp16", "kind": "attend", "dtype": "fp16", "B": 16, "Hq": 16, "Hkv": 2, "D": 128, "S": 32768,
         "T": 5, "lo": 1999, "hi": 32768, "ragged": True, "gate": False},
        # a prompt's chunk over what came before it
        {"name": "attend_chunk_16k", "kind": "attend", "dtype": "bf16", "B": 1, "Hq": 16, "Hkv": 2, "D": 256, "S": 16384,
         "T": 2048, "lo": 16301, "hi": 16301, "ragged": False, "gate": True},
        # the same in 32 bits, two short chunks
        {"name": "attend_chunk_fp32", "kind": "attend", "dtype": "fp32", "B": 2, "Hq": 8, "Hkv": 8, "D": 64, "S": 4096,
         "T": 509, "lo": 1999, "hi": 4000, "ragged": True, "gate": False},
        # a decode step of a batch of mid-length sequences: write, then attend
        {"name": "step_batch", "kind": "step", "dtype": "bf16", "B": 16, "Hq": 32, "Hkv": 8, "D": 128, "S": 16384, "T": 1,
         "lo": 1000, "hi": 16301, "ragged": False, "gate": False},
    ]


# ------------------------------------------------------------------- drawing
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(("write", "read", "attend", "attend", "attend", "step"))
    c = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "B": _log(rng, 1, 64),
         "Hkv": rng.choice((1, 2, 4, 8)), "D": rng.choice((32, 64, 64, 96, 128, 128, 160, 256))}
    row = c["B"] * c["Hkv"] * c["D"]
    most = max(64, min(262144, (1 << 28) // row))       # rows of 2^28 elements of keys
    if kind in ("write", "read"):
        c["T"] = 1 if kind == "write" and rng.random() < 0.3 else _log(rng, 2, min(most, 65536 if kind == "write" else most))
        c["ragged"] = c["T"] > 1 and rng.random() < 0.4
        c["S"] = c["T"] + _log(rng, 1, 1000)
        c["lo"], c["hi"] = (0, c["S"] - c["T"]) if kind == "write" else (c["T"], c["S"])
        return c
    c["T"] = 1 if kind == "step" or rng.random() < 0.5 else _log(rng, 2, 16 if rng.random() < 0.6 else 2048)
    c["T"] = min(c["T"], most)
    c["ragged"] = c["T"] > 1 and rng.random() < 0.4
    c["Hq"] = c["Hkv"] * rng.choice((1, 2, 4, 8))
    c["gate"] = rng.random() < 0.5
    c["hi"] = max(c["T"], _log(rng, 16, most))
    c["lo"] = rng.randint(c["T"], c["hi"])
    c["S"] = c["hi"] + rng.choice((0, 0, 1, 100))
    return c


def _cost(c):
    """Seconds at 30 TFLOP/s in 32 bits, 300 in 16 bits, and 1 TB/s."""
    w = work(c)
    return w["flops"] / (3e13 if c["dtype"] == "fp32" else 3e14) + w["bytes"] / 1e12


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        # (the plain form holds every score: at most 4 GB of them)
        if _cost(c) <= most and c["B"] * c.get("Hq", 0) * c["T"] * c["S"] <= 1 << 30:
            return c


# -------------------------------------------------------------------- inputs
def _groups(D):
    return (D + 63) // 64


def _lens(c):
    """Rows that each sequence holds (write: before the new ones), spread over [lo, hi]."""
    return [c["lo"] + int((c["hi"] - c["lo"]) * ((b + 1) * 0.6180339887 % 1.0) + 0.5) for b in range(c["B"])]


def _counts(c):
    """New tokens (read: rows wanted) of each sequence: T, or fewer in a padded batch."""
    return [max(1, c["T"] - (b % 3) * c["T"] // 4) if c["ragged"] else c["T"] for b in range(c["B"])]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kind, B, Hkv, S, D, T = (case[x] for x in ("kind", "B", "Hkv", "S", "D", "T"))

    def make(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    st = {"case": case, "lens": torch.tensor(_lens(case), dtype=torch.int32, device=DEV),
          "count": torch.tensor(_counts(case), dtype=torch.int32, device=DEV) if case["ragged"] else None}
    # channels of keys differ in size by a few times
    size = torch.exp(0.5 * make(Hkv, 1, D, dtype=torch.float32))
    if kind == "write":
        st["k4"], st["v4"] = (torch.zeros(B, Hkv, S, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
        st["step"] = torch.zeros(B, Hkv, S, 2, _groups(D), dtype=_step_type(dt), device=DEV)
    else:
        # rows that earlier steps wrote
        held = []
        for scaled in (True, False):
            codes = torch.empty(B, Hkv, S, D // 2, dtype=torch.uint8, device=DEV)
            steps = torch.empty(B, Hkv, S, _groups(D), dtype=_step_type(dt), device=DEV)
            for b in range(B):
                rows = make(Hkv, S, D)
                if scaled:
                    rows = (rows.float() * size).to(dt)
                codes[b], steps[b] = _quantise(rows)
            held.append((codes, steps))
        st["k4"], st["v4"], st["step"] = held[0][0], held[1][0], torch.stack((held[0][1], held[1][1]), 3)
    if kind == "read":
        st["first"] = st["lens"] - (case["T"] if st["count"] is None else st["count"])
        return st
    if kind in ("write", "step"):
        # new rows straight from their projection
        st["k_new"] = (make(B, T, Hkv, D).float() * size.view(Hkv, D)).to(dt).transpose(1, 2)
        st["v_new"] = make(B, T, Hkv, D).transpose(1, 2)
    if kind == "step":
        st["start"] = st["lens"] - 1
    if kind != "write":
        st["q"] = make(B, T, case["Hq"], D).transpose(1, 2)
        st["gate"] = make(B, T, case["Hq"], D).transpose(1, 2) if case["gate"] else None
    return st


# ---------------------------------------------------------------------- pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    if "cache4" not in _modules:
        sys.path.insert(1, os.path.abspath("fused-block-sparse-attention_amd"))
        from fbsa_amd import cache4
        _modules["cache4"] = cache4
    cache4, case = _modules["cache4"], st["case"]
    kind, held, count = case["kind"], (st["k4"], st["v4"], st["step"]), st["count"]
    if kind == "write":
        cache4.append(*held, st["k_new"], st["v_new"], st["lens"], count=count)
        return list(cache4.read(*held, st["lens"], case["T"], count=count, dtype=st["k_new"].dtype))
    if kind == "read":
        return list(cache4.read(*held, st["first"], case["T"], count=count, dtype=DTYPES[case["dtype"]]))
    if kind == "step":
        cache4.append(*held, st["k_new"], st["v_new"], st["start"])
    return list(cache4.cache_attention(st["q"], *held, st["lens"], count=count, out_gate=st["gate"], need_lse=True))


_modules = {}


def _step_type(dt):
    return torch.float16 if dt == torch.float16 else torch.bfloat16


def _quantise(x):
    """Packed codes (..., D / 2) and steps (..., groups) of rows x (..., D)."""
    D = x.shape[-1]
    half = x.dtype == torch.float16
    x = x.float()
    pad = torch.nn.functional.pad(x, (0, -D % 64)).view(*x.shape[:-1], -1, 64)
    want = pad.abs().amax(-1).double() / 6
    # unit: the last of 6 significant bits, a power of two put together from its exponent (pow may be off by a bit)
    e = torch.frexp(want).exponent.clamp(min=-17 if half else -119)
    unit = ((e.long() + (1023 - 6)) << 52).view(torch.float64)
    step = ((want / unit).round() * unit).clamp(max=10752.0 if half else 42 * 2.0 ** 120).float()
    s, a = step.unsqueeze(-1), pad.abs()
    # (ties go to the even code: borders at 0.25, 1.25, 2.5 and 5 belong to the code below, the others above)
    code = (a > 0.25 * s).to(torch.uint8)
    for border, above in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += a >= border * s if above else a > border * s
    code += (pad < 0).to(torch.uint8) * 8
    code = code.flatten(-2)[..., :D]
    return code[..., 0::2] + code[..., 1::2] * 16, step.to(torch.float16 if half else torch.bfloat16)


def _values(codes, step):
    """What packed codes (..., D / 2) and steps (..., groups) stand for, in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat((table, -table))
    pairs = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = table[pairs.int()]
    return x * step.float().repeat_interleave(64, -1)[..., :x.shape[-1]]


def _write(st, at, T):
    """Rows k_new, v_new (t < count) at row at[b] + t of the cache; the others keep what they hold."""
    B, Hkv, S, half = st["k4"].shape
    t = torch.arange(T, device=DEV)
    ok = t < (torch.full_like(at, T) if st["count"] is None else st["count"].long()).view(B, 1)
    ok, row = ok.view(B, 1, T, 1), (at.view(B, 1) + t).view(B, 1, T, 1)
    for codes, step, new in ((st["k4"], st["step"][..., 0, :], st["k_new"]), (st["v4"], st["step"][..., 1, :], st["v_new"])):
        for held, x in zip((codes, step), _quantise(new)):
            there = row.expand(B, Hkv, T, held.shape[-1])
            held.scatter_(2, there, torch.where(ok, x, held.gather(2, there)))


def _read(st, first, T, dt):
    """Rows first[b] + t for t < count[b], zeros past them."""
    B, Hkv, S, half = st["k4"].shape
    t = torch.arange(T, device=DEV)
    ok = t < (torch.full_like(first, T) if st["count"] is None else st["count"].long()).view(B, 1)
    row = (first.view(B, 1) + t).clamp(max=S - 1).view(B, 1, T, 1)
    out = []
    for i, codes in enumerate((st["k4"], st["v4"])):
        x = _values(codes.gather(2, row.expand(B, Hkv, T, half)), st["step"][..., i, :].gather(
            2, row.expand(B, Hkv, T, st["step"].shape[-1])))
        out.append(x.masked_fill(~ok.view(B, 1, T, 1), 0.0).to(dt))
    return out


def _run_plain(st):
    case = st["case"]
    kind, S, T = case["kind"], case["S"], case["T"]
    lens = st["lens"].long()
    if kind == "write":
        _write(st, lens, T)
        return _read(st, lens, T, st["k_new"].dtype)
    if kind == "read":
        return _read(st, st["first"].long(), T, DTYPES[case["dtype"]])
    if kind == "step":
        _write(st, st["start"].long(), T)
    k, v = _values(st["k4"], st["step"][..., 0, :]), _values(st["v4"], st["step"][..., 1, :])
    B, Hkv, _, D = k.shape
    q = st["q"].float()
    Hq = q.shape[1]
    G = Hq // Hkv
    count = torch.full_like(lens, T) if st["count"] is None else st["count"].long()
    row, t = torch.arange(S, device=DEV), torch.arange(T, device=DEV)
    q = q.reshape(B, Hkv, G * T, D) * D ** -0.5
    seen = (lens.view(B, 1) - count.view(B, 1) + t + 1).clamp(min=0)             # rows that query t sees
    seen = torch.where(t < count.view(B, 1), seen, 0)
    ok = row < seen.view(B, 1, 1, T, 1)
    s = torch.matmul(q, k.transpose(-1, -2)).view(B, Hkv, G, T, S).masked_fill(~ok, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (s - top).exp()
    total = p.sum(-1, keepdim=True)
    acc = torch.matmul(p.view(B, Hkv, G * T, S), v).view(B, Hkv, G, T, D)
    o = (acc / total.masked_fill(total == 0, 1.0)).reshape(B, Hq, T, D)
    if st["gate"] is not None:
        o = o / (1 + (-st["gate"].float()).exp())
    return [o.to(st["q"].dtype), (top + total.log()).reshape(B, Hq, T)]


# ---------------------------------------------------------------------- work
def work(case):
    """Inputs read once and outputs written once (of a cache the rows that
    sequences hold); multiply-adds of the visible (query, key) pairs."""
    kind, s, Hkv, D, T = case["kind"], 4 if case["dtype"] == "fp32" else 2, case["Hkv"], case["D"], case["T"]
    held = D // 2 + 2 * _groups(D)                        # bytes of a key or value row
    lens, counts = _lens(case), _counts(case)
    rows, padded = Hkv * sum(counts), Hkv * case["B"] * T
    if kind == "write":
        return {"bytes": 2 * rows * (D * s + held) + 2 * padded * D * s, "flops": 0}
    if kind == "read":
        return {"bytes": 2 * rows * held + 2 * padded * D * s, "flops": 0}
    Hq = case["Hq"]
    new = Hq * case["B"] * T
    pairs = Hq * sum(sum(max(0, n - c + t + 1) for t in range(c)) for n, c in zip(lens, counts))
    byt = (3 if case["gate"] else 2) * new * D * s + 4 * new + 2 * Hkv * sum(lens) * held
    if kind == "step":
        byt += 2 * rows * D * s
    return {"bytes": byt, "flops": 4 * pairs * D}


# ------------------------------------------------- the same in 64 bits (torch)
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_rows(x):
    """Rows x (..., D), in 64 bits: the values that the cache holds for them."""
    least, most = (-23, 10752.0) if x.dtype == torch.float16 else (-125, 42 * 2.0 ** 120)
    powers = torch.tensor([2.0 ** i for i in range(-200, 200)], dtype=torch.float64, device=x.device)
    out = x.double().clone()
    for g in range(0, x.shape[-1], 64):
        y = out[..., g:g + 64]
        m = y.abs().amax(-1, keepdim=True) / 6
        # the power of two at or below m, over 32: the last of 6 significant bits
        unit = powers[torch.searchsorted(powers, m, right=True).sub(6).clamp(min=least + 200)]
        step = torch.round(m / unit).mul(unit).clamp(max=most)
        t = y / step.masked_fill(step == 0, 1.0)
        a = t.abs()
        # spacing of the 4-bit floats at a; round() takes ties to the even one
        gap = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        out[..., g:g + 64] = torch.sign(t) * (torch.round(a / gap) * gap).clamp(max=6.0) * step
    return out


def _exact_held(st, which, b, h, lo, hi):
    """Rows [lo, hi) of a head's keys (0) or values (1), from the bytes."""
    codes = st["k4" if which == 0 else "v4"][b, h, lo:hi].int()
    table = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device=DEV)
    out = torch.empty(hi - lo, codes.shape[1] * 2, dtype=torch.float64, device=DEV)
    out[:, 0::2], out[:, 1::2] = table[codes % 16], table[codes // 16]
    for g in range(st["step"].shape[-1]):
        out[:, 64 * g:64 * g + 64] *= st["step"][b, h, lo:hi, which, g:g + 1].double()
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind, B, Hkv, D, T = (case[x] for x in ("kind", "B", "Hkv", "D", "T"))
    lens, counts = _lens(case), _counts(case)
    if kind in ("write", "read"):
        out = [torch.zeros(B, Hkv, T, D, dtype=torch.float64, device=DEV) for _ in range(2)]
        for i, x in enumerate(out):
            for b, (n, c) in enumerate(zip(lens, counts)):
                for h in range(Hkv):
                    if kind == "write":
                        x[b, h, :c] = _exact_rows(st["k_new" if i == 0 else "v_new"][b, h, :c])
                    else:
                        x[b, h, :c] = _exact_held(st, i, b, h, n - c, n)
        return out
    Hq = case["Hq"]
    G = Hq // Hkv
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=DEV)
    for h in range(Hkv):
        for b, (n, c) in enumerate(zip(lens, counts)):
            kb, vb = _exact_held(st, 0, b, h, 0, n), _exact_held(st, 1, b, h, 0, n)
            if kind == "step":
                kb[n - 1:], vb[n - 1:] = _exact_rows(st["k_new"][b, h]), _exact_rows(st["v_new"][b, h])
            hide = torch.arange(n, device=DEV) > (n - c + torch.arange(c, device=DEV)).view(c, 1)
            for g in range(h * G, h * G + G):
                x = (st["q"][b, g, :c].double() @ kb.t()).div_(math.sqrt(D)).masked_fill_(hide, -math.inf)
                lse[b, g, :c] = x.logsumexp(-1)
                o[b, g, :c] = x.sub_(lse[b, g, :c].unsqueeze(-1)).exp_() @ vb
    if case["gate"]:
        o *= st["gate"].double().sigmoid()
    return [o, lse]
